"""Attention over the 4-bit cache where the groups of a value row differ: a group of 64 values that stands for
NaN beside one of numbers, and groups (or rows) whose scales lie far apart. What one group holds must not reach
the others. Each group is compared with the 64-bit form of the channels of that group alone, so that a group of
small values is held to a tolerance of its own.
"""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O
from test_gpu_kv4 import DEV, DT, OUT_EPS, W_EPS, Cache, _status, f32, f64, gen, slots_of  # noqa: F401

pytestmark = pytest.mark.gpu


def check_groups(q, out, k, v, scaling, dtype, nan=()):
    """out [Hq, D] against the attention over k [n, Hk, D], v [n, Hv, D], group by group. nan: the
    (value head, group) pairs that stand for NaN."""
    q, out = f64(q), f64(out)
    hq, hv = q.shape[0], v.shape[1]
    ok = np.ones((k.shape[1], k.shape[0]), bool)
    for g in range(q.shape[1] // 64):
        only = np.zeros_like(v)
        only[..., 64 * g:64 * g + 64] = v[..., 64 * g:64 * g + 64]
        for vh, ng in nan:
            if ng == g:
                only[:, vh] = 0
        ref, tol = O.attention(q, k, only, ok, scaling, W_EPS[dtype])
        tol += OUT_EPS[dtype] * np.abs(ref) + 2.0 ** -25 * (dtype == "fp16")
        for h in range(hq):
            at = slice(64 * g, 64 * g + 64)
            if (h // (hq // hv), g) in nan:
                assert np.isnan(out[h, at]).all()
            else:
                err = np.abs(out[h, at] - ref[h, at])
                assert (err <= tol[h, at]).all(), f"head {h}, group {g}: {err.max():.3e} over {tol[h, at].min():.3e}"


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("lens", [[256, 700], [20000, 9001]], ids=["one CTA", "cut"])
def test_a_nan_value_group_stays_in_its_group(lens, what, dtype):
    """One token of request 0 has a value group that is not finite; its keys are numbers."""
    from saga_b200 import kv4
    hq, hk, hv, d, pl, at = 12, 1, 4, 128, 128, 40
    c = Cache(lens, hk, hv, d, pl, dtype, seed=21)
    k = torch.randn((1, hk, d), generator=gen(1), device=DEV).to(DT[dtype])
    v = torch.randn((1, hv, d), generator=gen(2), device=DEV).to(DT[dtype])
    v[0, 1, 5] = float(what)      # the first group of value head 1
    v[0, 2, 127] = float(what)    # the second of value head 2
    kv4.kv4_write(c.pool, k, v, slots_of(c.table, 0, at + 1, pl, at))
    c.k[0][at], c.v[0][at] = O.rows_value(f32(k))[0], O.rows_value(f32(v))[0]
    q = torch.randn((2, hq, 1, d), generator=gen(3), device=DEV).to(DT[dtype])
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens)
    check_groups(q[0, :, 0], out[0, :, 0], c.k[0], c.v[0], d ** -0.5, dtype, nan=[(1, 0), (2, 1)])
    check_groups(q[1, :, 0], out[1, :, 0], c.k[1], c.v[1], d ** -0.5, dtype)


@pytest.mark.parametrize("dtype,ratio", [("bf16", 1e8), ("bf16", 1e12), ("bf16", 1e30), ("fp32", 1e8), ("fp32", 1e12),
                                         ("fp32", 1e30), ("fp16", 1e8)])
@pytest.mark.parametrize("great", [0, 1])
@pytest.mark.parametrize("lens", [[300], [20000]], ids=["one CTA", "cut"])
def test_groups_of_values_far_apart(lens, great, dtype, ratio):
    """One group of every value row is `ratio` times greater than the other."""
    from saga_b200 import kv4
    hq, hk, hv, d, pl, n = 12, 1, 2, 128, 128, lens[0]
    c = Cache(lens, hk, hv, d, pl, dtype, seed=31)
    v = torch.randn((n, hv, d), generator=gen(4), device=DEV)
    v[..., 64 * great:64 * great + 64] *= ratio ** 0.5
    v[..., 64 - 64 * great:128 - 64 * great] *= ratio ** -0.5
    v = v.to(DT[dtype])
    k = torch.randn((n, hk, d), generator=gen(5), device=DEV).to(DT[dtype])
    kv4.kv4_write(c.pool, k, v, slots_of(c.table, 0, n, pl))
    q = torch.randn((1, hq, 1, d), generator=gen(6), device=DEV).to(DT[dtype])
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens)
    check_groups(q[0, :, 0], out[0, :, 0], O.rows_value(f32(k)), O.rows_value(f32(v)), d ** -0.5, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", [0, 3, 40, 600])
def test_rows_of_values_far_apart(at, d, dtype):
    """A row 10^12 times greater than the others whose weight is below 2^-90 of theirs: it adds less than 2^-48
    of a value, so the attention over the other rows is what the result is compared with."""
    from saga_b200 import kv4
    n, pl = 700, 64
    c = Cache([n], 1, 1, d, pl, dtype, seed=41)
    q = torch.randn((1, 2, 1, d), generator=gen(7), device=DEV)
    q[:, 1] = q[:, 0] * 0.9
    q = q.to(DT[dtype])
    k = torch.randn((n, 1, d), generator=gen(8), device=DEV) * 0.1
    q0 = q[0, 0, 0].float()
    k[at, 0] = -q0 * (90.0 * d ** 0.5 / float(q0 @ q0))        # scores of -90 and -81: e^-81 = 2^-116
    v = torch.randn((n, 1, d), generator=gen(9), device=DEV)
    v[at] *= 1e12
    k, v = k.to(DT[dtype]), v.to(DT[dtype])
    kv4.kv4_write(c.pool, k, v, slots_of(c.table, 0, n, pl))
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens)
    others = [i for i in range(n) if i != at]
    check_groups(q[0, :, 0], out[0, :, 0], O.rows_value(f32(k))[others], O.rows_value(f32(v))[others], d ** -0.5, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("size", [1e-30, 1.0, 1e20, 1e30, -1e30])
def test_value_rows_of_one_value(size, dtype):
    """Constant rows have the least scale, 2^-40, beside an offset of any size."""
    from saga_b200 import kv4
    n, d, pl = 200, 128, 64
    c = Cache([n], 1, 2, d, pl, dtype, seed=51)
    v = torch.full((n, 2, d), size, device=DEV).to(DT[dtype])
    k = torch.randn((n, 1, d), generator=gen(10), device=DEV).to(DT[dtype])
    kv4.kv4_write(c.pool, k, v, slots_of(c.table, 0, n, pl))
    q = torch.randn((1, 4, 1, d), generator=gen(11), device=DEV).to(DT[dtype])
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens)
    check_groups(q[0, :, 0], out[0, :, 0], O.rows_value(f32(k)), O.rows_value(f32(v)), d ** -0.5, dtype)


@pytest.mark.parametrize("heads,d", [((12, 1, 2), 128), ((8, 2, 4), 64), ((16, 4, 4), 128)], ids=str)
@pytest.mark.parametrize("n", [1021, 20000])
def test_fp32_is_as_exact_as_binary32(n, heads, d):
    """Over many positions the weights' relative errors average out like the result, so its relative error, over
    all heads, is the rms error of a weight. The scores, in powers of two and below 8, are rounded in binary32 about
    six times on their way: rms 2^-22 / 3^0.5 * 6^0.5 * ln 2 = 2.3e-7. The exponential is within 2^-22, the two terms
    of a query and of a weight within 2^-23 each: together rms 3.7e-7 at most. 2^-20 is 2.6 times that."""
    from saga_b200 import kv4
    hq, hk, hv = heads
    c = Cache([n], hk, hv, d, 128, "fp32", seed=61)
    q = torch.randn((1, hq, 1, d), generator=gen(12), device=DEV)
    out = f64(kv4.kv4_decode(q, c.pool, c.table, c.device_lens))[0, :, 0]
    ref, _ = O.attention(f64(q[0, :, 0]), c.k[0], c.v[0], np.ones((hk, n), bool), float(np.float32(d ** -0.5)), 0.0)
    assert np.linalg.norm(out - ref) <= 2.0 ** -20 * np.linalg.norm(ref)
