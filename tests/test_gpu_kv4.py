"""The 4-bit paged cache operators against plain 64-bit forms (oracle/kv4_oracle.py).

Quantised rows, bounds, block selections and page tables have to be equal bit
for bit; attention within the tolerance that the oracle derives from the
formats plus the rounding of the output type.
"""
import random

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# half an ulp of the output type (8, 11 and 24 significant bits); relative error of a weight: one
# rounding to fp16 (2^-11), or the two fp16 terms of fp32 (2^-22) and ex2 (2^-22)
OUT_EPS = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
W_EPS = {"bf16": 2.0 ** -11, "fp16": 2.0 ** -11, "fp32": 2.0 ** -20}


@pytest.fixture(autouse=True)
def _status():
    from saga_b200 import ops
    ops.read_status(DEV)
    yield
    ops.read_status(DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def f64(t):
    return t.detach().double().cpu().numpy()


def f32(t):
    return t.detach().float().cpu().numpy()


def slots_of(table, b, n, pl, start=0):
    pos = torch.arange(start, n, device=DEV)
    return table[b][pos // pl].long() * pl + pos % pl


class Cache:
    """A pool filled with requests of given lengths, and what it stands for."""

    def __init__(self, lens, hk, hv, d, pl, dtype="bf16", seed=0, bounds=False, scale=1.0, extra_pages=3,
                 garbage=True, offset=0.0):
        from saga_b200 import kv4
        self.lens, self.pl, self.d = lens, pl, d
        per = [(n + pl - 1) // pl for n in lens]
        pages = sum(per) + extra_pages
        self.pool = kv4.Kv4Pool(pages, pl, hk, hv, d, device=DEV, bounds=bounds)
        if garbage:  # what no request owns is full of NaN scales and every code
            self.pool.k.fill_(0xFF)
            self.pool.v.fill_(0xFF)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        width = max(per + [1]) + 1
        self.table = torch.full((len(lens), width), 0x7FFFFFF0, dtype=torch.int32, device=DEV)  # unused entries
        at = 0
        self.k, self.v = [], []
        g = gen(seed)
        for b, n in enumerate(lens):
            self.table[b, :per[b]] = order[at:at + per[b]].to(DEV)
            at += per[b]
            k = (torch.randn((n, hk, d), generator=g, device=DEV) * scale + offset).to(DT[dtype])
            v = (torch.randn((n, hv, d), generator=g, device=DEV) * 0.5).to(DT[dtype])
            kv4.kv4_write(self.pool, k, v, slots_of(self.table, b, n, pl))
            self.k.append(O.rows_value(f32(k)))
            self.v.append(O.rows_value(f32(v)))
        self.device_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def check(self, q, out, dtype, scaling, allowed=None, starts=None):
        out = f64(out)
        for b, n in enumerate(self.lens):
            ok = np.ones((self.k[b].shape[1], n), dtype=bool)
            if starts is not None:
                ok[:, :starts[b]] = False
            if allowed is not None:
                ok &= allowed[b]
            ref, tol = O.attention(f64(q[b, :, 0]), self.k[b], self.v[b], ok, scaling, W_EPS[dtype])
            tol = tol + OUT_EPS[dtype] * np.abs(ref) + 2.0 ** -25 * (dtype != "bf16")
            err = np.abs(out[b, :, 0] - ref)
            assert np.isfinite(out[b]).all()
            worst = (err - tol).max()
            assert worst <= 0, f"request {b} (len {n}): error {err.max():.3e} over tolerance by {worst:.3e}"


# ---------------------------------------------------------------------------
# writes, reads, bounds
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hk,hv,d,pl,T", [(1, 2, 128, 128, 300), (1, 5, 64, 64, 77), (3, 1, 128, 32, 1),
                                          (2, 2, 64, 256, 513), (4, 8, 128, 64, 33)])
def test_write_then_read_is_the_definition(dtype, hk, hv, d, pl, T):
    from saga_b200 import kv4
    g = gen(T)
    k = (torch.randn((T, hk, d), generator=g, device=DEV) * 3).to(DT[dtype])
    v = torch.randn((T, hv, d), generator=g, device=DEV).to(DT[dtype])
    pages = T // pl + 3
    slots = torch.randperm(pages * pl, generator=g, device=DEV)[:T]
    slots[T // 2] = -1
    pool = kv4.Kv4Pool(pages, pl, hk, hv, d, device=DEV)
    kv4.kv4_write(pool, k, v, slots)
    for out_dtype in DT.values():
        rk, rv = kv4.kv4_read(pool, slots, dtype=out_dtype)
        for got, x in ((rk, k), (rv, v)):
            ref = O.rows_value(f32(x))
            ref[T // 2] = 0.0
            ref = torch.from_numpy(ref).to(torch.float32).to(out_dtype)  # exact to binary32: one rounding
            assert torch.equal(got.cpu(), ref)


def test_write_takes_strided_and_unaligned_rows():
    from saga_b200 import kv4
    T, hk, hv, d, pl = 70, 2, 3, 64, 64
    g = gen(1)
    slots = torch.randperm(3 * pl, generator=g, device=DEV)[:T]
    ref = None
    base_k = torch.randn((T, hk, d), generator=g, device=DEV).to(torch.bfloat16)
    base_v = torch.randn((T, hv, d), generator=g, device=DEV).to(torch.bfloat16)
    wide_k = torch.zeros((T, hk, d + 3), dtype=torch.bfloat16, device=DEV)
    wide_k[:, :, 1:d + 1] = base_k
    views = [(base_k, base_v), (base_k.transpose(0, 1).contiguous().transpose(0, 1), base_v),
             (wide_k[:, :, 1:d + 1], base_v.transpose(0, 1).contiguous().transpose(0, 1)),
             (torch.flip(torch.flip(base_k, [0]).contiguous(), [0]), base_v)]
    for k, v in views:
        pool = kv4.Kv4Pool(3, pl, hk, hv, d, device=DEV)
        kv4.kv4_write(pool, k, v, slots)
        got = (pool.k.clone(), pool.v.clone())
        ref = ref or got
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d", [64, 128])
def test_unaligned_rows_of_every_type(dtype, d):
    """Rows that start between 16-byte boundaries are written as aligned ones are, and read so by the C entry."""
    from saga_b200 import _lib as L
    from saga_b200 import kv4
    T, hk, hv, pl = 300, 1, 2, 32
    g = gen(3)
    slots = torch.randperm(10 * pl, generator=g, device=DEV)[:T]
    k, v = (torch.randn((T, h, d), generator=g, device=DEV).to(DT[dtype]) for h in (hk, hv))
    wide = [torch.full((T, h, d + 3), 7.0, dtype=DT[dtype], device=DEV) for h in (hk, hv)]
    for w, x in zip(wide, (k, v)):
        w[:, :, 1:d + 1] = x
    pools = [kv4.Kv4Pool(10, pl, hk, hv, d, device=DEV) for _ in range(2)]
    kv4.kv4_write(pools[0], k, v, slots)
    kv4.kv4_write(pools[1], wide[0][:, :, 1:d + 1], wide[1][:, :, 1:d + 1], slots)
    assert torch.equal(pools[0].k, pools[1].k) and torch.equal(pools[0].v, pools[1].v)
    want = kv4.kv4_read(pools[0], slots, DT[dtype])
    at = [w[:, :, 1:d + 1] for w in wide]
    rc = L.lib.saga_kv4_read(pools[0]._ref, {"bf16": L.SAGA_BF16, "fp16": L.SAGA_FP16, "fp32": L.SAGA_FP32}[dtype], T,
                             slots.data_ptr(), at[0].data_ptr(), at[0].stride(0), at[0].stride(1), at[1].data_ptr(),
                             at[1].stride(0), at[1].stride(1), None, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    for w, x in zip(wide, want):
        assert torch.equal(w[:, :, 1:d + 1], x)
        assert (w[:, :, 0] == 7).all() and (w[:, :, d + 1:] == 7).all()


def test_one_value_for_all_heads_and_tokens():
    """Broadcast rows (zero strides)."""
    from saga_b200 import kv4
    d, pl = 64, 32
    row = torch.randn(d, generator=gen(2), device=DEV).to(torch.bfloat16)
    k, v = row.expand(5, 2, d), row.expand(5, 3, d)
    pool = kv4.Kv4Pool(1, pl, 2, 3, d, device=DEV)
    slots = torch.arange(5, device=DEV)
    kv4.kv4_write(pool, k, v, slots)
    rk, rv = kv4.kv4_read(pool, slots, dtype=torch.float32)
    ref = torch.from_numpy(O.rows_value(f32(row))).float().to(DEV)
    assert torch.equal(rk, ref.expand_as(rk)) and torch.equal(rv, ref.expand_as(rv))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_write_special_groups(dtype):
    """Constant, tiny, huge, signed-zero, NaN and infinite groups."""
    from saga_b200 import kv4
    d, pl = 128, 32
    rows = torch.zeros((12, 1, d))
    rows[1] = 3.7
    rows[2] = -0.0
    rows[3, 0, :64] = torch.linspace(-1e-13, 1e-13, 64)
    rows[4] = torch.linspace(-1.5e38, 1.5e38, d)
    rows[5] = torch.linspace(-3.3e38, 3.3e38, d)        # the range overflows: NaN
    rows[6, 0, 5] = float("nan")                        # one group only
    rows[7, 0, 100] = float("inf")
    rows[8, 0, 0] = float("-inf")
    rows[9] = 1000.0 + torch.linspace(0, 1, d)
    rows[10, 0, ::2] = 1e-30
    rows[11] = torch.linspace(-2, -1, d)
    k = rows.to(DT[dtype]).to(DEV)
    pool = kv4.Kv4Pool(1, pl, 1, 1, d, device=DEV)
    slots = torch.arange(12, device=DEV)
    kv4.kv4_write(pool, k, k, slots)
    got = kv4.kv4_read(pool, slots, dtype=torch.float32)[0].cpu().numpy()
    ref = O.rows_value(f32(k)).astype(np.float32)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got[~np.isnan(ref)], ref[~np.isnan(ref)])
    assert np.isnan(got[6, 0, :64]).all() and np.isfinite(got[6, 0, 64:]).all()


def test_slots_outside_the_pool_are_skipped_and_reported():
    from saga_b200 import _lib, kv4, ops
    d, pl = 64, 32
    k = torch.ones((4, 1, d), device=DEV, dtype=torch.bfloat16)
    pool = kv4.Kv4Pool(2, pl, 1, 1, d, device=DEV)
    slots = torch.tensor([3, -1, 2 * pl, -7], device=DEV)
    kv4.kv4_write(pool, k, k, slots)
    assert ops.read_status(DEV) == _lib.STATUS_PAGE_RANGE
    rk, _ = kv4.kv4_read(pool, torch.arange(2 * pl, device=DEV), dtype=torch.float32)
    assert rk[3].abs().sum() > 0 and int((rk.abs().sum((1, 2)) > 0).sum()) == 1
    assert ops.read_status(DEV) == 0
    rk, rv = kv4.kv4_read(pool, slots)
    assert ops.read_status(DEV) == _lib.STATUS_PAGE_RANGE
    assert float(rk[1:].abs().sum()) == 0 and float(rv[1:].abs().sum()) == 0 and float(rk[0, 0, 0]) == 1
    empty = torch.zeros(0, dtype=torch.int64, device=DEV)
    kv4.kv4_write(pool, k[:0], k[:0], empty)
    assert kv4.kv4_read(pool, empty)[0].shape == (0, 1, d)


@pytest.mark.parametrize("d,pl,hk", [(128, 128, 1), (64, 32, 3), (128, 64, 2)])
def test_bounds_of_completed_pages(d, pl, hk):
    from saga_b200 import kv4
    n = 5 * pl - 3
    c = Cache([n, 2 * pl], hk, 1, d, pl, seed=4, bounds=True, scale=2.0)
    for b, length in enumerate(c.lens):
        for p in range(length // pl):
            page = int(c.table[b, p])
            for h in range(hk):
                lo, hi = O.page_bounds(c.k[b][p * pl:(p + 1) * pl, h])
                assert np.array_equal(f32(c.pool.k_lo[page, h]), lo) and np.array_equal(f32(c.pool.k_hi[page, h]), hi)
    # the last three tokens, one at a time, complete the fifth page; a NaN row is left out
    page = int(c.table[0, 4])
    before = c.pool.k_lo[page].clone()
    vals = c.k[0][4 * pl:]
    for i in range(3):
        assert torch.equal(c.pool.k_lo[page], before)
        k = torch.randn((1, hk, d), generator=gen(i), device=DEV).to(torch.bfloat16)
        if i == 1:
            k[:] = float("nan")
        kv4.kv4_write(c.pool, k, k[:, :1], slots_of(c.table, 0, n + i + 1, pl, n + i))
        vals = np.concatenate((vals, O.rows_value(f32(k))))
    for h in range(hk):
        lo, hi = O.page_bounds(vals[:, h])
        assert np.array_equal(f32(c.pool.k_lo[page, h]), lo) and np.array_equal(f32(c.pool.k_hi[page, h]), hi)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

HEADS = [(12, 1, 2), (12, 1, 4), (15, 1, 5), (4, 4, 4), (8, 2, 4), (6, 2, 1), (32, 1, 1), (24, 1, 3), (12, 2, 3),
         (16, 1, 16), (20, 1, 4), (1, 1, 1), (32, 2, 8), (12, 3, 2)]
LENS = [1, 0, 31, 32, 33, 127, 128, 129, 255, 700]


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("d,dtype", [(128, "bf16"), (64, "fp16"), (128, "fp32"), (64, "fp32")])
def test_decode_heads_and_lengths(heads, d, dtype):
    from saga_b200 import kv4, ops
    hq, hk, hv = heads
    c = Cache(LENS, hk, hv, d, 64, dtype, seed=hq + d)
    q = torch.randn((len(LENS), hq, 1, d), generator=gen(9), device=DEV).to(DT[dtype])
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens)
    c.check(q, out, dtype, d ** -0.5)
    assert float(out[1].abs().sum()) == 0  # no positions: zeros
    assert ops.read_status(DEV) == 0
    for _ in range(2):
        assert torch.equal(kv4.kv4_decode(q, c.pool, c.table, c.device_lens), out)


@pytest.mark.parametrize("pl", [32, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_decode_long_items_cut_by_cta_borders(pl, dtype):
    from saga_b200 import kv4
    lens = [9001, 5, 20000, 0, 1, 3333]
    c = Cache(lens, 1, 2, 128, pl, dtype, seed=pl)
    q = torch.randn((len(lens), 12, 1, 128), generator=gen(3), device=DEV).to(DT[dtype]) * 2
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens)
    c.check(q, out, dtype, 128 ** -0.5)
    assert torch.equal(kv4.kv4_decode(q, c.pool, c.table, c.device_lens), out)


def test_decode_many_short_requests():
    """More (request, key head) rows than threads of a CTA."""
    from saga_b200 import kv4
    rng = random.Random(1)
    lens = [rng.choice((0, 1, 7, 40, 64, 65, 100)) for _ in range(330)]
    c = Cache(lens, 2, 2, 64, 32, seed=8)
    q = torch.randn((len(lens), 4, 1, 64), generator=gen(5), device=DEV).to(torch.bfloat16)
    c.check(q, kv4.kv4_decode(q, c.pool, c.table, c.device_lens), "bf16", 64 ** -0.5)
    none = torch.zeros_like(c.device_lens)
    assert float(kv4.kv4_decode(q, c.pool, c.table, none).abs().sum()) == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_decode_starts(dtype):
    """Sliding windows and left padding: positions before the start are not read into the result, whatever
    they hold; a start at or past the length leaves nothing."""
    from saga_b200 import kv4
    lens = [700, 700, 700, 64, 1, 5000, 33]
    starts = [0, 31, 699, 64, 5, 4100, 32]
    c = Cache(lens, 1, 2, 128, 64, dtype, seed=2)
    bad = torch.full((1, 2, 128), float("nan"), dtype=DT[dtype], device=DEV)
    for b, s in enumerate(starts):
        if 0 < s <= lens[b]:  # the position just before the window stands for NaN
            kv4.kv4_write(c.pool, bad[:, :1], bad, slots_of(c.table, b, s, 64, s - 1))
            c.k[b][s - 1] = 0
            c.v[b][s - 1] = 0
    q = torch.randn((len(lens), 12, 1, 128), generator=gen(4), device=DEV).to(DT[dtype])
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens,
                         starts=torch.tensor(starts, dtype=torch.int32, device=DEV))
    c.check(q, out, dtype, 128 ** -0.5, starts=starts)
    assert float(out[3].abs().sum()) == 0 and float(out[4].abs().sum()) == 0


def test_decode_nan_rows_reach_their_heads_only():
    from saga_b200 import kv4
    c = Cache([300, 300], 2, 4, 128, 64, seed=6)
    nan = torch.full((1, 2, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    one = torch.zeros((1, 4, 128), dtype=torch.bfloat16, device=DEV)
    nan[:, 0] = 0.1                      # key head 1 of request 0 only
    one[0, 3, 10] = float("inf")         # and the first group of value head 3
    kv4.kv4_write(c.pool, nan, one, slots_of(c.table, 0, 78, 64, 77))
    q = torch.randn((2, 8, 1, 128), generator=gen(7), device=DEV).to(torch.bfloat16)
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens)
    bad = torch.isnan(out).cpu()
    assert not bad[1].any() and not bad[0, :4].any() and bad[0, 4:].all()


@pytest.mark.parametrize("scaling", [None, 0.0, -0.3, 2.5])
def test_decode_scaling_and_peaked_weights(scaling):
    from saga_b200 import kv4
    c = Cache([2000], 1, 2, 64, 128, "fp16", seed=11, scale=2.0)
    q = (torch.randn((1, 8, 1, 64), generator=gen(12), device=DEV) * 3).half()
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens, scaling=scaling)
    c.check(q, out, "fp16", 64 ** -0.5 if scaling is None else scaling)


@pytest.mark.parametrize("size", [1e-30, 1e-4, 1.0, 1e4, 1e30])
def test_decode_query_and_value_sizes(size):
    """Queries and values far from one: the products run in fp16, about the greatest of each."""
    from saga_b200 import kv4
    n, d = 500, 128
    pool = kv4.Kv4Pool(4, 128, 1, 2, d, device=DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    g = gen(13)
    k = torch.randn((n, 1, d), generator=g, device=DEV)
    v = torch.randn((n, 2, d), generator=g, device=DEV) * size
    v[250] *= 1e-3  # a token whose values are small beside the others
    kv4.kv4_write(pool, k, v, torch.arange(n, device=DEV))
    q = torch.randn((1, 4, 1, d), generator=g, device=DEV) * size
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    scaling = d ** -0.5 / size
    out = f64(kv4.kv4_decode(q, pool, table, lens, scaling=scaling))
    ref, tol = O.attention(f64(q[0, :, 0]), O.rows_value(f32(k)), O.rows_value(f32(v)), np.ones((1, n), bool),
                           float(np.float32(scaling)), W_EPS["fp32"])
    assert (np.abs(out[0, :, 0] - ref) <= tol + 2.0 ** -24 * np.abs(ref)).all()


def test_decode_one_huge_value_row_that_hardly_counts():
    """A row 10^5 times greater than the others, in the same tile, with a weight of nearly zero."""
    from saga_b200 import kv4
    n, d = 64, 64
    pool = kv4.Kv4Pool(1, 64, 1, 1, d, device=DEV)
    g = gen(14)
    q = torch.randn((1, 2, 1, d), generator=g, device=DEV)
    k = torch.randn((n, 1, d), generator=g, device=DEV) * 0.1
    k[40] = -30 * q[0, :, 0].sum(0) / q[0, :, 0].norm()
    v = torch.randn((n, 1, d), generator=g, device=DEV)
    v[40] *= 1e5
    kv4.kv4_write(pool, k, v, torch.arange(n, device=DEV))
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    out = f64(kv4.kv4_decode(q, pool, torch.zeros((1, 1), dtype=torch.int32, device=DEV), lens))
    ref, _ = O.attention(f64(q[0, :, 0]), O.rows_value(f32(k)), O.rows_value(f32(v)), np.ones((1, n), bool), d ** -0.5,
                         0.0)
    assert np.abs(out[0, :, 0] - ref).max() <= 2.0 ** -10 * np.abs(ref).max()


def test_decode_strided_queries_and_table():
    from saga_b200 import kv4
    c = Cache([300, 65, 200], 1, 2, 64, 64, "fp16", seed=15)
    base = torch.randn((3, 2, 12, 1, 64 + 5), generator=gen(16), device=DEV).half()
    q = base[:, 1, :, :, 3:67]
    ref = kv4.kv4_decode(q.contiguous(), c.pool, c.table, c.device_lens)
    assert torch.equal(kv4.kv4_decode(q, c.pool, c.table, c.device_lens), ref)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(kv4.kv4_decode(by_head, c.pool, c.table, c.device_lens), ref)
    wide = torch.full((4, c.table.shape[1] + 9), 7, dtype=torch.int32, device=DEV)
    wide[:3, :c.table.shape[1]] = c.table
    assert torch.equal(kv4.kv4_decode(q, c.pool, wide[:, :c.table.shape[1]], c.device_lens), ref)


def test_decode_reports_pages_and_lengths_out_of_range():
    from saga_b200 import _lib, kv4, ops
    c = Cache([300, 65], 1, 1, 64, 64, seed=17)
    q = torch.randn((2, 4, 1, 64), generator=gen(18), device=DEV).to(torch.bfloat16)
    good = kv4.kv4_decode(q, c.pool, c.table, c.device_lens)
    bad = c.table.clone()
    bad[1, 0] = c.pool.num_pages
    out = kv4.kv4_decode(q, c.pool, bad, c.device_lens)
    assert ops.read_status(DEV) == _lib.STATUS_PAGE_RANGE and torch.equal(out[0], good[0])
    long = torch.tensor([300, 10 ** 9], dtype=torch.int32, device=DEV)
    out = kv4.kv4_decode(q, c.pool, c.table, long)  # cut to the table's row, whose unused entries are bad
    assert ops.read_status(DEV) == _lib.STATUS_PAGE_RANGE and torch.equal(out[0], good[0])
    negative = torch.tensor([300, -5], dtype=torch.int32, device=DEV)
    out = kv4.kv4_decode(q, c.pool, c.table, negative)
    assert ops.read_status(DEV) == 0 and float(out[1].abs().sum()) == 0


def test_offsets_past_32_bits():
    """A pool of more than 4 GiB per side: the last pages are addressed right."""
    from saga_b200 import kv4
    d, pl = 128, 128
    page = pl * (d // 2 + d // 16)
    pages = (5 << 30) // page
    pool = kv4.Kv4Pool(pages, pl, 1, 1, d, device=DEV, bounds=True)
    n = 2 * pl + 7
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device=DEV)
    g = gen(19)
    k = torch.randn((n, 1, d), generator=g, device=DEV).to(torch.bfloat16)
    v = torch.randn((n, 1, d), generator=g, device=DEV).to(torch.bfloat16)
    slots = slots_of(table, 0, n, pl)
    kv4.kv4_write(pool, k, v, slots)
    rk, rv = kv4.kv4_read(pool, slots, dtype=torch.float32)
    assert np.array_equal(f64(rk), O.rows_value(f32(k))) and np.array_equal(f64(rv), O.rows_value(f32(v)))
    q = torch.randn((1, 4, 1, d), generator=g, device=DEV).to(torch.bfloat16)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    out = f64(kv4.kv4_decode(q, pool, table, lens))
    ref, tol = O.attention(f64(q[0, :, 0]), f64(rk), f64(rv), np.ones((1, n), bool), d ** -0.5, W_EPS["bf16"])
    assert (np.abs(out[0, :, 0] - ref) <= tol + OUT_EPS["bf16"] * np.abs(ref)).all()
    lo, _ = O.page_bounds(f64(rk)[:pl, 0])
    assert np.array_equal(f32(pool.k_lo[pages - 1, 0]), lo)


# ---------------------------------------------------------------------------
# block selection
# ---------------------------------------------------------------------------

def _select_ref(c, q, top, first, last):
    hk = c.pool.key_heads
    out = []
    for b, n in enumerate(c.lens):
        rows = []
        for h in range(hk):
            g = q.shape[1] // hk
            lo = np.stack([f32(c.pool.k_lo[int(p), h]) for p in c.table[b, :n // c.pl]]) if n >= c.pl else None
            hi = np.stack([f32(c.pool.k_hi[int(p), h]) for p in c.table[b, :n // c.pl]]) if n >= c.pl else None
            rows.append(O.select(f32(q[b, h * g:(h + 1) * g, 0]), lo, hi, n, c.pl, top, first, last))
        out.append(rows)
    return out


@pytest.mark.parametrize("heads,d,dtype", [((12, 1, 2), 128, "bf16"), ((15, 1, 5), 64, "fp16"), ((8, 2, 4), 64, "fp32"),
                                           ((24, 1, 3), 128, "fp32"), ((4, 4, 4), 128, "bf16"),
                                           ((40, 1, 2), 64, "bf16")], ids=str)
@pytest.mark.parametrize("top,first,last", [(1, 0, 1), (2, 1, 1), (5, 1, 2), (9, 3, 4), (64, 1, 1)])
def test_select_and_sparse_decode(heads, d, dtype, top, first, last):
    from saga_b200 import kv4, ops
    hq, hk, hv = heads
    pl = 32
    c = Cache([1, 0, 31, 32, 33, 700, 1024, 1023, 2500], hk, hv, d, pl, dtype, seed=top + d, bounds=True)
    q = torch.randn((len(c.lens), hq, 1, d), generator=gen(21), device=DEV).to(DT[dtype])
    blocks, counts = kv4.kv4_select(q, c.pool, c.table, c.device_lens, top, keep_first=first, keep_last=last)
    ref = _select_ref(c, q, top, first, last)
    allowed = []
    for b, n in enumerate(c.lens):
        ok = np.zeros((hk, n), bool)
        for h in range(hk):
            assert int(counts[b, h]) == len(ref[b][h])
            assert blocks[b, h].tolist() == ref[b][h] + [-1] * (top - len(ref[b][h]))
            for p in ref[b][h]:
                ok[h, p * pl:(p + 1) * pl] = True
        allowed.append(ok)
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens, blocks=blocks, counts=counts)
    c.check(q, out, dtype, d ** -0.5, allowed=allowed)
    assert ops.read_status(DEV) == 0
    starts = [min(40, n) for n in c.lens]
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens, blocks=blocks, counts=counts,
                         starts=torch.tensor(starts, dtype=torch.int32, device=DEV))
    c.check(q, out, dtype, d ** -0.5, allowed=allowed, starts=starts)


def test_select_ties_go_to_the_lower_page_and_nan_is_last():
    from saga_b200 import kv4
    d, pl, n = 64, 32, 40
    pool = kv4.Kv4Pool(n, pl, 1, 1, d, device=DEV, bounds=True)
    table = torch.arange(n, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([n * pl], dtype=torch.int32, device=DEV)
    pool.k_lo.fill_(1.0)
    pool.k_hi.fill_(1.0)
    pool.k_hi[7] = pool.k_lo[7] = float("nan")
    pool.k_hi[3] = pool.k_lo[3] = -5.0
    pool.k_hi[20] = pool.k_lo[20] = 2.0
    pool.k_hi[21, :, 0] = pool.k_lo[21, :, 0] = -0.0
    q = torch.ones((1, 2, 1, d), device=DEV, dtype=torch.bfloat16)
    blocks, _ = kv4.kv4_select(q, pool, table, lens, 6)
    assert blocks[0, 0].tolist() == [0, 1, 2, 4, 20, 39]
    blocks, _ = kv4.kv4_select(q, pool, table, lens, n - 1)
    assert blocks[0, 0].tolist() == [p for p in range(n) if p != 7]
    blocks, _ = kv4.kv4_select(q, pool, table, lens, n - 2)
    assert blocks[0, 0].tolist() == [p for p in range(n) if p not in (3, 7)]
    zero = torch.zeros_like(q)  # all scores are +0 or -0: the lowest pages
    blocks, _ = kv4.kv4_select(zero, pool, table, lens, 5, keep_first=0)
    assert blocks[0, 0].tolist() == [0, 1, 2, 3, 39]


def test_pages_of_nan_keys_are_selected_last():
    from saga_b200 import kv4
    d, pl = 64, 32
    c = Cache([10 * pl], 1, 1, d, pl, seed=27, bounds=True)
    for p in (4, 6):
        k = torch.full((pl, 1, d), float("nan"), dtype=torch.bfloat16, device=DEV)
        kv4.kv4_write(c.pool, k, k, slots_of(c.table, 0, (p + 1) * pl, pl, p * pl))
        assert torch.isnan(c.pool.k_lo[int(c.table[0, p])].float()).all()
        assert torch.isnan(c.pool.k_hi[int(c.table[0, p])].float()).all()
    q = torch.randn((1, 3, 1, d), generator=gen(28), device=DEV).to(torch.bfloat16)
    blocks, _ = kv4.kv4_select(q, c.pool, c.table, c.device_lens, 8)
    assert blocks[0, 0].tolist() == [0, 1, 2, 3, 5, 7, 8, 9]
    blocks, _ = kv4.kv4_select(q, c.pool, c.table, c.device_lens, 9)
    assert blocks[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 7, 8, 9]


def test_select_nothing_between_the_kept_pages():
    """No scored page is taken; the scores have both signs, so their keys' range has 32 bits."""
    from saga_b200 import kv4
    d, pl, n = 64, 32, 40
    pool = kv4.Kv4Pool(n, pl, 1, 1, d, device=DEV, bounds=True)
    table = torch.arange(n, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([n * pl], dtype=torch.int32, device=DEV)
    x = torch.linspace(-2e30, 2e30, n, device=DEV).to(torch.bfloat16)
    pool.k_lo.copy_(x[:, None, None].expand_as(pool.k_lo))
    pool.k_hi.copy_(pool.k_lo)
    q = torch.ones((1, 2, 1, d), device=DEV, dtype=torch.bfloat16)
    for first, last in ((2, 1), (0, 1), (1, 3)):
        blocks, counts = kv4.kv4_select(q, pool, table, lens, first + last, keep_first=first, keep_last=last)
        assert blocks[0, 0].tolist() == list(range(first)) + list(range(n - last, n))
        assert int(counts[0, 0]) == first + last


def test_select_more_pages_than_fit_shared_memory():
    from saga_b200 import kv4
    d, pl, n, top = 64, 32, 9000, 50
    pool = kv4.Kv4Pool(n, pl, 1, 1, d, device=DEV, bounds=True)
    g = gen(23)
    x = torch.randn((n, 1, d), generator=g, device=DEV).to(torch.bfloat16)
    pool.k_lo.copy_(x)
    pool.k_hi.copy_(x)
    table = torch.randperm(n, generator=g, device=DEV).to(torch.int32)[None]
    q = torch.randn((1, 3, 1, d), generator=g, device=DEV).to(torch.bfloat16)
    lens = torch.tensor([n * pl - 5], dtype=torch.int32, device=DEV)
    blocks, counts = kv4.kv4_select(q, pool, table, lens, top)
    lo = f32(x[table[0].long(), 0])
    assert blocks[0, 0].tolist() == O.select(f32(q[0, :, 0]), lo, lo, n * pl - 5, pl, top)
    assert int(counts[0, 0]) == top


def test_sparse_decode_takes_any_block_list():
    """Blocks with holes (-1) or past the table are left out; counts cut the list; no blocks: zeros."""
    from saga_b200 import kv4
    c = Cache([1000, 1000, 1000], 1, 2, 64, 64, "fp16", seed=25)
    q = torch.randn((3, 4, 1, 64), generator=gen(26), device=DEV).half()
    blocks = torch.tensor([[[0, -1, 5, 15]], [[3, 4, 9, 11]], [[0, 1, 2, 3]]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([[4], [2], [0]], dtype=torch.int32, device=DEV)
    out = kv4.kv4_decode(q, c.pool, c.table, c.device_lens, blocks=blocks, counts=counts)
    allowed = [np.zeros((1, 1000), bool) for _ in range(3)]
    for b, pages in ((0, (0, 5, 15)), (1, (3, 4))):
        for p in pages:
            allowed[b][0, p * 64:(p + 1) * 64] = True
    c.check(q, out, "fp16", 0.125, allowed=allowed)
    assert float(out[2].abs().sum()) == 0


# ---------------------------------------------------------------------------
# page tables
# ---------------------------------------------------------------------------

def _tables_case(rng, B, pl, context, tokens, scarce=False, narrow=False):
    lens = [rng.randint(0, context) for _ in range(B)]
    new = [rng.choice((-1, 0, 1, 1, 1, rng.randint(0, max(1, 2 * tokens // max(B, 1))))) for _ in range(B)]
    held = [-(-n // pl) for n in lens]
    width = (context if narrow else context + max([1] + new)) // pl + 2
    spare = rng.randint(0, 3) if scarce else sum(-(-(n + max(m, 0)) // pl) for n, m in zip(lens, new)) + 2
    total = sum(held) + spare
    perm = list(range(total))
    rng.shuffle(perm)
    table = [[-1] * width for _ in range(B)]
    at = 0
    for b, h in enumerate(held):
        table[b][:h] = perm[at:at + h]
        at += h
    ring = [-9] * total
    first = rng.randint(0, max(total - 1, 0))
    for i, p in enumerate(perm[at:]):
        ring[(first + i) % total] = p
    return lens, new, table, ring, first, total - at


@pytest.mark.parametrize("B,pl,context,tokens", [(1, 32, 100, 5), (7, 64, 300, 40), (64, 128, 4000, 64),
                                                 (33, 32, 500, 3000), (300, 64, 900, 9000), (1500, 32, 200, 2048),
                                                 (5, 256, 0, 700), (2100, 64, 130, 5000)])
@pytest.mark.parametrize("kind", ["plenty", "scarce", "narrow", "few rows"])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_tables(B, pl, context, tokens, kind, in_place):
    from saga_b200 import _lib, kv4, ops
    rng = random.Random(f"{B}{pl}{tokens}{kind}")
    lens, new, table, ring, first, count = _tables_case(rng, B, pl, context, tokens, kind == "scarce",
                                                        kind == "narrow")
    rows = sum(max(m, 0) for m in new)
    num_tokens = rows // 2 if kind == "few rows" else rows + rng.randint(0, 9)
    i32 = dict(dtype=torch.int32, device=DEV)
    t_table, t_ring = torch.tensor(table, **i32), torch.tensor(ring, **i32)
    t_lens, t_state = torch.tensor(lens, **i32), torch.tensor([first, count], **i32)
    step = kv4.page_tables(t_table, t_lens, torch.tensor(new, **i32), t_ring, t_state, num_tokens, pl,
                           lens_out=t_lens if in_place else None, free_state_out=t_state if in_place else None)
    slots, positions, offsets, out_lens, state, failed = O.page_tables(table, lens, new, ring, first, count,
                                                                       num_tokens, pl)
    assert step.slots.tolist() == slots
    assert step.positions.tolist() == positions
    assert step.offsets.tolist() == offsets
    assert step.lens.tolist() == out_lens
    assert tuple(step.free_state.tolist()) == state
    assert t_table.tolist() == table
    assert t_ring.tolist() == ring
    assert ops.read_status(DEV) == (_lib.STATUS_OUT_OF_PAGES if failed else 0)
    assert (step.lens is t_lens) == in_place


def test_page_tables_of_no_requests_and_of_no_pages():
    from saga_b200 import _lib, kv4, ops
    i32 = dict(dtype=torch.int32, device=DEV)
    state = torch.tensor([2, 3], **i32)
    ring = torch.arange(5, **i32)
    none = torch.zeros(0, **i32)
    step = kv4.page_tables(torch.zeros((0, 4), **i32), none, none, ring, state, 3, 64)
    assert step.slots.tolist() == [-1] * 3 and step.offsets.tolist() == [0] and step.free_state.tolist() == [2, 3]
    one = torch.tensor([0, 0], **i32)
    step = kv4.page_tables(torch.zeros((2, 4), **i32), one, torch.tensor([1, -1], **i32), none, torch.zeros(2, **i32),
                           1, 64)
    assert step.slots.tolist() == [-1] and step.lens.tolist() == [0, 0] and step.free_state.tolist() == [0, 0]
    assert ops.read_status(DEV) == _lib.STATUS_OUT_OF_PAGES


@pytest.mark.parametrize("with_starts", [False, True])
def test_slot_map(with_starts):
    from saga_b200 import kv4
    pl = 32
    lens, starts = [70, 0, 1, 500, 64], [3, 5, 0, 499, 32]
    c = Cache(lens, 1, 1, 64, pl, seed=31)
    t = torch.tensor(starts, dtype=torch.int32, device=DEV) if with_starts else None
    total = sum(max(n - (s if with_starts else 0), 0) for n, s in zip(lens, starts))
    slots, offsets = kv4.slot_map(c.table, c.device_lens, total + 4, pl, starts=t)
    ref, offs = [], [0]
    for b, n in enumerate(lens):
        s = starts[b] if with_starts else 0
        if n > s:
            ref += slots_of(c.table, b, n, pl, s).tolist()
        offs.append(len(ref))
    assert slots.tolist() == ref + [-1] * 4 and offsets.tolist() == offs
    k, v = kv4.kv4_read(c.pool, slots[:total], dtype=torch.float32)
    at = slice(offs[3], offs[4])
    first = starts[3] if with_starts else 0
    assert np.array_equal(f64(k[at]), c.k[3][first:]) and np.array_equal(f64(v[at]), c.v[3][first:])
    assert kv4.slot_map(c.table, c.device_lens, 0, pl)[0].numel() == 0


# ---------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------

def test_a_captured_serving_step_advances_by_itself():
    """page_tables (in place), kv4_write, kv4_select and kv4_decode in one CUDA graph: every replay appends a
    token to every request and attends to the grown cache."""
    from saga_b200 import kv4, ops
    B, hq, hk, hv, d, pl, pages = 3, 12, 1, 2, 128, 32, 64
    i32 = dict(dtype=torch.int32, device=DEV)
    pool = kv4.Kv4Pool(pages, pl, hk, hv, d, device=DEV, bounds=True)
    table = torch.full((B, 20), -1, **i32)
    lens, ring, state = torch.zeros(B, **i32), torch.arange(pages, **i32), torch.tensor([0, pages], **i32)
    prompts = [100, 31, 1]
    g = gen(40)
    hist_k, hist_v = [], []
    new = torch.tensor(prompts, **i32)
    step = kv4.page_tables(table, lens, new, ring, state, sum(prompts), pl, lens_out=lens, free_state_out=state)
    k = torch.randn((sum(prompts), hk, d), generator=g, device=DEV).to(torch.bfloat16)
    v = torch.randn((sum(prompts), hv, d), generator=g, device=DEV).to(torch.bfloat16)
    kv4.kv4_write(pool, k, v, step.slots)
    for b, (i, j) in enumerate(zip(step.offsets.tolist(), step.offsets.tolist()[1:])):
        hist_k.append(O.rows_value(f32(k[i:j])))
        hist_v.append(O.rows_value(f32(v[i:j])))
    ones = torch.ones(B, **i32)
    kb, vb = torch.zeros((B, hk, d), dtype=torch.bfloat16, device=DEV), torch.zeros((B, hv, d), dtype=torch.bfloat16,
                                                                                    device=DEV)
    qb = torch.zeros((B, hq, 1, d), dtype=torch.bfloat16, device=DEV)

    def decode_step():
        st = kv4.page_tables(table, lens, ones, ring, state, B, pl, lens_out=lens, free_state_out=state)
        kv4.kv4_write(pool, kb, vb, st.slots)
        blocks, counts = kv4.kv4_select(qb, pool, table, lens, 3)
        return (kv4.kv4_decode(qb, pool, table, lens),
                kv4.kv4_decode(qb, pool, table, lens, blocks=blocks, counts=counts), blocks)

    saved = [t.clone() for t in (lens, ring, state, table, pool.k, pool.v, pool.k_lo, pool.k_hi)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        decode_step()
        for t, s in zip((lens, ring, state, table, pool.k, pool.v, pool.k_lo, pool.k_hi), saved):
            t.copy_(s)
        with torch.cuda.graph(graph, stream=side):
            dense, sparse, blocks = decode_step()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(40):
        kn = torch.randn((B, hk, d), generator=g, device=DEV).to(torch.bfloat16)
        vn = torch.randn((B, hv, d), generator=g, device=DEV).to(torch.bfloat16)
        q = torch.randn((B, hq, 1, d), generator=g, device=DEV).to(torch.bfloat16)
        kb.copy_(kn)
        vb.copy_(vn)
        qb.copy_(q)
        graph.replay()
        for b in range(B):
            hist_k[b] = np.concatenate((hist_k[b], O.rows_value(f32(kn[b:b + 1]))))
            hist_v[b] = np.concatenate((hist_v[b], O.rows_value(f32(vn[b:b + 1]))))
            n = len(hist_k[b])
            assert int(lens[b]) == n == prompts[b] + i + 1
            ok = np.ones((1, n), bool)
            ref, tol = O.attention(f64(q[b, :, 0]), hist_k[b], hist_v[b], ok, d ** -0.5, W_EPS["bf16"])
            assert (np.abs(f64(dense[b, :, 0]) - ref) <= tol + OUT_EPS["bf16"] * np.abs(ref)).all()
            picks = [p for p in blocks[b, 0].tolist() if p >= 0]
            ok[:] = False
            for p in picks:
                ok[0, p * pl:(p + 1) * pl] = True
            lo, hi = zip(*[O.page_bounds(hist_k[b][p * pl:(p + 1) * pl, 0]) for p in range(n // pl)]) if n >= pl else ((), ())
            assert picks == O.select(f32(q[b, :, 0]), lo, hi, n, pl, 3)
            ref, tol = O.attention(f64(q[b, :, 0]), hist_k[b], hist_v[b], ok, d ** -0.5, W_EPS["bf16"])
            assert (np.abs(f64(sparse[b, :, 0]) - ref) <= tol + OUT_EPS["bf16"] * np.abs(ref)).all()
    assert ops.read_status(DEV) == 0


def test_calls_on_two_streams_do_not_share_a_workspace():
    from saga_b200 import kv4
    caches = [Cache([20000 + i, 300], 1, 2, 128, 128, seed=50 + i) for i in range(2)]
    qs = [torch.randn((2, 12, 1, 128), generator=gen(60 + i), device=DEV).to(torch.bfloat16) for i in range(2)]
    ref = [kv4.kv4_decode(q, c.pool, c.table, c.device_lens) for q, c in zip(qs, caches)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        outs = []
        for s, q, c in zip(streams, qs, caches):
            with torch.cuda.stream(s):
                outs.append(kv4.kv4_decode(q, c.pool, c.table, c.device_lens))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, ref))


def test_graphs_captured_on_one_stream_do_not_share_a_workspace():
    from saga_b200 import kv4
    caches = [Cache([20000 + i, 300], 1, 2, 128, 128, seed=70 + i) for i in range(2)]
    qs = [torch.randn((2, 12, 1, 128), generator=gen(80 + i), device=DEV).to(torch.bfloat16) for i in range(2)]
    ref = [kv4.kv4_decode(q, c.pool, c.table, c.device_lens) for q, c in zip(qs, caches)]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, q, c in zip(graphs, qs, caches):
        with torch.cuda.graph(graph):
            outs.append(kv4.kv4_decode(q, c.pool, c.table, c.device_lens))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, ref):
            assert torch.equal(o, r)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------

def _args():
    c = Cache([100, 40], 1, 2, 64, 64, seed=70, bounds=True)
    q = torch.zeros((2, 4, 1, 64), dtype=torch.bfloat16, device=DEV)
    return c, q


@pytest.mark.parametrize("change,error", [
    (lambda a: a.update(query=a["query"].cpu()), "no CPU path"),
    (lambda a: a.update(query=a["query"][:, :, 0]), "query must be"),
    (lambda a: a.update(query=a["query"].expand(2, 4, 2, 64)), "query must be"),
    (lambda a: a.update(query=a["query"][..., :32]), "head_dim"),
    (lambda a: a.update(query=a["query"].transpose(1, 3).contiguous().transpose(1, 3)), "unit stride"),
    (lambda a: a.update(query=a["query"][:, :3]), "multiple of Hv"),
    (lambda a: a.update(query=a["query"].double()), "unsupported dtype"),
    (lambda a: a.update(lens=a["lens"].long()), "lens must be"),
    (lambda a: a.update(lens=a["lens"][:1]), "lens must have shape"),
    (lambda a: a.update(lens=a["lens"].cpu()), "no CPU path"),
    (lambda a: a.update(page_table=a["page_table"].long()), "page_table must be"),
    (lambda a: a.update(page_table=a["page_table"][:1]), "page_table must be"),
    (lambda a: a.update(page_table=a["page_table"].T.contiguous().T), "unit column stride"),
    (lambda a: a.update(page_table=a["page_table"][:, :0]), "max_pages"),
    (lambda a: a.update(starts=a["lens"].long()), "starts must be"),
    (lambda a: a.update(scaling=float("nan")), "scaling"),
    (lambda a: a.update(blocks=torch.zeros((2, 1, 3), dtype=torch.int32, device=DEV)), "go together"),
    (lambda a: a.update(blocks=torch.zeros((2, 2, 3), dtype=torch.int32, device=DEV),
                        counts=torch.zeros((2, 1), dtype=torch.int32, device=DEV)), "blocks must have shape"),
    (lambda a: a.update(blocks=torch.zeros((2, 1, 0), dtype=torch.int32, device=DEV),
                        counts=torch.zeros((2, 1), dtype=torch.int32, device=DEV)), "top must be positive"),
])
def test_decode_refuses(change, error):
    from saga_b200 import _lib, kv4
    c, q = _args()
    a = dict(query=q, pool=c.pool, page_table=c.table, lens=c.device_lens)
    kv4.kv4_decode(**a)
    change(a)
    with pytest.raises((ValueError, TypeError, _lib.SagaError), match=error):
        kv4.kv4_decode(**a)


def test_select_write_read_and_pool_refuse():
    from saga_b200 import _lib, kv4
    c, q = _args()
    errors = (ValueError, TypeError, _lib.SagaError)
    for kw, match in ((dict(top=0), "top"), (dict(top=1), "keep_first"), (dict(top=4, keep_last=0), "keep_last"),
                      (dict(top=4, keep_first=-1), "keep_first")):
        with pytest.raises(errors, match=match):
            kv4.kv4_select(q, c.pool, c.table, c.device_lens, **kw)
    plain = kv4.Kv4Pool(2, 64, 1, 2, 64, device=DEV)
    with pytest.raises(errors, match="bounds"):
        kv4.kv4_select(q, plain, c.table, c.device_lens, 4)
    k, v = torch.zeros((3, 1, 64), device=DEV), torch.zeros((3, 2, 64), device=DEV)
    slots = torch.arange(3, device=DEV)
    for args, match in (((k[:2], v, slots), "k must be"), ((k, v[:, :1], slots), "v must be"),
                        ((k, v.half(), slots), "share a dtype"), ((k, v, slots.int()), "slots must be"),
                        ((k.cpu(), v, slots), "no CPU path"), ((k, v, slots.cpu()), "no CPU path"),
                        ((k.double(), v.double(), slots), "unsupported dtype"),
                        ((k.transpose(0, 2).contiguous().transpose(0, 2), v, slots), "unit stride")):
        with pytest.raises(errors, match=match):
            kv4.kv4_write(plain, *args)
    with pytest.raises(errors, match="unsupported dtype"):
        kv4.kv4_read(plain, slots, dtype=torch.float64)
    with pytest.raises(errors, match="slots must be"):
        kv4.kv4_read(plain, slots.int())
    for args, match in (((2, 48, 1, 1, 64), "page_len"), ((2, 16, 1, 1, 64), "page_len"), ((2, 64, 1, 1, 96), "head_dim"),
                        ((0, 64, 1, 1, 64), "positive"), ((2, 64, 0, 1, 64), "positive")):
        with pytest.raises(errors, match=match):
            kv4.Kv4Pool(*args, device=DEV)


def test_tables_refuse():
    from saga_b200 import _lib, kv4
    i32 = dict(dtype=torch.int32, device=DEV)
    good = dict(page_table=torch.zeros((2, 4), **i32), lens=torch.zeros(2, **i32), new_lens=torch.ones(2, **i32),
                free_pages=torch.arange(8, **i32), free_state=torch.tensor([0, 8], **i32), num_tokens=2, page_len=64)
    kv4.page_tables(**good)
    for kw, match in ((dict(page_len=48), "page_len"), (dict(num_tokens=-1), "num_tokens"),
                      (dict(lens=good["lens"].long()), "lens"), (dict(new_lens=good["new_lens"][:1]), "new_lens"),
                      (dict(free_state=good["lens"][:1]), "free_state"), (dict(free_pages=good["free_pages"].long()),
                                                                          "free_pages"),
                      (dict(page_table=good["page_table"].cpu()), "no CPU path"),
                      (dict(lens_out=good["lens"].long()), "lens_out"),
                      (dict(page_table=good["page_table"][:1]), "page_table")):
        with pytest.raises((ValueError, TypeError, _lib.SagaError), match=match):
            kv4.page_tables(**{**good, **kw})
    with pytest.raises((ValueError, TypeError, _lib.SagaError), match="page_len"):
        kv4.slot_map(good["page_table"], good["lens"], 2, 33)
    with pytest.raises((ValueError, TypeError, _lib.SagaError), match="starts"):
        kv4.slot_map(good["page_table"], good["lens"], 2, 64, starts=good["lens"].long())


def test_compiled_step_matches_eager():
    """torch.compile traces a step through the custom ops without a graph break."""
    from saga_b200 import kv4
    B, hq, hk, hv, d, pl = 2, 8, 1, 2, 64, 32
    i32 = dict(dtype=torch.int32, device=DEV)
    g = gen(80)
    k, v = (torch.randn((B, h, d), generator=g, device=DEV).to(torch.bfloat16) for h in (hk, hv))
    q = torch.randn((B, hq, 1, d), generator=g, device=DEV).to(torch.bfloat16)
    results = []

    def run(pool, table, lens, ring, state):
        st = kv4.page_tables(table, lens, torch.ones_like(lens), ring, state, B, pl, lens_out=lens,
                             free_state_out=state)
        kv4.kv4_write(pool, k, v, st.slots)
        blocks, counts = kv4.kv4_select(q, pool, table, lens, 2)
        return (kv4.kv4_decode(q, pool, table, lens), kv4.kv4_decode(q, pool, table, lens, blocks=blocks, counts=counts),
                *kv4.kv4_read(pool, st.slots))

    for fn in (run, torch.compile(run, fullgraph=True)):
        c = Cache([100, 64], hk, hv, d, pl, seed=81, bounds=True, extra_pages=4)
        free = sorted(set(range(c.pool.num_pages)) - set(c.table[0, :4].tolist()) - set(c.table[1, :2].tolist()))
        ring, state = torch.tensor(free, **i32), torch.tensor([0, len(free)], **i32)
        outs = fn(c.pool, c.table, c.device_lens, ring, state)
        results.append([t.clone() for t in (*outs, c.table, c.device_lens, state, c.pool.k, c.pool.v)])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("top", [0, 6])
def test_serving_example(top):
    """The example's loop: lengths, pages and attention are right after admissions, steps and a finished
    request. With values of unit range in 15 steps, a rounding error of at most half a step on keys and values
    stays well below the signal; over all pages the outputs are close to the 16-bit ones."""
    from saga_b200.serve_kv4 import serve
    r = serve(requests=5, prompt=700, steps=40, top=top, page_len=32)
    assert r["lens"] == r["expected_lens"] and r["status"] == 0
    assert r["pages_held"] + r["pages_free"] == r["pages"]
    assert r["cache_bytes"] < 0.35 * r["cache_bytes_16bit"]  # 9/32 of it, and pages partly filled
    if not top:
        assert r["cosine_to_16bit"] > 0.97
