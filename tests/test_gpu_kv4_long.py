"""The decode kernel's loop over many tiles per warp: ring stages reused, page numbers fetched in further batches
of 32, the stabilisers raised over sums of earlier tiles. The loop is reached by many requests over the same
pages (a decode only reads), with a few different queries, whose results are compared one by one.
"""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O
from test_gpu_kv4 import DEV, DT, OUT_EPS, W_EPS, Cache, _status, f64, gen, slots_of  # noqa: F401

pytestmark = pytest.mark.gpu

N, PL = 20300, 128


def tiles_per_warp(requests, tiles):
    """Tiles of one item that a warp gets at least somewhere: a CTA's run then holds a whole item."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    run = -(-requests * (tiles + 16) // sms)
    assert run >= 2 * (tiles + 16)
    return tiles // 8


def rising(hq, hk, hv, d, dtype, seed):
    """A request of N positions whose keys grow along one direction, and queries that lie along it (scores rise by
    tens of powers of two), against it, anywhere, and close to zero."""
    from saga_b200 import kv4
    c = Cache([N], hk, hv, d, PL, dtype, seed=seed)
    u = torch.randn(d, generator=gen(seed), device=DEV)
    u /= u.norm()
    k = torch.randn((N, hk, d), generator=gen(seed + 1), device=DEV)
    k += (torch.arange(N, device=DEV) / N * 8)[:, None, None] * u
    v = torch.randn((N, hv, d), generator=gen(seed + 2), device=DEV)
    k, v = k.to(DT[dtype]), v.to(DT[dtype])
    kv4.kv4_write(c.pool, k, v, slots_of(c.table, 0, N, PL))
    c.k[0], c.v[0] = O.rows_value(k.float().cpu().numpy()), O.rows_value(v.float().cpu().numpy())
    q = torch.randn((4, hq, 1, d), generator=gen(seed + 3), device=DEV)
    q[0] += 6 * d ** 0.5 * u
    q[1] -= 6 * d ** 0.5 * u
    q[3] *= 1e-3
    return c, q.to(DT[dtype])


def check(q, out, c, d, dtype, allowed=None):
    """out [R, Hq, 1, D]: request r has query r % 4 and, with `allowed`, positions allowed[r % len(allowed)]."""
    out = f64(out)
    lists = allowed if allowed is not None else [np.ones((c.k[0].shape[1], N), bool)]
    for x in range(4):
        for y, ok in enumerate(lists):
            mine = [r for r in range(out.shape[0]) if r % 4 == x and r % len(lists) == y]
            if not mine:
                continue
            ref, tol = O.attention(f64(q[x, :, 0]), c.k[0], c.v[0], ok, d ** -0.5, W_EPS[dtype])
            tol = tol + OUT_EPS[dtype] * np.abs(ref) + 2.0 ** -25 * (dtype == "fp16")
            err = np.abs(out[mine, :, 0] - ref)
            assert (err <= tol).all(), f"query {x}, list {y}: {(err - tol).max():.3e} over"


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("heads,d", [((12, 1, 1), 128), ((12, 1, 4), 128), ((15, 1, 5), 64)], ids=str)
def test_many_tiles_per_warp(heads, d, dtype):
    from saga_b200 import kv4
    requests, (hq, hk, hv) = 300, heads
    c, q = rising(hq, hk, hv, d, dtype, seed=90)
    assert tiles_per_warp(requests, -(-N // 32)) > 64
    table = c.table.expand(requests, -1).contiguous()
    lens = torch.full((requests,), N, dtype=torch.int32, device=DEV)
    qs = q.repeat(requests // 4, 1, 1, 1)
    out = kv4.kv4_decode(qs, c.pool, table, lens)
    check(q, out, c, d, dtype)
    assert torch.equal(kv4.kv4_decode(qs, c.pool, table, lens), out)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_many_tiles_per_warp_from_block_lists(dtype):
    from saga_b200 import kv4
    requests, hq, hk, hv, d, top = 300, 12, 1, 2, 128, 140
    c, q = rising(hq, hk, hv, d, dtype, seed=95)
    assert tiles_per_warp(requests, top * PL // 32) > 64
    table = c.table.expand(requests, -1).contiguous()
    lens = torch.full((requests,), N, dtype=torch.int32, device=DEV)
    rng = np.random.default_rng(5)
    pages = -(-N // PL)
    lists = [np.sort(rng.permutation(pages)[:top]) for _ in range(3)]
    lists[1] = np.arange(top)
    allowed = []
    for x in lists:
        ok = np.zeros((1, pages * PL), bool)
        for p in x:
            ok[0, p * PL:(p + 1) * PL] = True
        allowed.append(ok[:, :N])
    blocks = torch.tensor(np.stack(lists), dtype=torch.int32, device=DEV).repeat(requests // 3, 1)[:, None].contiguous()
    counts = torch.full((requests, 1), top, dtype=torch.int32, device=DEV)
    out = kv4.kv4_decode(q.repeat(requests // 4, 1, 1, 1), c.pool, table, lens, blocks=blocks, counts=counts)
    check(q, out, c, d, dtype, allowed)
