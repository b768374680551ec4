"""Plain 64-bit forms of the 4-bit paged cache operators (test infrastructure).

Restates the definitions in include/saga_b200.h with numpy: the quantiser with
its binary32 steps, attention in float64, the block scores in binary32 by
halves, and the page tables one request at a time.
"""
import numpy as np

GROUP = 64
F32 = np.float32


def bf16_towards(x, up):
    """bfloat16 neighbour of x (float32 array) at or below it, or at or above it."""
    x = np.asarray(x, dtype=F32)
    if up:
        return -bf16_towards(-x, False)
    t = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(F32)
    below = ((t.view(np.uint32) + np.uint32(0x10000))).view(F32)
    return np.where(t > x, below, t).astype(F32)


def quantise(x):
    """(codes, s, z) of rows [..., D]; a group that is not finite has s = z = NaN and code 0."""
    x = np.asarray(x, dtype=F32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(g).all(-1)
        safe = np.where(bad[..., None], F32(0), g)
        z = bf16_towards(safe.min(-1), False)
        s = (safe.max(-1) - z).astype(F32) * (F32(1) / F32(15))
        s = bf16_towards(np.maximum(s.astype(F32), F32(2.0 ** -40)), True)
        bad |= ~np.isfinite(z) | ~np.isfinite(s)
        r = (F32(1) / s).astype(F32)
        c = np.rint(((safe - z[..., None]).astype(F32) * r[..., None]).astype(F32))
    c = np.where(bad[..., None], 0, np.clip(c, 0, 15)).astype(np.int64)
    nan = F32("nan")
    return c, np.where(bad, nan, s).astype(F32), np.where(bad, nan, z).astype(F32)


def stands_for(c, s, z):
    """The values of codes, float64 (they are exact there)."""
    return (c * s[..., None].astype(np.float64) + z[..., None].astype(np.float64)).reshape(
        *c.shape[:-2], c.shape[-2] * GROUP)


def rows_value(x):
    """What rows [..., D] stand for once written, float64."""
    return stands_for(*quantise(x))


def page_bounds(values):
    """(lo, hi) per channel of a page's key values [page_len, D] (NaN values left out; NaN where all are),
    bfloat16 values."""
    v = np.asarray(values).astype(F32)
    none = np.isnan(v).all(0)
    lo = np.where(np.isnan(v), F32(np.inf), v).min(0)
    hi = np.where(np.isnan(v), F32(-np.inf), v).max(0)
    return tuple(np.where(none, F32("nan"), b) for b in (bf16_towards(np.where(none, 0, lo), False),
                                                         bf16_towards(np.where(none, 0, hi), True)))


def block_score(q, lo, hi):
    """Score of one page for the queries [G, D] of a key head, binary32 by halves; NaN if any is."""
    q, lo, hi = (np.asarray(t, dtype=F32) for t in (q, lo, hi))
    x = (q * np.where(q > 0, hi, lo)).astype(F32)
    while x.shape[-1] > 1:
        h = x.shape[-1] // 2
        x = (x[..., :h] + x[..., h:]).astype(F32)
    return x[:, 0].max() if not np.isnan(x).any() else F32("nan")


def select(q, lo, hi, n, page_len, top, keep_first=1, keep_last=1):
    """Blocks (list) of one request and key head. lo, hi: [complete pages, D]."""
    pages = -(-n // page_len)
    if pages <= top:
        return list(range(pages))
    kept = [p for p in range(pages) if p < keep_first or p >= pages - keep_last]
    rest = [p for p in range(pages) if keep_first <= p < pages - keep_last]
    score = {p: block_score(q, lo[p], hi[p]) for p in rest}
    rest.sort(key=lambda p: (0, -float(score[p]), p) if score[p] == score[p] else (1, 0.0, p))
    return sorted(kept + rest[:top - len(kept)])


def attention(q, k, v, allowed, scaling, w_eps):
    """Attention of one request in float64. q [Hq, D]; k [n, Hk, D], v [n, Hv, D] values that the cache
    stands for; allowed [Hk, n] bool. Returns (out [Hq, D], tolerance [Hq, D]).

    The tolerance has the weights' relative error: w_eps for their rounding, and 2^-18 of the sum of
    |q k| for the scores (binary32 sums of up to 128 products of about 24 bits, with the scales'
    products; 2^-18 leaves a factor of 8). A weight multiplies a value about the middle of its
    group's range, at most half the range from it: at most the greatest |v| for values on both sides
    of zero, and at most twice it always; and a group's range is at least 15 * 2^-40, the least scale.
    """
    hq, d = q.shape
    hk, hv = k.shape[1], v.shape[1]
    out, tol = np.zeros((hq, d)), np.zeros((hq, d))
    q = q.astype(np.float64)
    for h in range(hq):
        ok = allowed[h // (hq // hk)]
        if not ok.any():
            continue
        kk, vv = k[ok, h // (hq // hk)], v[ok, h // (hq // hv)]
        with np.errstate(all="ignore"):
            w = kk @ q[h] * scaling
            size = (np.abs(kk) @ np.abs(q[h])).max() * abs(scaling)
            p = np.exp(w - w.max())
            p /= p.sum()
            out[h] = p @ vv
            tol[h] = (w_eps + 2.0 ** -18 * size) * (2 * (p @ np.abs(vv).max(-1)) + 15 * 2.0 ** -40) + 2.0 ** -24 * np.abs(vv).max()
    return out, tol


def page_tables(table, lens, new, ring, first, count, num_tokens, page_len):
    """One step of the block tables, request by request. Arguments are lists (changed in place: table,
    ring). Returns slots, positions, offsets, lens, (first, count), failed."""
    lens = list(lens)
    width, size = len(table[0]) if table else 0, len(ring)
    slots, positions, offsets = [-1] * num_tokens, [0] * num_tokens, [0]
    wanted = taken = 0
    failed = False
    for b, (n, m) in enumerate(zip(lens, new)):
        m = max(m, 0)
        start = offsets[-1]
        offsets.append(start + m)
        if n + m > width * page_len or start + m > num_tokens:
            failed |= m > 0
            continue
        held = -(-n // page_len)
        need = -(-(n + m) // page_len) - held
        wanted += need
        if need and wanted > count:
            failed = True
            continue
        for j in range(need):
            table[b][held + j] = ring[(first + wanted - need + j) % size]
        taken += need
        for j in range(m):
            positions[start + j] = n + j
            slots[start + j] = table[b][(n + j) // page_len] * page_len + (n + j) % page_len
        lens[b] = n + m
    back = 0
    for b, m in enumerate(new):
        if m < 0:
            for j in range(-(-lens[b] // page_len)):
                ring[(first + count + back) % size] = table[b][j]
                back += 1
            lens[b] = 0
    state = ((first + taken) % size if size else 0, count - taken + back)
    return slots, positions, offsets, lens, state, failed
