"""What is measured of the 4-bit paged cache operators, and what they have to compute.

Four operators serve a decode loop whose keys and values are held in 4 bits, in pages:

``tables``  block tables and slot maps from the requests' lengths: every request's new tokens get
            pages from a free list, a slot (page * page_len + offset) and a position.
``write``   one step's key and value rows are quantised into the slots of the pages, the bounds of
            the key pages that the step fills are taken, and the rows are read back as the values
            that the cache now stands for.
``decode``  attention of one query position per request over its own length of the cache.
``sparse``  the same over a few blocks (pages) per request and key head, selected for the query by
            a score that reads only the pages' key bounds.

The cache. A row (one token, one head) is cut into groups of 64 values. With all steps in binary32:
lo, hi = the group's least and greatest value; z = lo rounded down to bfloat16; s = (hi - z) *
(1/15), at least 2**-40, rounded up to bfloat16; r = 1 / s; code = (x - z) * r rounded to the nearest (ties to
even), within 0..15. The group stands for s * code + z.

Block scores. A complete page keeps, per key head and channel, the least and the greatest value that
its keys stand for, rounded outwards to bfloat16. Its score for a key head is the greatest, over the
head's queries, of the sum over the channels of q * (greatest where q > 0, else least): an upper bound
of the page's scores. The sum is taken in binary32 by halves (channel d with channel d + D/2, then
d + D/4, and so on), so that a selection is the same wherever it is computed. The first page and the
last are always kept; ties go to the lowest page; the selected pages are listed in ascending order.
"""
import math
import random

import torch

own = False

GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------

def listed():
    return [
        # the tables of one decode step of 64 running requests: one launch's latency is all there is
        dict(name="tables_decode_64", op="tables", requests=64, kind="decode", context=65600, tokens=64, page_len=128),
        # a scheduler's mixed step: prompt chunks, single tokens, idle and finished requests
        dict(name="tables_mixed_512", op="tables", requests=512, kind="mixed", context=16512, tokens=65536,
             page_len=64),
        # the decode tokens of 64 sequences, the 12/1/4-head layer: latency again
        dict(name="write_decode_64", op="write", tokens=64, key_heads=1, value_heads=4, head_dim=128, page_len=128,
             dtype="bf16"),
        # a packed prompt of several requests, an odd number of rows, the 15/1/5-head layer at head_dim 64
        dict(name="write_prompt_64", op="write", tokens=16511, key_heads=1, value_heads=5, head_dim=64, page_len=64,
             dtype="fp16"),
        # a long prompt of the 12/1/4-head layer
        dict(name="write_prompt_long", op="write", tokens=131072, key_heads=1, value_heads=4, head_dim=128,
             page_len=128, dtype="bf16"),
        # one chat request with a short history: launch latency
        dict(name="decode_single", op="decode", batch=1, context=1021, ragged=False, query_heads=12, key_heads=1,
             value_heads=2, head_dim=128, page_len=128, dtype="bf16"),
        # eight equal 32K contexts of the 12/1/2-head layer
        dict(name="decode_32k", op="decode", batch=8, context=32768, ragged=False, query_heads=12, key_heads=1,
             value_heads=2, head_dim=128, page_len=128, dtype="bf16"),
        # sixteen ragged contexts at head_dim 64, five value heads
        dict(name="decode_ragged_64", op="decode", batch=16, context=16512, ragged=True, query_heads=15, key_heads=1,
             value_heads=5, head_dim=64, page_len=64, dtype="fp16"),
        # an unmerged model in 32 bits, as many key heads as value heads
        dict(name="decode_fp32", op="decode", batch=4, context=4099, ragged=True, query_heads=16, key_heads=4,
             value_heads=4, head_dim=128, page_len=256, dtype="fp32"),
        # the largest: 64 long contexts of the 12/1/4-head layer
        dict(name="decode_64x64k", op="decode", batch=64, context=65600, ragged=False, query_heads=12, key_heads=1,
             value_heads=4, head_dim=128, page_len=128, dtype="bf16"),
        # one very long document, 64 of its 1024 blocks
        dict(name="sparse_128k", op="sparse", batch=1, context=131072, ragged=False, query_heads=12, key_heads=1,
             value_heads=2, head_dim=128, page_len=128, dtype="bf16", top=64),
        # a batch of ragged long contexts, small blocks
        dict(name="sparse_64x64k", op="sparse", batch=64, context=65600, ragged=True, query_heads=12, key_heads=1,
             value_heads=4, head_dim=128, page_len=64, dtype="bf16", top=48),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("tables", "write", "decode", "decode", "sparse", "sparse"))
    if op == "tables":
        requests = _log_int(rng, 1, 1024)
        kind = rng.choice(("decode", "mixed"))
        return dict(op=op, requests=requests, kind=kind, context=_log_int(rng, 16, 65600),
                    tokens=requests if kind == "decode" else _log_int(rng, requests, 131072),
                    page_len=rng.choice((32, 64, 128, 256)))
    heads = rng.choice(((12, 1, 2), (12, 1, 4), (15, 1, 5), (12, 2, 2), (8, 2, 4), (16, 4, 4), (6, 2, 1), (24, 1, 3)))
    head_dim = rng.choice((64, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    page_len = rng.choice((32, 64, 128, 256))
    if op == "write":
        return dict(op=op, tokens=_log_int(rng, 1, 131072), key_heads=heads[1], value_heads=heads[2],
                    head_dim=head_dim, page_len=page_len, dtype=dtype)
    context = _log_int(rng, 1, 131072)
    row = (heads[1] + heads[2]) * head_dim
    most = 64 * 65600 * 5 * 128 // 4                       # a quarter of the largest listed cache
    batch = _log_int(rng, 1, max(1, min(128, most // (context * row))))
    case = dict(op=op, batch=batch, context=context, ragged=rng.random() < 0.7, query_heads=heads[0],
                key_heads=heads[1], value_heads=heads[2], head_dim=head_dim, page_len=page_len, dtype=dtype)
    if op == "sparse":
        case["top"] = _log_int(rng, 2, 128)
    return case


def _lengths(case):
    """The cached tokens of each request: all `context`, or ragged with `context` the longest."""
    if not case["ragged"]:
        return [case["context"]] * case["batch"]
    rng = random.Random(f"{case['batch']}:{case['context']}")
    return [case["context"]] + [_log_int(rng, max(1, case["context"] // 16), case["context"])
                                for _ in range(case["batch"] - 1)]


def work(case):
    op = case["op"]
    if op == "tables":
        t, b = case["tokens"], case["requests"]
        pages = t // case["page_len"] + b
        return {"bytes": t * (8 + 4) + b * 4 * 5 + pages * 8, "flops": t}
    esz = 4 if case["dtype"] == "fp32" else 2
    d = case["head_dim"]
    packed = d // 2 + d // GROUP * 4
    if op == "write":
        rows = case["tokens"] * (case["key_heads"] + case["value_heads"])
        bounds = case["tokens"] // case["page_len"] * case["key_heads"] * d * 2 * 2
        return {"bytes": rows * 2 * (d * esz + packed) + case["tokens"] * 8 + bounds, "flops": rows * d * 8}
    lens = _lengths(case)
    qo = 2 * case["batch"] * case["query_heads"] * d * esz
    if op == "sparse":
        pl = case["page_len"]
        scored = sum(n // pl for n in lens if (n + pl - 1) // pl > case["top"])
        read = sum(min(n, case["top"] * pl) for n in lens)
        return {"bytes": scored * case["key_heads"] * d * 4 + read * (case["key_heads"] + case["value_heads"]) * packed
                + qo, "flops": scored * case["query_heads"] * d * 2 + read * case["query_heads"] * d * 4}
    read = sum(lens)
    return {"bytes": read * (case["key_heads"] + case["value_heads"]) * packed + qo,
            "flops": read * case["query_heads"] * d * 4}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------

def _tables_inputs(case, seed):
    """Lengths, this step's token counts, a page table with the pages that the lengths already hold,
    and the free list's ring (pages in a shuffled order; first entry and number of entries)."""
    rng = random.Random(seed)
    b, pl = case["requests"], case["page_len"]
    lens = [rng.randint(0, case["context"]) for _ in range(b)]
    if case["kind"] == "decode":
        new = [1] * b
    else:
        # a few requests take most of the step's tokens as prompt chunks; some idle, some are finished (-1)
        left = case["tokens"] - rng.randint(0, case["tokens"] // 50)
        new = []
        for i in range(b):
            kind = rng.random()
            n = 1 if kind < 0.5 else 0 if kind < 0.6 else -1 if kind < 0.7 else rng.randint(1, max(1, 6 * case["tokens"] // b))
            n = min(n, left)
            left -= max(n, 0)
            new.append(n)
        rng.shuffle(new)
    most = max(1, 6 * case["tokens"] // b)                   # sizes go by the case, not by the seed
    width = (case["context"] + most + pl - 1) // pl + 1
    held = [(n + pl - 1) // pl for n in lens]
    total = b * ((case["context"] + pl - 1) // pl) + case["tokens"] // pl + b + 7
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((b, width), -1, dtype=torch.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = perm[at:at + h]
        at += h
    # the ring holds the remaining pages, from a place near its end so that it wraps around
    ring = torch.full((total,), -1, dtype=torch.int32)
    first, count = total - 3, total - at
    ring[(first + torch.arange(count)) % total] = perm[at:]
    return lens, new, table, ring, first, count


def _write_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t, d, pl = case["tokens"], case["head_dim"], case["page_len"]
    dt = DTYPES[case["dtype"]]
    channel = 1.0 + 2.0 * torch.rand((1, case["key_heads"], d), generator=g, device=DEV)
    k = (torch.randn((t, case["key_heads"], d), generator=g, device=DEV) * channel).to(dt)
    v = (torch.randn((t, case["value_heads"], d), generator=g, device=DEV) * 0.5).to(dt)
    rng = random.Random(seed)
    if t <= 256:                                            # a decode step: one token for each of t requests
        order = rng.sample(range(t), t)
        slots, pages = [p * pl + rng.randrange(pl) for p in order], t
        return k, v, torch.tensor(slots, dtype=torch.int64, device=DEV), pages
    # a prompt: requests of a few hundred tokens in pages of a shuffled order, some padding rows (-1) at the end
    pages = t // pl + t // 200 + 2
    order = rng.sample(range(pages), pages)
    real = t - rng.randint(0, t // 64)
    slots, at = [], 0
    while len(slots) < real:
        n = min(rng.randint(1, 400), real - len(slots), (pages - at) * pl)
        if n == 0:
            break
        slots += [order[at + i // pl] * pl + i % pl for i in range(n)]
        at += (n + pl - 1) // pl
    slots += [-1] * (t - len(slots))
    return k, v, torch.tensor(slots, dtype=torch.int64, device=DEV), pages


def _cache_shape(case):
    pl = case["page_len"]
    lens = _lengths(case)
    per = [(n + pl - 1) // pl for n in lens]
    return lens, per, sum(per)


def _attention_inputs(case, seed):
    """Query, the order of the pages, and a maker of each request's key and value rows [len, H, D]. A few
    keys of every request lie along a query head, so that its attention has peaks."""
    b, d, hq, hk, hv = (case[x] for x in ("batch", "head_dim", "query_heads", "key_heads", "value_heads"))
    dt = DTYPES[case["dtype"]]
    lens, per, total = _cache_shape(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn((b, hq, 1, d), generator=g, device=DEV).to(dt)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros((b, max(per)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n]
        at += n
    shuffled = list(range(b))
    random.Random(seed).shuffle(shuffled)
    lens = [lens[i] for i in shuffled]
    table = table[shuffled]

    def rows(i):
        gi = torch.Generator(device=DEV).manual_seed(seed * 1000003 + i + 1)
        n = lens[i]
        k = torch.randn((n, hk, d), generator=gi, device=DEV)
        v = torch.randn((n, hv, d), generator=gi, device=DEV) * 0.5
        for h in range(hk):
            at_ = torch.randint(0, n, (max(1, n // 512),), generator=gi, device=DEV)
            qh = q[i, h * (hq // hk), 0].float()
            k[at_, h] = k[at_, h] + 4.0 * qh / qh.norm()
        return k.to(dt), v.to(dt)

    return q, lens, table.to(DEV), total, rows


def _slots_of(table_row, n, pl):
    pos = torch.arange(n, device=DEV)
    return table_row[pos // pl].long() * pl + pos % pl


# ------------------------------------------------------------------------------------------------
# the plain form
# ------------------------------------------------------------------------------------------------

def _bf16_down(x):
    t = (x.view(torch.int32) & -65536).view(torch.float32)
    return torch.where(t > x, (t.view(torch.int32) + 65536).view(torch.float32), t)


def _bf16_up(x):
    return -_bf16_down(-x)


def _quantise(x):
    """Codes [..., D] (uint8), scales and zeros [..., D/64] (float32 with bfloat16 values)."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    z = _bf16_down(lo)
    s = _bf16_up(((hi - z) * (1.0 / 15.0)).clamp_min(2.0 ** -40))
    c = torch.round((g - z[..., None]) * (1.0 / s)[..., None]).clamp(0, 15)
    return c.flatten(-2).to(torch.uint8), s, z


def _stands_for(c, s, z):
    return (c.unflatten(-1, (-1, GROUP)).float() * s[..., None] + z[..., None]).flatten(-2)


class _PlainPool:
    def __init__(self, pages, page_len, hk, hv, d, bounds):
        self.page_len = page_len
        self.d = d
        self.k, self.v = ([torch.zeros((pages * page_len, h, d), dtype=torch.uint8, device=DEV),
                           torch.zeros((pages * page_len, h, d // GROUP), device=DEV),
                           torch.zeros((pages * page_len, h, d // GROUP), device=DEV)] for h in (hk, hv))
        self.k_lo = self.k_hi = None
        if bounds:
            self.k_lo, self.k_hi = (torch.zeros((pages, hk, d), dtype=torch.bfloat16, device=DEV) for _ in range(2))

    def write(self, k, v, slots):
        keep = slots >= 0
        at = slots[keep]
        for pool, x in ((self.k, k), (self.v, v)):
            for part, y in zip(pool, _quantise(x[keep])):
                part[at] = y
        if self.k_lo is not None:
            full = at[at % self.page_len == self.page_len - 1] // self.page_len
            for some in full.split(4096):
                idx = (some[:, None] * self.page_len + torch.arange(self.page_len, device=DEV)).flatten()
                x = _stands_for(*(part[idx] for part in self.k)).unflatten(0, (-1, self.page_len))
                self.k_lo[some] = _bf16_down(x.amin(1)).to(torch.bfloat16)
                self.k_hi[some] = _bf16_up(x.amax(1)).to(torch.bfloat16)

    def read(self, slots):
        at = slots.clamp_min(0)
        keep = (slots >= 0)[:, None, None]
        return tuple(torch.where(keep, _stands_for(*(part[at] for part in pool)), 0.0) for pool in (self.k, self.v))


def _plain_tables(st):
    table, lens, new, ring, state = st["table"], st["lens"], st["new"], st["ring"], st["state"]
    pl, tokens = st["page_len"], st["tokens"]
    b, width = table.shape
    add = new.clamp_min(0)
    end = lens + add
    cu = torch.zeros(b + 1, dtype=torch.int64, device=DEV)
    cu[1:] = add.cumsum(0)
    held = (lens + pl - 1) // pl
    fits = (end <= width * pl) & (cu[1:] <= tokens)
    need = torch.where(fits, (end + pl - 1) // pl - held, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= state[1]))
    taken = torch.where(granted, need, 0)
    # new pages into the table
    nth = torch.arange(width, device=DEV) - held[:, None]
    page = ring[(state[0] + (upto - need)[:, None] + nth) % ring.numel()]
    table.copy_(torch.where((nth >= 0) & (nth < taken[:, None]), page, table))
    # the tokens' slots and positions
    tok = torch.arange(tokens, device=DEV)
    req = torch.searchsorted(cu[1:].contiguous(), tok, right=True)
    real = req < b
    req = req.clamp_max(b - 1)
    real = real & granted[req]
    pos = torch.where(real, lens[req] + tok - cu[req], 0)
    slots = torch.where(real, table[req, pos // pl].long() * pl + pos % pl, -1)
    # finished requests return their pages to the ring's end
    done = new < 0
    back = torch.where(done, held, 0)
    nth = torch.arange(width, device=DEV).expand(b, width)
    at = (state[0] + state[1] + (back.cumsum(0) - back)[:, None] + nth) % ring.numel()
    longer = torch.cat((ring, ring[:1]))                                  # its last entry takes what is not returned
    longer[torch.where(nth < back[:, None], at, ring.numel())] = table
    ring.copy_(longer[:-1])
    return dict(slots=slots, positions=pos.to(torch.int32), offsets=cu.to(torch.int32),
                lens=torch.where(done, 0, torch.where(granted, end, lens)).to(torch.int32),
                free_state=torch.stack(((state[0] + taken.sum()) % ring.numel(),
                                        state[1] - taken.sum() + back.sum())).to(torch.int32),
                page_table=table, free_pages=ring)


def _head_softmax(w, mask):
    w = torch.where(mask, w, -float("inf"))
    p = torch.exp(w - w.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_select(q, pool, table, lens, top):
    """Blocks [B, Hk, top] (ascending, -1 beyond the count) and counts [B, Hk]."""
    b, hq, _, d = q.shape
    hk = pool.k_lo.shape[1]
    nth = torch.arange(table.shape[1], device=DEV)
    pages = (lens[:, None] + pool.page_len - 1) // pool.page_len
    lo, hi = (x[table.long()].float().transpose(1, 2)[:, :, None] for x in (pool.k_lo, pool.k_hi))   # [B, Hk, 1, W, D]
    qs = q.reshape(b, hk, hq // hk, 1, d)
    x = qs * torch.where(qs > 0, hi, lo)
    while x.shape[-1] > 1:
        half = x.shape[-1] // 2
        x = x[..., :half] + x[..., half:]
    score = x[..., 0].amax(2)                                              # [B, Hk, W]
    kept = ((nth == 0) | (nth == pages - 1))[:, None]
    real = (nth < pages)[:, None]
    score = torch.where(kept, float("inf"), torch.where(real, score, -float("inf")))
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    best = torch.where(best < pages[:, None], best, table.shape[1]).sort(-1).values
    best = torch.where(best < table.shape[1], best, -1).to(torch.int32)
    blocks = torch.cat((best, best.new_full((b, hk, top - best.shape[-1]), -1)), -1)
    return blocks, pages.clamp_max(top).to(torch.int32).expand(b, hk)


def _plain_decode(q, pool, table, lens):
    b, hq, _, d = q.shape
    pl = pool.page_len
    pos = torch.arange(table.shape[1] * pl, device=DEV)
    slots = torch.where(pos < lens[:, None], table.long()[:, pos // pl] * pl + pos % pl, -1)
    k, v = pool.read(slots.flatten())
    k, v = (x.unflatten(0, slots.shape).transpose(1, 2) for x in (k, v))   # [B, H, n, D]
    w = torch.matmul(q.reshape(b, k.shape[1], -1, d), k.transpose(2, 3)).reshape(b, hq, -1) * (1.0 / math.sqrt(d))
    p = _head_softmax(w, (pos < lens[:, None])[:, None])
    return torch.matmul(p.reshape(b, v.shape[1], -1, p.shape[-1]), v).reshape(q.shape)


def _plain_sparse(q, pool, table, lens, top):
    b, hq, _, d = q.shape
    pl, hk = pool.page_len, pool.k_lo.shape[1]
    blocks, counts = _plain_select(q, pool, table, lens, top)
    pos = torch.where(blocks[..., None] >= 0, blocks[..., None] * pl + torch.arange(pl, device=DEV), 1 << 30).flatten(2)
    mask = pos < lens[:, None, None]                                       # [B, Hk, n]
    page = torch.gather(table[:, None].expand(b, hk, -1), 2, torch.where(mask, pos // pl, 0)).long()
    k, v = pool.read(torch.where(mask, page * pl + pos % pl, -1).flatten())
    k, v = (x.unflatten(0, mask.shape) for x in (k, v))                    # [B, Hk, n, H, D]
    head = torch.arange(hq, device=DEV)
    kh, vh = head // (hq // hk), head // (hq // v.shape[3])
    k, v = k[:, kh, :, kh].transpose(0, 1), v[:, kh, :, vh].transpose(0, 1)    # [B, Hq, n, D]
    w = torch.matmul(q, k.transpose(2, 3))[:, :, 0] * (1.0 / math.sqrt(d))
    return torch.matmul(_head_softmax(w, mask[:, kh])[:, :, None], v), blocks, counts


def _plain_run(st):
    op = st["op"]
    if op == "tables":
        return _plain_tables(st)
    pool = st["pool"]
    if op == "write":
        pool.write(st["k"], st["v"], st["slots"])
        k, v = pool.read(st["slots"])
        return dict(k=k.to(st["k"].dtype), v=v.to(st["v"].dtype), k_lo=pool.k_lo, k_hi=pool.k_hi)
    if op == "decode":
        return dict(out=_plain_decode(st["q"].float(), pool, st["table"], st["lens"]).to(st["q"].dtype))
    out, blocks, counts = _plain_sparse(st["q"].float(), pool, st["table"], st["lens"], st["top"])
    return dict(out=out.to(st["q"].dtype), blocks=blocks, counts=counts)


# ------------------------------------------------------------------------------------------------
# prepare and run
# ------------------------------------------------------------------------------------------------

def prepare(case, seed):
    op = case["op"]
    if op == "tables":
        lens, new, table, ring, first, count = _tables_inputs(case, seed)
        wide = torch.int32 if own else torch.int64
        return dict(op=op, page_len=case["page_len"], tokens=case["tokens"], table=table.to(DEV),
                    lens=torch.tensor(lens, dtype=wide, device=DEV), new=torch.tensor(new, dtype=wide, device=DEV),
                    ring=ring.to(DEV), state=torch.tensor([first, count], dtype=wide, device=DEV))
    pl, d, hk, hv = case["page_len"], case["head_dim"], case["key_heads"], case["value_heads"]

    # The pool is the handle that a serving program keeps: its bytes are laid out as each side likes.
    def pool_of(pages, bounds):
        if own:
            from saga_b200 import kv4
            return kv4.Kv4Pool(pages, pl, hk, hv, d, device=DEV, bounds=bounds)
        return _PlainPool(pages, pl, hk, hv, d, bounds)

    def write(pool, k, v, slots):
        if own:
            from saga_b200 import kv4
            kv4.kv4_write(pool, k, v, slots)
        else:
            for some in torch.arange(slots.numel(), device=DEV).split(16384):
                pool.write(k[some], v[some], slots[some])

    if op == "write":
        k, v, slots, pages = _write_inputs(case, seed)
        return dict(op=op, k=k, v=v, slots=slots, pool=pool_of(pages, True))
    q, lens, table, pages, rows = _attention_inputs(case, seed)
    pool = pool_of(pages, op == "sparse")
    for i, n in enumerate(lens):
        k, v = rows(i)
        write(pool, k, v, _slots_of(table[i], n, pl))
    return dict(op=op, q=q, pool=pool, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                top=case.get("top"))


def run(state):
    if not own:
        return _plain_run(state)
    from saga_b200 import kv4
    op = state["op"]
    if op == "tables":
        t = kv4.page_tables(state["table"], state["lens"], state["new"], state["ring"], state["state"],
                            state["tokens"], state["page_len"])
        return dict(slots=t.slots, positions=t.positions, offsets=t.offsets, lens=t.lens, free_state=t.free_state,
                    page_table=state["table"], free_pages=state["ring"])
    pool = state["pool"]
    if op == "write":
        kv4.kv4_write(pool, state["k"], state["v"], state["slots"])
        k, v = kv4.kv4_read(pool, state["slots"], dtype=state["k"].dtype)
        return dict(k=k, v=v, k_lo=pool.k_lo, k_hi=pool.k_hi)
    if op == "decode":
        return dict(out=kv4.kv4_decode(state["q"], pool, state["table"], state["lens"]))
    blocks, counts = kv4.kv4_select(state["q"], pool, state["table"], state["lens"], state["top"])
    out = kv4.kv4_decode(state["q"], pool, state["table"], state["lens"], blocks=blocks, counts=counts)
    return dict(out=out, blocks=blocks, counts=counts)


# ------------------------------------------------------------------------------------------------
# from the definition, in 64 bits
# ------------------------------------------------------------------------------------------------

def _r32(x):
    """A float64 tensor rounded to binary32 (held in float64)."""
    return x.to(torch.float32).to(torch.float64)


def _towards(x, up):
    """bfloat16 neighbour of x at or below it (above it): 8 significant bits."""
    m, e = torch.frexp(x)
    m = m * 256.0
    return torch.ldexp((torch.ceil(m) if up else torch.floor(m)) / 256.0, e)


def _exact_rows(x):
    """What the cache stands for after these rows [..., D] are written, in 64 bits."""
    y = x.double().reshape(*x.shape[:-1], -1, GROUP)
    z = _towards(y.min(-1).values, False)
    fifteenth = _r32(torch.tensor(1.0, dtype=torch.float64) / 15.0).item()
    s = _r32(_r32(y.max(-1).values - z) * fifteenth)
    s = _towards(torch.maximum(s, torch.tensor(2.0 ** -40, dtype=torch.float64, device=s.device)), True)
    r = _r32(1.0 / s)
    code = torch.round(_r32(_r32(y - z[..., None]) * r[..., None]))
    code = torch.clamp(code, 0.0, 15.0)
    return (s[..., None] * code + z[..., None]).reshape(x.shape)


def _exact_tables(case, seed):
    lens, new, table, ring, first, count = _tables_inputs(case, seed)
    pl, tokens = case["page_len"], case["tokens"]
    table, ring = table.tolist(), ring.tolist()
    width, size = len(table[0]), len(ring)
    slots, positions, offsets = [-1] * tokens, [0] * tokens, [0]
    wanted = taken = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        m = max(m, 0)
        start = offsets[-1]
        offsets.append(start + m)
        if n + m > width * pl or start + m > tokens:
            continue
        held = -(-n // pl)
        need = -(-(n + m) // pl) - held
        wanted += need
        if need and wanted > count:
            continue
        for j in range(need):
            table[i][held + j] = ring[(first + wanted - need + j) % size]
        taken += need
        for j in range(m):
            positions[start + j] = n + j
            slots[start + j] = table[i][(n + j) // pl] * pl + (n + j) % pl
        lens[i] = n + m
    end = first + count
    back = 0
    for i, m in enumerate(new):
        if m < 0:
            for j in range(-(-lens[i] // pl)):
                ring[(end + back) % size] = table[i][j]
                back += 1
            lens[i] = 0
    i32 = dict(dtype=torch.int32)
    return dict(slots=torch.tensor(slots), positions=torch.tensor(positions, **i32),
                offsets=torch.tensor(offsets, **i32), lens=torch.tensor(lens, **i32),
                free_state=torch.tensor([(first + taken) % size, count - taken + back], **i32),
                page_table=torch.tensor(table, **i32), free_pages=torch.tensor(ring, **i32))


def exact(case, seed):
    op, pl = case["op"], case.get("page_len")
    if op == "tables":
        return _exact_tables(case, seed)
    if op == "write":
        k, v, slots, pages = _write_inputs(case, seed)
        real = slots >= 0
        k, v = (torch.where(real[:, None, None], _exact_rows(x), 0.0) for x in (k, v))
        lo, hi = (torch.zeros((pages, case["key_heads"], case["head_dim"]), dtype=torch.float64, device=DEV)
                  for _ in range(2))
        held = torch.zeros((pages * pl, case["key_heads"], case["head_dim"]), dtype=torch.float64, device=DEV)
        held[slots[real]] = k[real]
        full = slots[real & (slots % pl == pl - 1)] // pl      # the pages whose last slot was written
        held = _r32(held.reshape(pages, pl, case["key_heads"], case["head_dim"])[full])
        lo[full] = _towards(held.min(1).values, False) if len(full) else lo[full]
        hi[full] = _towards(held.max(1).values, True) if len(full) else hi[full]
        return dict(k=k, v=v, k_lo=lo, k_hi=hi)
    q, lens, _, _, rows = _attention_inputs(case, seed)
    hq, hk, hv, d = (case[x] for x in ("query_heads", "key_heads", "value_heads", "head_dim"))
    q = q.double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    all_blocks, all_counts = [], []
    for i, n in enumerate(lens):
        k, v = (_exact_rows(x) for x in rows(i))
        logit = torch.stack([k[:, h // (hq // hk)] @ q[i, h, 0] for h in range(hq)]) / math.sqrt(d)
        if op == "sparse":
            top, full, pages = case["top"], n // pl, -(-n // pl)
            allowed = torch.zeros((hk, pages), dtype=torch.bool, device=DEV)
            if pages <= top:
                allowed[:] = True
            else:
                kp = _r32(k[:full * pl]).reshape(full, pl, hk, d)
                lo, hi = _towards(kp.min(1).values, False), _towards(kp.max(1).values, True)
                for h in range(hk):
                    best = torch.full((full,), -float("inf"), dtype=torch.float64, device=DEV)
                    for j in range(h * (hq // hk), (h + 1) * (hq // hk)):
                        part = _r32(torch.where(q[i, j, 0] > 0, hi[:, h], lo[:, h]) * q[i, j, 0])
                        width = d
                        while width > 1:
                            width //= 2
                            part = _r32(part[:, :width] + part[:, width:2 * width])
                        best = torch.maximum(best, part[:, 0])
                    ranked = sorted(range(1, pages - 1), key=lambda p, s=best.tolist(): (-s[p], p))
                    allowed[h, [0, pages - 1] + ranked[:top - 2]] = True
            listed_ = torch.full((hk, top), -1, dtype=torch.int32)
            for h in range(hk):
                mine = allowed[h].nonzero()[:, 0].to(torch.int32).cpu()
                listed_[h, :mine.numel()] = mine
            all_blocks.append(listed_)
            all_counts.append(torch.full((hk,), min(top, pages), dtype=torch.int32))
            token = allowed.repeat_interleave(pl, 1)[:, :n].repeat_interleave(hq // hk, 0)
            logit = torch.where(token, logit, -float("inf"))
        p = torch.softmax(logit, -1)
        for h in range(hq):
            out[i, h, 0] = p[h] @ v[:, h // (hq // hv)]
    if op == "decode":
        return dict(out=out)
    return dict(out=out, blocks=torch.stack(all_blocks), counts=torch.stack(all_counts))
