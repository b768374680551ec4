"""Serving with a paged key/value cache held in 4 bits.

The operators of one decode step, in the order a serving loop calls them:

    step = page_tables(table, lens, new_lens, free_pages, free_state, num_tokens, page_len)
    kv4_write(pool, k, v, step.slots)                       # quantise the step's rows into their slots
    out = kv4_decode(q, pool, table, step.lens)             # attention over each request's own length
or, over a few selected blocks of each request,
    blocks, counts = kv4_select(q, pool, table, step.lens, top)
    out = kv4_decode(q, pool, table, step.lens, blocks=blocks, counts=counts)

Requests have lengths of their own, on the device; nothing here reads them on
the host, so a step can be captured in a CUDA graph. Like ``saga_b200.ops``,
the functions enqueue on the current CUDA stream and raise on host tensors.
The format of the cache is described in include/saga_b200.h. The reference
has no counterpart: its caches are 16-bit tensors with one length for the whole
batch (speedup.py:119-139).
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib as L
from .ops import _dt, _require_cuda, _stream, status_tensor

GROUP = 64  # values that share a scale
_SCRATCH: dict = {}


def _scratch(device: torch.device, nbytes: int) -> torch.Tensor:
    """Workspace of the calling stream on ``device``. The kernels do not care
    what it holds. Smaller ones are kept, since a CUDA graph may refer to them."""
    have = _SCRATCH.setdefault((device.index, _stream(device)), [])
    if not have or have[-1].numel() < nbytes:
        grown = max(nbytes, 2 * have[-1].numel() if have else 0)
        have.append(torch.empty(grown, dtype=torch.uint8, device=device))
    return have[-1]


class Kv4Pool:
    """Pages of keys and values in 4 bits, ``page_len`` positions each.

    A position's slot is ``page * page_len + offset``. With ``bounds`` the pool
    also keeps the key bounds that ``kv4_select`` reads (``k_lo``, ``k_hi``:
    bfloat16 ``[num_pages, key_heads, head_dim]``).
    """

    def __init__(self, num_pages: int, page_len: int, key_heads: int, value_heads: int, head_dim: int,
                 device="cuda", bounds: bool = False):
        nbytes = L.lib.saga_kv4_page_bytes(int(head_dim), int(page_len))
        if nbytes == 0:
            raise ValueError(L.lib.saga_last_error().decode())
        if num_pages <= 0 or key_heads <= 0 or value_heads <= 0:
            raise ValueError("num_pages, key_heads and value_heads must be positive")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("saga_b200 ops take CUDA tensors (there is no CPU path)")
        self.num_pages, self.page_len = int(num_pages), int(page_len)
        self.key_heads, self.value_heads, self.head_dim = int(key_heads), int(value_heads), int(head_dim)
        self.k = torch.zeros((num_pages, key_heads, nbytes), dtype=torch.uint8, device=device)
        self.v = torch.zeros((num_pages, value_heads, nbytes), dtype=torch.uint8, device=device)
        self.device = self.k.device
        self.k_lo = self.k_hi = None
        if bounds:
            self.k_lo, self.k_hi = (torch.zeros((num_pages, key_heads, head_dim), dtype=torch.bfloat16,
                                                device=self.device) for _ in range(2))

    def descriptor(self) -> L.SagaKv4Pool:
        p = L.SagaKv4Pool()
        p.Hk, p.Hv, p.D = self.key_heads, self.value_heads, self.head_dim
        p.page_len, p.num_pages = self.page_len, self.num_pages
        p.k, p.v = self.k.data_ptr(), self.v.data_ptr()
        if self.k_lo is not None:
            p.k_lo, p.k_hi = self.k_lo.data_ptr(), self.k_hi.data_ptr()
        return p

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_lo, self.k_hi) if t is not None)


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _int_tensor(name, t, dtype, shape=None, contiguous=True):
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {list(shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _rows(pool: Kv4Pool, k, v, slots):
    _require_cuda(k, v, slots)
    _same_device(pool.device, k=k, v=v, slots=slots)
    T = slots.numel()
    _int_tensor("slots", slots, torch.int64, (T,))
    if k.dtype != v.dtype:
        raise TypeError("k and v must share a dtype")
    for name, t, heads in (("k", k, pool.key_heads), ("v", v, pool.value_heads)):
        if tuple(t.shape) != (T, heads, pool.head_dim):
            raise ValueError(f"{name} must be [{T}, {heads}, {pool.head_dim}]")
        if t.numel() and t.stride(2) != 1:
            raise ValueError(f"{name} needs a unit stride along head_dim")
    return T


def kv4_write(pool: Kv4Pool, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise the rows ``k`` [T, Hk, D] and ``v`` [T, Hv, D] into ``slots``
    (int64 [T]; -1 skips a row). A slot outside the pool sets
    ``STATUS_PAGE_RANGE`` and skips the row. In a pool with bounds, a page whose
    last slot is written gets its key bounds. Two rows must not name one slot."""
    T = _rows(pool, k, v, slots)
    with torch.cuda.device(pool.device):
        L.check(L.lib.saga_kv4_write(ctypes.byref(pool.descriptor()), _dt(k), T, k.data_ptr(), k.stride(0),
                                     k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(),
                                     status_tensor(pool.device).data_ptr(), _stream(pool.device)), "saga_kv4_write")


def kv4_read(pool: Kv4Pool, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16
             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """What the slots stand for: ``k`` [T, Hk, D] and ``v`` [T, Hv, D] rounded
    to ``dtype``; zeros for slot -1 (and, with ``STATUS_PAGE_RANGE``, for a slot
    outside the pool). E.g. the history that a prompt chunk attends to."""
    T = slots.numel()
    k = torch.empty((T, pool.key_heads, pool.head_dim), dtype=dtype, device=pool.device)
    v = torch.empty((T, pool.value_heads, pool.head_dim), dtype=dtype, device=pool.device)
    _rows(pool, k, v, slots)
    with torch.cuda.device(pool.device):
        L.check(L.lib.saga_kv4_read(ctypes.byref(pool.descriptor()), _dt(k), T, slots.data_ptr(), k.data_ptr(),
                                    k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                                    status_tensor(pool.device).data_ptr(), _stream(pool.device)), "saga_kv4_read")
    return k, v


def _table(name, t, B):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be {torch.int32}")
    if t.dim() != 2 or t.shape[0] < B or (t.numel() and t.stride(1) != 1):
        raise ValueError(f"{name} must be an int32 [B, max_pages] tensor with unit column stride")


def _kv4_args(q, pool, page_table, lens):
    _require_cuda(q, page_table, lens)
    if q.dim() != 4 or q.shape[2] != 1:
        raise ValueError("query must be [B, Hq, 1, D]")
    B, Hq, _, D = q.shape
    if D != pool.head_dim:
        raise ValueError(f"query has head_dim {D}, the pool {pool.head_dim}")
    if q.numel() and q.stride(3) != 1:
        raise ValueError("query needs a unit stride along head_dim")
    _same_device(pool.device, query=q, page_table=page_table, lens=lens)
    _table("page_table", page_table, B)
    _int_tensor("lens", lens, torch.int32, (B,))
    a = L.SagaKv4Args()
    a.pool = pool.descriptor()
    a.dtype, a.B, a.Hq = _dt(q), B, Hq
    a.q, a.q_sb, a.q_sh = q.data_ptr(), q.stride(0), q.stride(1)
    a.page_table, a.pt_sb, a.max_pages = page_table.data_ptr(), page_table.stride(0), page_table.shape[1]
    a.lens = lens.data_ptr()
    a.status = status_tensor(pool.device).data_ptr()
    return a


def _kv4_run(fn_name, a, op, device):
    with torch.cuda.device(device):
        nbytes = L.lib.saga_kv4_workspace_bytes(ctypes.byref(a), op)
        if nbytes == 0:
            raise L.SagaError(L.SAGA_ERR_INVALID, "saga_kv4_workspace_bytes")
        ws = _scratch(device, nbytes)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        L.check(getattr(L.lib, fn_name)(ctypes.byref(a), _stream(device)), fn_name)


def kv4_decode(query: torch.Tensor, pool: Kv4Pool, page_table: torch.Tensor, lens: torch.Tensor,
               scaling: Optional[float] = None, starts: Optional[torch.Tensor] = None,
               blocks: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``query`` [B, Hq, 1, D] over the 4-bit cache -> [B, Hq, 1, D].

    Request b attends to its positions [starts[b], lens[b]) (int32 [B]; no
    ``starts`` = 0: a start serves padding on the left or a sliding window).
    ``page_table`` is int32 [B, max_pages]. A request without positions gets
    zeros. With ``blocks`` and ``counts`` (``kv4_select``) each key head attends
    to those pages alone. ``scaling`` defaults to 1/sqrt(D).
    """
    a = _kv4_args(query, pool, page_table, lens)
    a.scaling = float(1.0 / math.sqrt(a.pool.D) if scaling is None else scaling)
    if starts is not None:
        _require_cuda(starts)
        _same_device(pool.device, starts=starts)
        a.starts = _int_tensor("starts", starts, torch.int32, (a.B,)).data_ptr()
    if (blocks is None) != (counts is None):
        raise ValueError("blocks and counts go together")
    if blocks is not None:
        _require_cuda(blocks, counts)
        _same_device(pool.device, blocks=blocks, counts=counts)
        if blocks.dim() != 3:
            raise ValueError("blocks must be [B, Hk, top]")
        a.top = blocks.shape[2]
        a.blocks = _int_tensor("blocks", blocks, torch.int32, (a.B, pool.key_heads, a.top)).data_ptr()
        a.counts = _int_tensor("counts", counts, torch.int32, (a.B, pool.key_heads)).data_ptr()
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if a.B == 0:
        return out
    a.out, a.o_sb, a.o_sh = out.data_ptr(), out.stride(0), out.stride(1)
    _kv4_run("saga_kv4_decode", a, L.SAGA_KV4_DECODE, pool.device)
    return out


def kv4_select(query: torch.Tensor, pool: Kv4Pool, page_table: torch.Tensor, lens: torch.Tensor, top: int,
               keep_first: int = 1, keep_last: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """The ``top`` pages that each key head's queries attend to, by a score that
    reads only the pages' key bounds (an upper bound of the page's scores).

    Returns ``blocks`` int32 [B, Hk, top], ascending, -1 beyond ``counts`` int32
    [B, Hk]. The first ``keep_first`` and the last ``keep_last`` (>= 1: the last
    page is still filling) pages are always kept; ties go to the lower page;
    a request with at most ``top`` pages keeps them all.
    """
    a = _kv4_args(query, pool, page_table, lens)
    if pool.k_lo is None:
        raise ValueError("kv4_select needs a pool with bounds=True")
    a.top, a.keep_first, a.keep_last = int(top), int(keep_first), int(keep_last)
    if a.top <= 0:
        raise ValueError("top must be positive")
    blocks = torch.empty((a.B, pool.key_heads, a.top), dtype=torch.int32, device=pool.device)
    counts = torch.empty((a.B, pool.key_heads), dtype=torch.int32, device=pool.device)
    if a.B == 0:
        return blocks, counts
    a.blocks, a.counts = blocks.data_ptr(), counts.data_ptr()
    _kv4_run("saga_kv4_select", a, L.SAGA_KV4_SELECT, pool.device)
    return blocks, counts


class PageStep(NamedTuple):
    """What ``page_tables`` says about a step's token rows and requests."""
    slots: torch.Tensor       # int64 [num_tokens], -1 where there is no token
    positions: torch.Tensor   # int32 [num_tokens], 0 where there is no token
    offsets: torch.Tensor     # int32 [B + 1]: request b's rows are offsets[b] .. offsets[b + 1]
    lens: torch.Tensor        # int32 [B], after the step
    free_state: torch.Tensor  # int32 [2], after the step


def page_tables(page_table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
                free_state: torch.Tensor, num_tokens: int, page_len: int, lens_out: Optional[torch.Tensor] = None,
                free_state_out: Optional[torch.Tensor] = None) -> PageStep:
    """Block tables and slot maps of one step, built on the GPU.

    Request b holds ``lens[b]`` positions and adds ``new_lens[b]`` (int32 [B]);
    its tokens are consecutive rows of the step's ``num_tokens`` rows. The pages
    that it needs come from the front of the ring ``free_pages`` (int32; room for
    every page; ``free_state`` int32 [2] = index of the first free entry, number
    of free entries) and are entered in ``page_table`` (int32 [B, max_pages], in
    place). A request that cannot be given all its pages, table entries or rows
    gets nothing: slots -1, its length unchanged, ``STATUS_OUT_OF_PAGES`` set.
    ``new_lens[b] < 0`` finishes request b: its pages return to the ring's end
    and its length becomes 0.

    ``lens_out`` and ``free_state_out`` may be ``lens`` and ``free_state`` (an
    update in place, e.g. inside a CUDA graph); by default they are new tensors.
    """
    _require_cuda(page_table, lens, new_lens, free_pages, free_state, lens_out, free_state_out)
    B, dev = lens.numel(), page_table.device
    _same_device(dev, lens=lens, new_lens=new_lens, free_pages=free_pages, free_state=free_state, lens_out=lens_out,
                 free_state_out=free_state_out)
    _table("page_table", page_table, B)
    if lens_out is None:
        lens_out = torch.empty_like(lens)
    if free_state_out is None:
        free_state_out = torch.empty_like(free_state)
    for name, t, shape in (("lens", lens, (B,)), ("new_lens", new_lens, (B,)), ("free_state", free_state, (2,)),
                           ("free_pages", free_pages, (free_pages.numel(),)), ("lens_out", lens_out, (B,)),
                           ("free_state_out", free_state_out, (2,))):
        _int_tensor(name, t, torch.int32, shape)
    num_tokens = int(num_tokens)
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    positions = torch.empty(num_tokens, dtype=torch.int32, device=dev)
    offsets = torch.empty(B + 1, dtype=torch.int32, device=dev)
    a = L.SagaPageTableArgs()
    a.B, a.page_len, a.max_pages = B, int(page_len), page_table.shape[1]
    a.page_table, a.pt_sb = page_table.data_ptr(), page_table.stride(0)
    a.lens, a.new_lens = lens.data_ptr(), new_lens.data_ptr()
    a.free_pages, a.ring, a.free_state = free_pages.data_ptr(), free_pages.numel(), free_state.data_ptr()
    a.num_tokens, a.slots, a.positions = num_tokens, slots.data_ptr(), positions.data_ptr()
    a.offsets, a.lens_out, a.free_state_out = offsets.data_ptr(), lens_out.data_ptr(), free_state_out.data_ptr()
    a.status = status_tensor(dev).data_ptr()
    with torch.cuda.device(dev):
        ws = _scratch(dev, max(16 * B, 16))
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        L.check(L.lib.saga_page_tables(ctypes.byref(a), _stream(dev)), "saga_page_tables")
    return PageStep(slots, positions, offsets, lens_out, free_state_out)


def slot_map(page_table: torch.Tensor, lens: torch.Tensor, num_tokens: int, page_len: int,
             starts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The slots (int64 [num_tokens]) of the positions [starts[b], lens[b]) that
    the requests already hold, packed in order of the requests, and their
    offsets (int32 [B + 1]). Rows beyond the last position get -1."""
    _require_cuda(page_table, lens, starts)
    B, dev = lens.numel(), page_table.device
    _same_device(dev, lens=lens, starts=starts)
    _table("page_table", page_table, B)
    _int_tensor("lens", lens, torch.int32, (B,))
    if starts is not None:
        _int_tensor("starts", starts, torch.int32, (B,))
    num_tokens = int(num_tokens)
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    offsets = torch.empty(B + 1, dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        L.check(L.lib.saga_slot_map(B, int(page_len), page_table.data_ptr(), page_table.stride(0),
                                    page_table.shape[1], starts.data_ptr() if starts is not None else None,
                                    lens.data_ptr(), num_tokens, slots.data_ptr(), offsets.data_ptr(),
                                    status_tensor(dev).data_ptr(), _stream(dev)), "saga_slot_map")
    return slots, offsets
