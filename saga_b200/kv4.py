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
import re
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib as L
from .ops import _DT, _STATUS, status_tensor

try:
    from . import _fastcall as _fast  # after torch, whose libraries it uses
except ImportError as e:
    raise ImportError("saga_b200/_fastcall is missing or does not load: build it with "
                      "`python -m saga_b200.build --force`") from e


def _check_built_for(module) -> None:
    """Refuses a call module built against another torch, whose tensors may be laid out otherwise."""
    built, have = getattr(module, "torch_version", None), re.match(r"\d+\.\d+\.\d+", torch.__version__).group()
    if built != have:
        raise ImportError(f"saga_b200/_fastcall was built for torch {built}, this is {have}: build it again with "
                          "`python -m saga_b200.build --force`")


_check_built_for(_fast)
_fast.bind(*(ctypes.cast(getattr(L.lib, f), ctypes.c_void_p).value for f in
             ("saga_kv4_write", "saga_kv4_read", "saga_kv4_workspace_bytes", "saga_kv4_decode", "saga_kv4_select",
              "saga_page_tables")))

GROUP = 64  # values that share a scale
_I32, _I64 = torch.int32, torch.int64
_raw_stream = torch._C._cuda_getCurrentRawStream


def _status(index: int) -> int:
    t = _STATUS.get(index)
    return (status_tensor(torch.device("cuda", index)) if t is None else t).data_ptr()


class _on_device:
    """Makes a device current for a C call, where it is not."""

    def __init__(self, index: int):
        self.index = index

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch._C._cuda_setDevice(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch._C._cuda_setDevice(self.before)


def _bad_cuda():
    raise ValueError("saga_b200 ops take CUDA tensors (there is no CPU path)")


def _bad(name: str, t, index: int, dtype, shape):
    """The error that says what is wrong with an integer argument."""
    if not t.is_cuda:
        _bad_cuda()
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{index}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {list(shape)}")
    raise ValueError(f"{name} must be contiguous")


def _ints(name: str, t, index: int, dtype, shape) -> int:
    """Address of a contiguous integer tensor of this device, type and shape."""
    if not (t.dtype is dtype and t.get_device() == index and t.shape == shape and t.is_contiguous()):
        _bad(name, t, index, dtype, shape)
    return t.data_ptr()


class Kv4Pool:
    """Pages of keys and values in 4 bits, ``page_len`` positions each.

    A position's slot is ``page * page_len + offset``. With ``bounds`` the pool
    also keeps the key bounds that ``kv4_select`` reads (``k_lo``, ``k_hi``:
    bfloat16 ``[num_pages, key_heads, head_dim]``). Its tensors can be written
    to, but not exchanged: the calls know their addresses.
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
        k = torch.zeros((num_pages, key_heads, nbytes), dtype=torch.uint8, device=device)
        v = torch.zeros((num_pages, value_heads, nbytes), dtype=torch.uint8, device=device)
        lo = hi = None
        if bounds:
            lo, hi = (torch.zeros((num_pages, key_heads, head_dim), dtype=torch.bfloat16, device=device)
                      for _ in range(2))
        self._bind(k, v, int(page_len), int(head_dim), lo, hi)

    @classmethod
    def of(cls, k: torch.Tensor, v: torch.Tensor, page_len: int, head_dim: int, k_lo: Optional[torch.Tensor] = None,
           k_hi: Optional[torch.Tensor] = None) -> "Kv4Pool":
        """The pool whose tensors these are (``pool.k``, ``pool.v``, ...)."""
        nbytes = L.lib.saga_kv4_page_bytes(int(head_dim), int(page_len))
        if nbytes == 0:
            raise ValueError(L.lib.saga_last_error().decode())
        if not (k.is_cuda and v.is_cuda):
            _bad_cuda()
        for name, t in (("k", k), ("v", v)):
            if t.dtype != torch.uint8 or t.dim() != 3 or t.shape[2] != nbytes or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous uint8 [num_pages, heads, {nbytes}] tensor")
        if k.device != v.device or k.shape[0] != v.shape[0]:
            raise ValueError("k and v must share a device and num_pages")
        if (k_lo is None) != (k_hi is None):
            raise ValueError("k_lo and k_hi go together")
        for name, t in (("k_lo", k_lo), ("k_hi", k_hi)):
            if t is not None and not (t.dtype is torch.bfloat16 and t.device == k.device and t.is_contiguous()
                                      and t.shape == (k.shape[0], k.shape[1], head_dim)):
                raise ValueError(f"{name} must be a contiguous bfloat16 [num_pages, key_heads, head_dim] tensor")
        pool = cls.__new__(cls)
        pool._bind(k, v, int(page_len), int(head_dim), k_lo, k_hi)
        return pool

    def _bind(self, k, v, page_len, head_dim, k_lo, k_hi):
        self.k, self.v, self.k_lo, self.k_hi = k, v, k_lo, k_hi
        self.page_len, self.head_dim = page_len, head_dim
        self.num_pages, self.key_heads, self.value_heads = k.shape[0], k.shape[1], v.shape[1]
        self.device = k.device
        self._index = self.device.index
        self._desc = self.descriptor()
        self._ref = ctypes.byref(self._desc)
        self._status = _status(self._index)
        self._handle = _fast.pool(ctypes.addressof(self._desc), self._index, self._status)

    def __setattr__(self, name, value):
        if "_handle" in self.__dict__:
            raise AttributeError(f"{name} of a Kv4Pool is fixed: Kv4Pool.of makes a pool of other tensors")
        super().__setattr__(name, value)

    def __delattr__(self, name):
        raise AttributeError(f"{name} of a Kv4Pool is fixed: Kv4Pool.of makes a pool of other tensors")

    def descriptor(self) -> L.SagaKv4Pool:
        """The C descriptor of the pool's tensors."""
        p = L.SagaKv4Pool()
        p.Hk, p.Hv, p.D = self.key_heads, self.value_heads, self.head_dim
        p.page_len, p.num_pages = self.page_len, self.num_pages
        p.k, p.v = self.k.data_ptr(), self.v.data_ptr()
        if self.k_lo is not None:
            p.k_lo, p.k_hi = self.k_lo.data_ptr(), self.k_hi.data_ptr()
        return p

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_lo, self.k_hi) if t is not None)


def _rows(pool: Kv4Pool, k, v, slots) -> int:
    T = slots.numel()
    _ints("slots", slots, pool._index, _I64, (T,))
    for name, t, heads in (("k", k, pool.key_heads), ("v", v, pool.value_heads)):
        if t.get_device() != pool._index:
            if not t.is_cuda:
                _bad_cuda()
            raise ValueError(f"{name} is on {t.device}, not on {pool.device}")
        if t.shape != (T, heads, pool.head_dim):
            raise ValueError(f"{name} must be [{T}, {heads}, {pool.head_dim}]")
        if t.stride(2) != 1 and t.numel():
            raise ValueError(f"{name} needs a unit stride along head_dim")
    if k.dtype is not v.dtype:
        raise TypeError("k and v must share a dtype")
    return T


def _dtype_code(dtype) -> int:
    code = _DT.get(dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {dtype} (bf16, fp16 or fp32)")
    return code


def kv4_write(pool: Kv4Pool, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise the rows ``k`` [T, Hk, D] and ``v`` [T, Hv, D] into ``slots``
    (int64 [T]; -1 skips a row). A slot outside the pool sets
    ``STATUS_PAGE_RANGE`` and skips the row. In a pool with bounds, a page whose
    last slot is written gets its key bounds. Two rows must not name one slot."""
    if torch.compiler.is_compiling():
        return torch.ops.saga.kv4_write(*_tensors(pool), k, v, slots)
    if _fast.write(pool._handle, k, v, slots):
        return
    k, v = k.resolve_neg(), v.resolve_neg()
    T = _rows(pool, k, v, slots)
    ks, vs = k.stride(), v.stride()
    with _on_device(pool._index):
        rc = L.lib.saga_kv4_write(pool._ref, _dtype_code(k.dtype), T, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0],
                                  vs[1], slots.data_ptr(), pool._status, _raw_stream(pool._index))
    if rc:
        L.check(rc, "saga_kv4_write")


def kv4_read(pool: Kv4Pool, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16
             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """What the slots stand for: ``k`` [T, Hk, D] and ``v`` [T, Hv, D] rounded
    to ``dtype``; zeros for slot -1 (and, with ``STATUS_PAGE_RANGE``, for a slot
    outside the pool). E.g. the history that a prompt chunk attends to."""
    if torch.compiler.is_compiling():
        return torch.ops.saga.kv4_read(*_tensors(pool), slots, dtype)
    got = _fast.read(pool._handle, slots, dtype)
    if got is not None:
        return got
    T = slots.numel()
    code = _dtype_code(dtype)
    at = _ints("slots", slots, pool._index, _I64, (T,))
    D = pool.head_dim
    k = torch.empty((T, pool.key_heads, D), dtype=dtype, device=pool.device)
    v = torch.empty((T, pool.value_heads, D), dtype=dtype, device=pool.device)
    with _on_device(pool._index):
        rc = L.lib.saga_kv4_read(pool._ref, code, T, at, k.data_ptr(), pool.key_heads * D, D, v.data_ptr(),
                                 pool.value_heads * D, D, pool._status, _raw_stream(pool._index))
    if rc:
        L.check(rc, "saga_kv4_read")
    return k, v


def _table(t, index: int, B: int) -> Tuple[int, int]:
    """Address and row stride of a page table. The stride of a dimension of one says nothing."""
    if t.dtype is not _I32:
        raise TypeError(f"page_table must be {_I32}")
    if not t.is_cuda:
        _bad_cuda()
    if t.get_device() != index:
        raise ValueError(f"page_table is on {t.device}, not on cuda:{index}")
    if t.dim() != 2 or t.shape[0] < B or (t.stride(1) != 1 and t.shape[1] > 1 and t.numel()):
        raise ValueError("page_table must be an int32 [B, max_pages] tensor with unit column stride")
    return t.data_ptr(), t.shape[1] if t.shape[0] == 1 else t.stride(0)


def _kv4_args(q, pool: Kv4Pool, page_table, lens) -> L.SagaKv4Args:
    index = pool._index
    if q.get_device() != index:
        if not q.is_cuda:
            _bad_cuda()
        raise ValueError(f"query is on {q.device}, not on {pool.device}")
    shape = q.shape
    if len(shape) != 4 or shape[2] != 1:
        raise ValueError("query must be [B, Hq, 1, D]")
    if shape[3] != pool.head_dim:
        raise ValueError(f"query has head_dim {shape[3]}, the pool {pool.head_dim}")
    qs = q.stride()
    if qs[3] != 1 and q.numel():
        raise ValueError("query needs a unit stride along head_dim")
    B = shape[0]
    a = L.SagaKv4Args()
    a.pool = pool._desc
    a.dtype = _dtype_code(q.dtype)
    a.B = B
    a.Hq = shape[1]
    a.q = q.data_ptr()
    a.q_sb = qs[0]
    a.q_sh = qs[1]
    a.page_table, a.pt_sb = _table(page_table, index, B)
    a.max_pages = page_table.shape[1]
    a.lens = _ints("lens", lens, index, _I32, (B,))
    a.status = pool._status
    return a


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """A workspace for one call. Not one that is kept: ctypes lets other threads run during a call, whose launches
    on the same stream may come between this call's."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _kv4_run(fn, name: str, a: L.SagaKv4Args, op: int, pool: Kv4Pool) -> None:
    index = pool._index
    with _on_device(index):
        ref = ctypes.byref(a)
        nbytes = L.lib.saga_kv4_workspace_bytes(ref, op)
        if nbytes == 0:
            raise L.SagaError(L.SAGA_ERR_INVALID, "saga_kv4_workspace_bytes")
        workspace = _workspace(nbytes, pool.device)
        a.workspace = workspace.data_ptr()
        a.workspace_bytes = nbytes
        rc = fn(ref, _raw_stream(index))
    if rc:
        L.check(rc, name)


def kv4_decode(query: torch.Tensor, pool: Kv4Pool, page_table: torch.Tensor, lens: torch.Tensor,
               scaling: Optional[float] = None, starts: Optional[torch.Tensor] = None,
               blocks: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``query`` [B, Hq, 1, D] over the 4-bit cache -> [B, Hq, 1, D].

    Request b attends to its positions [starts[b], lens[b]) (int32 [B]; no
    ``starts`` = 0: a start serves padding on the left or a sliding window).
    ``page_table`` is int32 [B, max_pages]. A request without positions gets
    zeros; a value group that stands for NaN reaches its own channels alone. With ``blocks`` and ``counts`` (``kv4_select``) each key head attends
    to those pages alone. ``scaling`` defaults to 1/sqrt(D).
    """
    if torch.compiler.is_compiling():
        return torch.ops.saga.kv4_decode(*_tensors(pool), query, page_table, lens, scaling, starts, blocks, counts)
    out = _fast.decode(pool._handle, query, page_table, lens, scaling, starts, blocks, counts)
    if out is not None:
        return out
    query = query.resolve_neg()
    a = _kv4_args(query, pool, page_table, lens)
    B, Hq, D = a.B, a.Hq, pool.head_dim
    a.scaling = D ** -0.5 if scaling is None else float(scaling)
    if starts is not None:
        a.starts = _ints("starts", starts, pool._index, _I32, (B,))
    if blocks is not None or counts is not None:
        if blocks is None or counts is None:
            raise ValueError("blocks and counts go together")
        if blocks.dim() != 3:
            raise ValueError("blocks must be [B, Hk, top]")
        top = blocks.shape[2]
        if top == 0:
            raise ValueError("top must be positive (blocks is empty)")
        a.top = top
        a.blocks = _ints("blocks", blocks, pool._index, _I32, (B, pool.key_heads, top))
        a.counts = _ints("counts", counts, pool._index, _I32, (B, pool.key_heads))
    out = torch.empty((B, Hq, 1, D), dtype=query.dtype, device=pool.device)
    if B == 0:
        return out
    a.out = out.data_ptr()
    a.o_sb = Hq * D
    a.o_sh = D
    _kv4_run(L.lib.saga_kv4_decode, "saga_kv4_decode", a, L.SAGA_KV4_DECODE, pool)
    return out


def kv4_select(query: torch.Tensor, pool: Kv4Pool, page_table: torch.Tensor, lens: torch.Tensor, top: int,
               keep_first: int = 1, keep_last: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """The ``top`` pages that each key head's queries attend to, by a score that
    reads only the pages' key bounds (an upper bound of the page's scores).

    Returns ``blocks`` int32 [B, Hk, top], ascending, -1 beyond ``counts`` int32
    [B, Hk]. The first ``keep_first`` and the last ``keep_last`` (>= 1: the last
    page is still filling) pages are always kept; ties go to the lower page;
    a request with at most ``top`` pages keeps them all. A window's start is not
    taken: pages before it may be chosen, which ``kv4_decode`` with ``starts``
    leaves out, so ask for that many more.
    """
    if torch.compiler.is_compiling():
        return torch.ops.saga.kv4_select(*_tensors(pool), query, page_table, lens, top, keep_first, keep_last)
    if pool.k_lo is not None:
        got = _fast.select(pool._handle, query, page_table, lens, top, keep_first, keep_last)
        if got is not None:
            return got
    query = query.resolve_neg()
    a = _kv4_args(query, pool, page_table, lens)
    if pool.k_lo is None:
        raise ValueError("kv4_select needs a pool with bounds=True")
    top = int(top)
    if top <= 0:
        raise ValueError("top must be positive")
    a.top, a.keep_first, a.keep_last = top, int(keep_first), int(keep_last)
    blocks = torch.empty((a.B, pool.key_heads, top), dtype=_I32, device=pool.device)
    counts = torch.empty((a.B, pool.key_heads), dtype=_I32, device=pool.device)
    if a.B == 0:
        return blocks, counts
    a.blocks, a.counts = blocks.data_ptr(), counts.data_ptr()
    _kv4_run(L.lib.saga_kv4_select, "saga_kv4_select", a, L.SAGA_KV4_SELECT, pool)
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
    Pages are granted in order: after a request that did not get its pages, none
    that needs a page gets one in this step, so running requests come first.
    ``new_lens[b] < 0`` finishes request b: its pages return to the ring's end
    and its length becomes 0 (in a ring without room for them it keeps both, and
    ``STATUS_PAGE_RANGE`` is set).

    ``lens_out`` and ``free_state_out`` may be ``lens`` and ``free_state`` (an
    update in place, e.g. inside a CUDA graph); by default they are new tensors.
    """
    if torch.compiler.is_compiling():
        step = PageStep(*torch.ops.saga.page_tables(page_table, lens, new_lens, free_pages, free_state, num_tokens,
                                                    page_len))
        if lens_out is not None:
            step = step._replace(lens=lens_out.copy_(step.lens))
        if free_state_out is not None:
            step = step._replace(free_state=free_state_out.copy_(step.free_state))
        return step
    if not page_table.is_cuda:
        _bad_cuda()
    got = _fast.tables(page_table, lens, new_lens, free_pages, free_state, num_tokens, page_len, lens_out,
                       free_state_out, _status(page_table.get_device()))
    if got is not None:
        return PageStep._make(got)
    index, dev = page_table.get_device(), page_table.device
    B, ring = lens.numel(), free_pages.numel()
    num_tokens = int(num_tokens)
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    a = L.SagaPageTableArgs()
    a.B = B
    a.page_len = int(page_len)
    a.page_table, a.pt_sb = _table(page_table, index, B)
    a.max_pages = page_table.shape[1]
    a.lens = _ints("lens", lens, index, _I32, (B,))
    a.new_lens = _ints("new_lens", new_lens, index, _I32, (B,))
    a.free_pages = _ints("free_pages", free_pages, index, _I32, (ring,))
    a.ring = ring
    a.free_state = _ints("free_state", free_state, index, _I32, (2,))
    if lens_out is None:
        lens_out = torch.empty_like(lens)
    if free_state_out is None:
        free_state_out = torch.empty_like(free_state)
    a.lens_out = _ints("lens_out", lens_out, index, _I32, (B,))
    a.free_state_out = _ints("free_state_out", free_state_out, index, _I32, (2,))
    slots = torch.empty(num_tokens, dtype=_I64, device=dev)
    positions = torch.empty(num_tokens, dtype=_I32, device=dev)
    offsets = torch.empty(B + 1, dtype=_I32, device=dev)
    a.num_tokens = num_tokens
    a.slots, a.positions, a.offsets = slots.data_ptr(), positions.data_ptr(), offsets.data_ptr()
    a.status = _status(index)
    nbytes = max(16 * B, 16)
    with _on_device(index):
        workspace = _workspace(nbytes, dev)
        a.workspace = workspace.data_ptr()
        a.workspace_bytes = nbytes
        rc = L.lib.saga_page_tables(ctypes.byref(a), _raw_stream(index))
    if rc:
        L.check(rc, "saga_page_tables")
    return PageStep(slots, positions, offsets, lens_out, free_state_out)


def slot_map(page_table: torch.Tensor, lens: torch.Tensor, num_tokens: int, page_len: int,
             starts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The slots (int64 [num_tokens]) of the positions [starts[b], lens[b]) that
    the requests already hold, packed in order of the requests, and their
    offsets (int32 [B + 1]). Rows beyond the last position get -1."""
    if torch.compiler.is_compiling():
        return torch.ops.saga.slot_map(page_table, lens, num_tokens, page_len, starts)
    if not page_table.is_cuda:
        _bad_cuda()
    index, dev = page_table.get_device(), page_table.device
    B = lens.numel()
    table, row = _table(page_table, index, B)
    at = _ints("lens", lens, index, _I32, (B,))
    first = None if starts is None else _ints("starts", starts, index, _I32, (B,))
    num_tokens = int(num_tokens)
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    slots = torch.empty(num_tokens, dtype=_I64, device=dev)
    offsets = torch.empty(B + 1, dtype=_I32, device=dev)
    with _on_device(index):
        rc = L.lib.saga_slot_map(B, int(page_len), table, row, page_table.shape[1], first, at, num_tokens,
                                  slots.data_ptr(), offsets.data_ptr(), _status(index), _raw_stream(index))
    if rc:
        L.check(rc, "saga_slot_map")
    return slots, offsets


# ---------------------------------------------------------------------------
# torch custom ops (opaque to torch.compile). A pool goes in as its tensors:
# k, v, k_lo, k_hi, page_len, head_dim.
# ---------------------------------------------------------------------------

def _tensors(pool: Kv4Pool):
    return pool.k, pool.v, pool.k_lo, pool.k_hi, pool.page_len, pool.head_dim


@torch.library.custom_op("saga::kv4_write", mutates_args=("k_pool", "v_pool", "k_lo", "k_hi"))
def _op_kv4_write(k_pool: torch.Tensor, v_pool: torch.Tensor, k_lo: Optional[torch.Tensor],
                  k_hi: Optional[torch.Tensor], page_len: int, head_dim: int, k: torch.Tensor, v: torch.Tensor,
                  slots: torch.Tensor) -> None:
    kv4_write(Kv4Pool.of(k_pool, v_pool, page_len, head_dim, k_lo, k_hi), k, v, slots)


@_op_kv4_write.register_fake
def _(k_pool, v_pool, k_lo, k_hi, page_len, head_dim, k, v, slots):
    return None


@torch.library.custom_op("saga::kv4_read", mutates_args=())
def _op_kv4_read(k_pool: torch.Tensor, v_pool: torch.Tensor, k_lo: Optional[torch.Tensor],
                 k_hi: Optional[torch.Tensor], page_len: int, head_dim: int, slots: torch.Tensor,
                 dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    return kv4_read(Kv4Pool.of(k_pool, v_pool, page_len, head_dim, k_lo, k_hi), slots, dtype)


@_op_kv4_read.register_fake
def _(k_pool, v_pool, k_lo, k_hi, page_len, head_dim, slots, dtype):
    return tuple(t.new_empty((slots.numel(), t.shape[1], head_dim), dtype=dtype) for t in (k_pool, v_pool))


@torch.library.custom_op("saga::kv4_decode", mutates_args=())
def _op_kv4_decode(k_pool: torch.Tensor, v_pool: torch.Tensor, k_lo: Optional[torch.Tensor],
                   k_hi: Optional[torch.Tensor], page_len: int, head_dim: int, query: torch.Tensor,
                   page_table: torch.Tensor, lens: torch.Tensor, scaling: Optional[float],
                   starts: Optional[torch.Tensor], blocks: Optional[torch.Tensor],
                   counts: Optional[torch.Tensor]) -> torch.Tensor:
    return kv4_decode(query, Kv4Pool.of(k_pool, v_pool, page_len, head_dim, k_lo, k_hi), page_table, lens, scaling,
                      starts, blocks, counts)


@_op_kv4_decode.register_fake
def _(k_pool, v_pool, k_lo, k_hi, page_len, head_dim, query, page_table, lens, scaling, starts, blocks, counts):
    return query.new_empty(query.shape)


@torch.library.custom_op("saga::kv4_select", mutates_args=())
def _op_kv4_select(k_pool: torch.Tensor, v_pool: torch.Tensor, k_lo: Optional[torch.Tensor],
                   k_hi: Optional[torch.Tensor], page_len: int, head_dim: int, query: torch.Tensor,
                   page_table: torch.Tensor, lens: torch.Tensor, top: int, keep_first: int,
                   keep_last: int) -> Tuple[torch.Tensor, torch.Tensor]:
    return kv4_select(query, Kv4Pool.of(k_pool, v_pool, page_len, head_dim, k_lo, k_hi), page_table, lens, top,
                      keep_first, keep_last)


@_op_kv4_select.register_fake
def _(k_pool, v_pool, k_lo, k_hi, page_len, head_dim, query, page_table, lens, top, keep_first, keep_last):
    rows = (query.shape[0], k_pool.shape[1])
    return query.new_empty((*rows, top), dtype=torch.int32), query.new_empty(rows, dtype=torch.int32)


@torch.library.custom_op("saga::page_tables", mutates_args=("page_table", "free_pages"))
def _op_page_tables(page_table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
                    free_state: torch.Tensor, num_tokens: int, page_len: int
                    ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(page_tables(page_table, lens, new_lens, free_pages, free_state, num_tokens, page_len))


@_op_page_tables.register_fake
def _(page_table, lens, new_lens, free_pages, free_state, num_tokens, page_len):
    return (lens.new_empty(num_tokens, dtype=torch.int64), lens.new_empty(num_tokens), lens.new_empty(lens.numel() + 1),
            torch.empty_like(lens), torch.empty_like(free_state))


@torch.library.custom_op("saga::slot_map", mutates_args=())
def _op_slot_map(page_table: torch.Tensor, lens: torch.Tensor, num_tokens: int, page_len: int,
                 starts: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    return slot_map(page_table, lens, num_tokens, page_len, starts)


@_op_slot_map.register_fake
def _(page_table, lens, num_tokens, page_len, starts):
    return lens.new_empty(num_tokens, dtype=torch.int64), lens.new_empty(lens.numel() + 1)
