"""Calls of the 4-bit cache operators that the compiled host module leaves to Python: valid calls with an integer
scaling, numpy integers or odd views make the same calls of the C ABI, with a workspace of their own.
"""
import ctypes
import threading

import numpy as np
import pytest
import torch

from test_gpu_kv4 import DEV, Cache, _status, gen  # noqa: F401

pytestmark = pytest.mark.gpu


def queries(c, hq, seed=3, dtype=torch.bfloat16):
    return torch.randn((len(c.lens), hq, 1, c.d), generator=gen(seed), device=DEV).to(dtype)


def test_integers_of_other_types():
    from saga_b200 import kv4
    c = Cache([3000, 40, 900], 1, 2, 64, 64, seed=61, bounds=True)
    q = queries(c, 12)
    for scaling in (1, np.float32(1.0), np.int64(1)):
        assert torch.equal(kv4.kv4_decode(q, c.pool, c.table, c.device_lens, scaling=scaling),
                           kv4.kv4_decode(q, c.pool, c.table, c.device_lens, scaling=1.0))
    want = kv4.kv4_select(q, c.pool, c.table, c.device_lens, 7, 2, 3)
    got = kv4.kv4_select(q, c.pool, c.table, c.device_lens, np.int64(7), np.int32(2), np.int64(3))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    i32 = dict(dtype=torch.int32, device=DEV)
    steps = []
    for integer in (int, np.int64):
        table, lens = torch.full((3, 9), -1, **i32), torch.zeros(3, **i32)
        ring, state = torch.arange(20, **i32), torch.tensor([18, 20], **i32)
        step = kv4.page_tables(table, lens, torch.tensor([70, 1, 300], **i32), ring, state, integer(375), integer(64))
        steps.append((*step, table, ring))
    assert all(torch.equal(a, b) for a, b in zip(*steps))


def test_a_call_from_python_shares_no_workspace_with_a_call_begun_inside_it():
    """ctypes lets other threads run during a call: what such a thread would do is done here inside the call."""
    from saga_b200 import _lib as L
    from saga_b200 import kv4
    c = Cache([300, 70], 1, 2, 64, 64, seed=62)
    q = queries(c, 4)
    spans = []

    def other(args, stream):
        a = ctypes.cast(args, ctypes.POINTER(L.SagaKv4Args)).contents
        spans.append((a.workspace, a.workspace_bytes))
        if len(spans) < 3:
            kv4._kv4_run(other, "other", kv4._kv4_args(q, c.pool, c.table, c.device_lens), L.SAGA_KV4_DECODE, c.pool)
        return 0

    other(ctypes.byref(L.SagaKv4Args(workspace=0, workspace_bytes=0)), None)
    spans = sorted(spans[1:])
    assert len(spans) == 2 and spans[0][0] + spans[0][1] <= spans[1][0]


def test_tables_from_python_share_no_workspace_with_a_call_begun_inside(monkeypatch):
    from saga_b200 import _lib as L
    from saga_b200 import kv4
    i32 = dict(dtype=torch.int32, device=DEV)
    spans = []

    def call():
        kv4.page_tables(torch.zeros((2, 4), **i32), torch.zeros(2, **i32), torch.ones(2, **i32), torch.arange(8, **i32),
                        torch.tensor([0, 8], **i32), np.int64(2), 64)

    def other(args, stream):
        a = ctypes.cast(args, ctypes.POINTER(L.SagaPageTableArgs)).contents
        spans.append((a.workspace, a.workspace_bytes))
        if len(spans) < 2:
            call()
        return 0

    monkeypatch.setattr(L.lib, "saga_page_tables", other)
    call()
    spans.sort()
    assert len(spans) == 2 and spans[0][0] + spans[0][1] <= spans[1][0]


def test_threads_on_one_stream():
    """Calls of both kinds from several threads on one stream give what each gives alone."""
    from saga_b200 import kv4
    caches = [Cache([9000 + 100 * i, 30], 1, 2, 128, 128, seed=63 + i) for i in range(4)]
    qs = [queries(c, 12, seed=70 + i) for i, c in enumerate(caches)]
    scalings = [1, 1.0, np.float64(0.5), 0.25]
    want = [kv4.kv4_decode(q, c.pool, c.table, c.device_lens, scaling=float(s))
            for q, c, s in zip(qs, caches, scalings)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    wrong, gate = [], threading.Barrier(len(caches))

    def work(i):
        with torch.cuda.stream(stream):
            gate.wait()
            outs = [kv4.kv4_decode(qs[i], caches[i].pool, caches[i].table, caches[i].device_lens, scaling=scalings[i])
                    for _ in range(50)]
            stream.synchronize()
            wrong.extend(i for o in outs if not torch.equal(o, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(caches))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_the_negative_bit_is_not_ignored(dtype):
    """A view whose sign is only noted on the tensor (as of a conjugate's imaginary part) stands for its values."""
    from saga_b200 import kv4
    c = Cache([200, 90], 1, 2, 64, 32, "fp32", seed=68, bounds=True)
    q = queries(c, 8, dtype=dtype)
    neg = torch._neg_view(-q)
    assert neg.is_neg() and torch.equal(neg, q)
    assert torch.equal(kv4.kv4_decode(neg, c.pool, c.table, c.device_lens),
                       kv4.kv4_decode(q, c.pool, c.table, c.device_lens))
    for a, b in zip(kv4.kv4_select(neg, c.pool, c.table, c.device_lens, 3),
                    kv4.kv4_select(q, c.pool, c.table, c.device_lens, 3)):
        assert torch.equal(a, b)
    k, v = (torch.randn((40, h, 64), generator=gen(h), device=DEV).to(dtype) for h in (1, 2))
    slots = torch.arange(40, device=DEV)
    pools = [kv4.Kv4Pool(2, 32, 1, 2, 64, device=DEV) for _ in range(2)]
    kv4.kv4_write(pools[0], k, v, slots)
    kv4.kv4_write(pools[1], torch._neg_view(-k), torch._neg_view(-v), slots)
    assert torch.equal(pools[0].k, pools[1].k) and torch.equal(pools[0].v, pools[1].v)


def test_strides_of_dimensions_of_one():
    """The stride of a table's only column, and of its only row, says nothing."""
    from saga_b200 import kv4
    c = Cache([200], 1, 2, 64, 32, seed=69, bounds=True)
    q = queries(c, 8)
    row = c.table.as_strided(c.table.shape, (1, 1))
    assert row.stride(0) == 1 and row.shape[1] > 1
    assert torch.equal(kv4.kv4_decode(q, c.pool, row, c.device_lens), kv4.kv4_decode(q, c.pool, c.table, c.device_lens))
    for a, b in zip(kv4.kv4_select(q, c.pool, row, c.device_lens, 3), kv4.kv4_select(q, c.pool, c.table, c.device_lens, 3)):
        assert torch.equal(a, b)
    for a, b in zip(kv4.slot_map(row, c.device_lens, 200, 32), kv4.slot_map(c.table, c.device_lens, 200, 32)):
        assert torch.equal(a, b)
    c = Cache([20, 32, 5], 1, 2, 64, 32, seed=70)
    q = queries(c, 8)
    one = c.table[:, 0].contiguous()
    column = one.view(1, 3).t()
    assert column.stride() == (1, 3)
    assert torch.equal(kv4.kv4_decode(q, c.pool, column, c.device_lens),
                       kv4.kv4_decode(q, c.pool, one[:, None], c.device_lens))
    i32 = dict(dtype=torch.int32, device=DEV)
    tables = [torch.full((1, 3), -1, **i32).t(), torch.full((3, 1), -1, **i32)]
    steps = [kv4.page_tables(t, torch.zeros(3, **i32), torch.tensor([5, 0, 32], **i32), torch.arange(9, **i32),
                             torch.tensor([0, 9], **i32), 37, 32) for t in tables]
    assert all(torch.equal(a, b) for a, b in zip(*steps)) and torch.equal(*tables)
    tables = [torch.full((5, 1), -1, **i32).t(), torch.full((1, 5), -1, **i32)]
    steps = [kv4.page_tables(t, torch.zeros(1, **i32), torch.tensor([100], **i32), torch.arange(9, **i32),
                             torch.tensor([0, 9], **i32), 100, 32) for t in tables]
    assert all(torch.equal(a, b) for a, b in zip(*steps)) and torch.equal(*tables)
