"""Host-side checks of the 4-bit cache operators that need no GPU: struct layouts, refusals of the C ABI
before any CUDA call, refusals of host tensors, and the oracle's own properties."""
import ctypes
import os
import random
import subprocess
import tempfile

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O
from saga_b200 import _lib as L
from saga_b200 import kv4

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "saga_b200.h")


@pytest.mark.parametrize("name", ["SagaKv4Pool", "SagaKv4Args", "SagaPageTableArgs"])
def test_struct_layouts_match_c(name):
    cls = getattr(L, name)
    fields = [f for f, _ in cls._fields_]
    prog = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){",
            f'printf("%zu\\n", sizeof({name}));']
    prog += [f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields] + ["return 0;}"]
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        open(c, "w").write("\n".join(prog))
        subprocess.run(["gcc", "-std=c99", c, "-o", exe], check=True)
        vals = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(cls)
    assert [getattr(cls, f).offset for f in fields] == vals[1:]


def _pool(**kw):
    p = L.SagaKv4Pool()
    for k, v in {**dict(Hk=1, Hv=2, D=128, page_len=128, num_pages=4, k=4096, v=8192), **kw}.items():
        setattr(p, k, v)
    return p


def _args(pool=None, **kw):
    a = L.SagaKv4Args()
    a.pool = pool or _pool()
    base = dict(dtype=L.SAGA_BF16, B=2, Hq=12, q=64, q_sb=12 * 128, q_sh=128, out=64, o_sb=12 * 128, o_sh=128,
                page_table=64, pt_sb=8, max_pages=8, lens=64, scaling=0.1, workspace=4096, workspace_bytes=1)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("a,code,needle", [
    (_args(_pool(D=96)), L.SAGA_ERR_UNSUPPORTED, "head_dim"),
    (_args(_pool(page_len=48)), L.SAGA_ERR_INVALID, "page_len"),
    (_args(_pool(page_len=16)), L.SAGA_ERR_INVALID, "page_len"),
    (_args(_pool(Hk=5)), L.SAGA_ERR_INVALID, "multiple of Hk"),
    (_args(_pool(Hv=5)), L.SAGA_ERR_INVALID, "multiple of Hv"),
    (_args(_pool(Hk=0)), L.SAGA_ERR_INVALID, "Hk"),
    (_args(_pool(k=None)), L.SAGA_ERR_INVALID, "non-NULL"),
    (_args(_pool(v=8200)), L.SAGA_ERR_INVALID, "aligned"),
    (_args(_pool(num_pages=0)), L.SAGA_ERR_INVALID, "num_pages"),
    (_args(_pool(num_pages=1 << 30)), L.SAGA_ERR_UNSUPPORTED, "tiles"),
    (_args(_pool(k_lo=4096)), L.SAGA_ERR_INVALID, "go together"),
    (_args(dtype=7), L.SAGA_ERR_INVALID, "dtype"),
    (_args(B=-1), L.SAGA_ERR_INVALID, "B >= 0"),
    (_args(B=1 << 30), L.SAGA_ERR_UNSUPPORTED, "rows"),
    (_args(q=None), L.SAGA_ERR_INVALID, "q must"),
    (_args(out=None), L.SAGA_ERR_INVALID, "out must"),
    (_args(lens=None), L.SAGA_ERR_INVALID, "lens must"),
    (_args(page_table=None), L.SAGA_ERR_INVALID, "page_table"),
    (_args(page_table=66), L.SAGA_ERR_INVALID, "page_table"),
    (_args(max_pages=0), L.SAGA_ERR_INVALID, "max_pages"),
    (_args(pt_sb=7), L.SAGA_ERR_INVALID, "max_pages"),
    (_args(max_pages=1 << 25, pt_sb=1 << 25), L.SAGA_ERR_UNSUPPORTED, "2^31"),
    (_args(scaling=float("inf")), L.SAGA_ERR_INVALID, "scaling"),
    (_args(blocks=64, top=4), L.SAGA_ERR_INVALID, "go together"),
    (_args(blocks=64, counts=64, top=0), L.SAGA_ERR_INVALID, "top"),
    (_args(workspace=None), L.SAGA_ERR_WORKSPACE, "workspace"),
    (_args(), L.SAGA_ERR_WORKSPACE, "workspace"),
])
def test_decode_refused_on_the_host(a, code, needle):
    assert L.lib.saga_kv4_decode(ctypes.byref(a), None) == code
    assert needle in L.lib.saga_last_error().decode()


@pytest.mark.parametrize("kw,needle", [
    (dict(), "bounds"),
    (dict(pool=_pool(k_lo=4096, k_hi=4096), top=4), "blocks and counts"),
    (dict(pool=_pool(k_lo=4096, k_hi=4096), top=4, blocks=64, counts=64, keep_last=0), "keep_last"),
    (dict(pool=_pool(k_lo=4096, k_hi=4096), top=1, blocks=64, counts=64, keep_first=1, keep_last=1), "keep_first"),
])
def test_select_refused_on_the_host(kw, needle):
    a = _args(**{"top": 4, "keep_last": 1, **kw})
    assert L.lib.saga_kv4_select(ctypes.byref(a), None) == L.SAGA_ERR_INVALID
    assert needle in L.lib.saga_last_error().decode()


def test_other_entry_points_refuse_on_the_host():
    lib = L.lib
    assert lib.saga_kv4_page_bytes(128, 128) == 128 * 72 and lib.saga_kv4_page_bytes(64, 32) == 32 * 36
    assert lib.saga_kv4_page_bytes(80, 128) == 0 and lib.saga_kv4_page_bytes(64, 0) == 0
    assert lib.saga_kv4_workspace_bytes(ctypes.byref(_args(_pool(D=32))), L.SAGA_KV4_DECODE) == 0
    assert lib.saga_kv4_workspace_bytes(ctypes.byref(_args()), 9) == 0
    assert lib.saga_kv4_decode(None, None) == L.SAGA_ERR_INVALID
    p = _pool()
    assert lib.saga_kv4_write(None, 0, 1, 64, 0, 0, 64, 0, 0, 64, None, None) == L.SAGA_ERR_INVALID
    assert lib.saga_kv4_write(ctypes.byref(p), 9, 1, 64, 0, 0, 64, 0, 0, 64, None, None) == L.SAGA_ERR_INVALID
    assert lib.saga_kv4_write(ctypes.byref(p), 0, -1, 64, 0, 0, 64, 0, 0, 64, None, None) == L.SAGA_ERR_INVALID
    assert lib.saga_kv4_read(ctypes.byref(p), 0, 1, None, 64, 0, 0, 64, 0, 0, None, None) == L.SAGA_ERR_INVALID
    assert lib.saga_kv4_write(ctypes.byref(p), 0, 0, None, 0, 0, None, 0, 0, None, None, None) == L.SAGA_OK
    empty = _args(B=0, q=None, out=None)
    assert lib.saga_kv4_decode(ctypes.byref(empty), None) == L.SAGA_OK
    t = L.SagaPageTableArgs()
    assert lib.saga_page_tables(None, None) == L.SAGA_ERR_INVALID
    for kw in (dict(page_len=48), dict(B=-1), dict(num_tokens=-1), dict(num_tokens=1 << 31), dict(offsets=None),
               dict(slots=None), dict(ring=5, free_pages=None), dict(lens=None), dict(workspace=None),
               dict(workspace_bytes=31), dict(max_pages=9)):
        base = dict(B=2, page_len=64, max_pages=8, page_table=64, pt_sb=8, lens=64, new_lens=64, free_pages=64, ring=4,
                    free_state=64, num_tokens=4, slots=64, positions=64, offsets=64, lens_out=64, free_state_out=64,
                    workspace=4096, workspace_bytes=32)
        for k, v in {**base, **kw}.items():
            setattr(t, k, v)
        assert lib.saga_page_tables(ctypes.byref(t), None) < 0, kw
    assert lib.saga_slot_map(1, 64, None, 8, 8, None, 64, 4, 64, 64, None, None) == L.SAGA_ERR_INVALID
    assert lib.saga_slot_map(1, 63, 64, 8, 8, None, 64, 4, 64, 64, None, None) == L.SAGA_ERR_INVALID


def test_host_tensors_are_refused():
    i32 = dict(dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU path"):
        kv4.Kv4Pool(2, 64, 1, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="no CPU path"):
        kv4.Kv4Pool.of(torch.zeros((2, 1, 64 * 36), dtype=torch.uint8), torch.zeros((2, 1, 64 * 36), dtype=torch.uint8),
                       64, 64)
    with pytest.raises(ValueError, match="no CPU path"):
        kv4.page_tables(torch.zeros((1, 2), **i32), torch.zeros(1, **i32), torch.ones(1, **i32), torch.arange(2, **i32),
                        torch.tensor([0, 2], **i32), 1, 64)
    with pytest.raises(ValueError, match="no CPU path"):
        kv4.slot_map(torch.zeros((1, 2), **i32), torch.zeros(1, **i32), 1, 64)


def test_custom_ops_have_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        pool = [torch.empty((8, h, 64 * 36), dtype=torch.uint8, device="cuda") for h in (1, 2)]
        lo = torch.empty((8, 1, 64), dtype=torch.bfloat16, device="cuda")
        head = (*pool, lo, lo, 64, 64)
        q = torch.empty((3, 4, 1, 64), dtype=torch.bfloat16, device="cuda")
        i32 = dict(dtype=torch.int32, device="cuda")
        table, lens = torch.empty((3, 5), **i32), torch.empty(3, **i32)
        out = torch.ops.saga.kv4_decode(*head, q, table, lens, None, None, None, None)
        assert out.shape == q.shape and out.dtype == q.dtype
        blocks, counts = torch.ops.saga.kv4_select(*head, q, table, lens, 7, 1, 1)
        assert blocks.shape == (3, 1, 7) and counts.shape == (3, 1)
        slots = torch.empty(6, dtype=torch.int64, device="cuda")
        k, v = torch.ops.saga.kv4_read(*head, slots, torch.float16)
        assert k.shape == (6, 1, 64) and v.shape == (6, 2, 64) and v.dtype == torch.float16
        assert torch.ops.saga.kv4_write(*head, k, v, slots) is None
        got = torch.ops.saga.page_tables(table, lens, lens, torch.empty(9, **i32), torch.empty(2, **i32), 11, 64)
        assert [tuple(t.shape) for t in got] == [(11,), (11,), (4,), (3,), (2,)] and got[0].dtype == torch.int64


def test_oracle_quantiser_encloses_and_is_within_half_a_step():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((200, 128)) * np.exp(rng.uniform(-20, 20, (200, 1)))).astype(np.float32)
    c, s, z = O.quantise(x)
    v = O.stands_for(c, s, z)
    step = np.repeat(s, 64, -1).astype(np.float64)
    # half a step, and what binary32 loses of a quotient below 16
    assert (np.abs(v - x) <= step * (0.5 + 2.0 ** -18)).all()
    assert (z <= x.reshape(200, 2, 64).min(-1)).all()
    assert np.array_equal(O.rows_value(np.full((1, 64), 2.5)), np.full((1, 64), 2.5))


def test_oracle_score_is_an_upper_bound():
    rng = np.random.default_rng(1)
    k, q = rng.standard_normal((32, 64)), rng.standard_normal((3, 64)).astype(np.float32)
    lo, hi = O.page_bounds(k)
    assert O.block_score(q, lo, hi) >= (q.astype(np.float64) @ k.T).max() - 1e-4


def test_oracle_page_tables_keep_every_page_once():
    """Random traffic through the oracle: no page is ever held twice or lost."""
    rng = random.Random(3)
    pl, pages, B = 32, 40, 6
    table, lens = [[-1] * 12 for _ in range(B)], [0] * B
    ring, state = list(range(pages)), (0, pages)
    for _ in range(300):
        new = [rng.choice((-1, 0, 1, 1, rng.randint(0, 90))) for _ in range(B)]
        rows = sum(max(m, 0) for m in new)
        before = list(lens)
        slots, _, offsets, lens, state, failed = O.page_tables(table, lens, new, ring, *state, rows, pl)
        held = [table[b][j] for b in range(B) for j in range(-(-lens[b] // pl))]
        free = [ring[(state[0] + i) % pages] for i in range(state[1])]
        assert sorted(held + free) == list(range(pages))
        for b in range(B):
            if lens[b] == before[b] + max(new[b], 0) and new[b] > 0 and lens[b] != before[b]:
                assert all(x >= 0 for x in slots[offsets[b]:offsets[b + 1]])
        assert failed or all(x >= 0 for x in slots)
