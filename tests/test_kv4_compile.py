"""slot_map under torch.compile: its custom op, the op's fake, and a prompt chunk's history read through it."""
import pytest
import torch


def test_slot_map_has_a_fake():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from saga_b200 import kv4  # noqa: F401
    with FakeTensorMode():
        i32 = dict(dtype=torch.int32, device="cuda")
        table, lens = torch.empty((3, 5), **i32), torch.empty(3, **i32)
        for starts in (None, torch.empty(3, **i32)):
            slots, offsets = torch.ops.saga.slot_map(table, lens, 11, 64, starts)
            assert slots.shape == (11,) and slots.dtype == torch.int64
            assert offsets.shape == (4,) and offsets.dtype == torch.int32


@pytest.mark.gpu
@pytest.mark.parametrize("with_starts", [False, True])
def test_a_compiled_history_matches_eager(with_starts):
    from saga_b200 import kv4
    from test_gpu_kv4 import DEV, Cache
    c = Cache([70, 0, 130], 1, 2, 64, 32, seed=7)
    starts = torch.tensor([3, 0, 129], dtype=torch.int32, device=DEV) if with_starts else None

    def history(pool, table, lens, starts):
        slots, offsets = kv4.slot_map(table, lens, 210, pool.page_len, starts=starts)
        return (*kv4.kv4_read(pool, slots), slots, offsets)

    want = history(c.pool, c.table, c.device_lens, starts)
    got = torch.compile(history, fullgraph=True)(c.pool, c.table, c.device_lens, starts)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
