"""Page tables where the ring of free pages is too small for what comes back to it."""
import pytest
import torch

from test_gpu_kv4 import DEV, _status  # noqa: F401

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("tokens", [3, 1500])  # tokens placed by the scanning CTA, and by a launch of their own
@pytest.mark.parametrize("in_place", [False, True])
def test_a_full_ring_takes_no_more_pages(tokens, in_place):
    """Eight entries, six of them free: the first finished request's two pages fit, the next one's do not."""
    from saga_b200 import _lib, kv4, ops
    pl = 64
    table = torch.tensor([[20, 21, -1], [22, 23, 24], [-1, -1, -1], [25, -1, -1]], **I32)
    lens = torch.tensor([65, 180, 0, 64], **I32)
    ring = torch.tensor([3, 4, 5, -9, -9, 0, 1, 2], **I32)      # free: entries 5, 6, 7, 0, 1, 2
    state = torch.tensor([5, 6], **I32)
    new = torch.tensor([-1, -1, 3, -1], **I32)
    step = kv4.page_tables(table, lens, new, ring, state, tokens, pl, lens_out=lens if in_place else None,
                           free_state_out=state if in_place else None)
    assert step.lens.tolist() == [0, 180, 3, 64]
    assert ring.tolist() == [3, 4, 5, 20, 21, 0, 1, 2]
    assert step.free_state.tolist() == [6, 7]
    assert table[1].tolist() == [22, 23, 24] and table[2].tolist() == [0, -1, -1] and int(table[3, 0]) == 25
    assert step.slots[:3].tolist() == [0, 1, 2] and set(step.slots[3:].tolist()) <= {-1}
    assert ops.read_status(DEV) == _lib.STATUS_PAGE_RANGE
    # once pages have been taken there is room
    step = kv4.page_tables(table, step.lens, torch.tensor([200, 0, 0, -1], **I32), ring, step.free_state, 200, pl)
    assert ops.read_status(DEV) == _lib.STATUS_OUT_OF_PAGES     # 200 positions need more than the table's row
    step = kv4.page_tables(table, step.lens, torch.tensor([190, 0, 0, 0], **I32), ring, step.free_state, 190, pl)
    assert ops.read_status(DEV) == 0 and table[0].tolist() == [1, 2, 3]
    step = kv4.page_tables(table, step.lens, torch.tensor([0, -1, 0, 0], **I32), ring, step.free_state, 0, pl)
    assert ops.read_status(DEV) == 0 and step.lens.tolist() == [190, 0, 3, 0]
    free = [ring[(int(step.free_state[0]) + i) % 8].item() for i in range(int(step.free_state[1]))]
    assert free == [4, 5, 20, 21, 25, 22, 23, 24]


def test_no_ring_at_all_keeps_the_pages():
    from saga_b200 import _lib, kv4, ops
    table = torch.tensor([[7, 8]], **I32)
    step = kv4.page_tables(table, torch.tensor([100], **I32), torch.tensor([-1], **I32), torch.zeros(0, **I32),
                           torch.zeros(2, **I32), 2, 64)
    assert step.lens.tolist() == [100] and step.free_state.tolist() == [0, 0] and step.slots.tolist() == [-1, -1]
    assert ops.read_status(DEV) == _lib.STATUS_PAGE_RANGE


def test_many_finished_requests_in_a_ring_with_room_for_some():
    """More requests than threads of the scanning CTA: those that fit are the first ones."""
    from saga_b200 import _lib, kv4, ops
    B, room, pl = 2500, 1333, 32
    table = torch.arange(B, **I32)[:, None].contiguous()
    ring = torch.full((room,), -9, **I32)
    step = kv4.page_tables(table, torch.full((B,), 20, **I32), torch.full((B,), -1, **I32), ring,
                           torch.tensor([1000, 0], **I32), 0, pl)
    assert step.lens.tolist() == [0] * room + [20] * (B - room)
    assert step.free_state.tolist() == [1000, room]
    assert ring.roll(-1000).tolist() == list(range(room))
    assert ops.read_status(DEV) == _lib.STATUS_PAGE_RANGE
