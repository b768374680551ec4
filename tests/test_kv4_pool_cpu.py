"""A pool's tensors and sizes are bound into its descriptor once, so they cannot be exchanged on the pool."""
import pytest
import torch

from saga_b200 import kv4


@pytest.mark.parametrize("name", ["k", "v", "k_lo", "k_hi", "page_len", "head_dim", "num_pages"])
def test_a_bound_pool_refuses_other_tensors(name):
    pool = kv4.Kv4Pool.__new__(kv4.Kv4Pool)
    setattr(pool, name, None)                # before it is bound
    pool.__dict__["_handle"] = object()
    with pytest.raises(AttributeError, match="Kv4Pool.of"):
        setattr(pool, name, torch.zeros(1))
    with pytest.raises(AttributeError, match="Kv4Pool.of"):
        delattr(pool, name)
    assert getattr(pool, name) is None
