"""Key bounds of long writes: more than 4096 rows in one call are looked at by strips of rows, where one CTA may
take the bounds of many pages, and a page may be longer than a strip."""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O
from test_gpu_kv4 import DEV, DT, _status, f32, gen  # noqa: F401

pytestmark = pytest.mark.gpu


def rows_of(order, T, pl, pages, rng):
    """T slots of a pool of `pages` pages."""
    if order == "in order":
        return np.arange(T)
    if order == "shifted":
        return np.arange(T) + 5
    if order == "pages permuted":
        page = rng.permutation(pages)
        return (page[:, None] * pl + np.arange(pl)).reshape(-1)[:T]
    if order == "any":
        return rng.permutation(pages * pl)[:T]
    # the last slots of all pages one after the other: a strip completes as many pages as it has rows
    last = np.arange(pages) * pl + pl - 1
    others = np.setdiff1d(np.arange(pages * pl), last)
    at = (T - pages) // 2
    return np.concatenate((others[:at], last, others[at:T - pages]))


@pytest.mark.parametrize("order", ["in order", "shifted", "pages permuted", "any", "last slots together"])
@pytest.mark.parametrize("T", [4097, 10007])
@pytest.mark.parametrize("pl,d,hk", [(32, 64, 2), (32, 128, 1), (256, 128, 1), (512, 64, 1), (512, 128, 2)])
def test_bounds_of_long_writes(pl, d, hk, T, order):
    from saga_b200 import kv4
    rng = np.random.default_rng(T + pl)
    pages = T // pl + 3
    slots = rows_of(order, T, pl, pages, rng)
    assert len(set(slots.tolist())) == T and slots.max() < pages * pl
    k = (torch.randn((T, hk, d), generator=gen(1), device=DEV) * 2).to(torch.bfloat16)
    k[::97, :, 3] = float("nan")      # groups that stand for NaN are left out of the bounds
    v = torch.zeros((T, 1, d), dtype=torch.bfloat16, device=DEV)
    pool = kv4.Kv4Pool(pages, pl, hk, 1, d, device=DEV, bounds=True)
    pool.k_lo.fill_(7)
    pool.k_hi.fill_(7)
    kv4.kv4_write(pool, k, v, torch.from_numpy(slots).to(DEV))
    held = np.zeros((pages * pl, hk, d))
    held[slots] = O.rows_value(f32(k))
    held = held.reshape(pages, pl, hk, d)
    lo, hi = (np.full((pages, hk, d), 7, np.float32) for _ in range(2))
    for p in np.unique(slots[slots % pl == pl - 1] // pl):
        for h in range(hk):
            lo[p, h], hi[p, h] = O.page_bounds(held[p, :, h])
    assert np.array_equal(f32(pool.k_lo), lo, equal_nan=True) and np.array_equal(f32(pool.k_hi), hi, equal_nan=True)
