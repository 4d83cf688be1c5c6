"""The key-value cache where it could go wrong.

The plain cases, and the helper that holds a cache next to its oracle, are in test_gpu_kvcache.py.
"""
import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from test_gpu_kvcache import Case

pytestmark = pytest.mark.gpu


def check_evict(c, budget, recent=0, sinks=0, w=None):
    new = c.cache.evict(*c.on_gpu(), budget, recent=recent, sinks=sinks, weights=None if w is None else torch.tensor(w).cuda())
    np.testing.assert_array_equal(new.cpu().numpy(), O.evict(c.ref, c.table, c.lengths, budget, recent, sinks, w))
    c.check_pool()


# -- eviction ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("lengths", [(5000, 3), (17000, 0, 9000)])
def test_evict_to_nothing(gpu, lengths, prompt):
    """A budget of 0 for rows that a cluster of blocks takes: everything goes, and nothing is written."""
    c = Case(16, 2, 2, heads=2, lengths=lengths, page_size=256)
    w = c.rng.random((len(lengths), 2, max(lengths)), np.float32) if prompt else None
    for recent, sinks in ((0, 0), (100, 4)):
        check_evict(c, 0, recent, sinks, w)


@pytest.mark.parametrize("prompt", [False, True])
def test_evict_very_long(gpu, prompt):
    """More tokens than the shared memory of a cluster's eight blocks holds the weights of (16384 each)."""
    c = Case(16, 2, 2, heads=1, lengths=(150001, 140000), page_size=1024)
    w = c.rng.random((2, 1, 150001), np.float32) if prompt else None
    check_evict(c, 70000, 500, 4, w)


@pytest.mark.parametrize("prompt", [False, True])
def test_evict_infinite_weights(gpu, prompt):
    """Protected tokens come before any weight, the infinite ones too, however many there are and wherever they lie."""
    c = Case(32, 4, 4, heads=3, lengths=(200,), page_size=16)
    w = c.rng.random((1, 3, 200), np.float32)
    w[0, 0, :150] = np.inf
    w[0, 1, 20:60] = np.inf
    w[0, 2] = np.inf
    w[0, 2, 190:] = np.nan
    if not prompt:
        pg, off, _ = O.sequence(c.ref, c.table[0], 200)
        for h in range(3):
            c.ref["weights"][pg, h, off] = w[0, h]
        c.cache.weights.copy_(torch.tensor(c.ref["weights"]))
    check_evict(c, 50, 12, 3, w if prompt else None)


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("bad", [(1,), (0, 1, 2), (8,), (1, 8, 9), (0, 1, 2, 3, 4, 5, 6, 7, 8, 9), ()])
@pytest.mark.parametrize("budget", [48, 40, 1])
def test_evict_missing_pages(gpu, bad, budget, prompt):
    """Pages outside the pool: their tokens are not there to be kept, and no kept token is moved to where it would be lost."""
    c = Case(32, 4, 4, heads=2, lengths=(160, 150), page_size=16)
    for i, p in enumerate(bad):
        c.table[0, p] = (-1, c.pages, 2 ** 31 - 1)[i % 3]
    w = c.rng.random((2, 2, 160), np.float32) if prompt else None
    check_evict(c, budget, 9, 2, w)


def test_evict_missing_pages_of_long_rows(gpu):
    """The same where a cluster of blocks takes a row, with pages missing in the shares of several of them."""
    c = Case(16, 2, 2, heads=2, lengths=(20000,), page_size=64)
    c.table[0, [0, 3, 40, 41, 42, 100, 200, 250, 312]] = -1
    check_evict(c, 9000, 700, 4)
    check_evict(c, 8999)
