"""The key-value cache where it could go wrong.

The plain cases, and the helper that holds a cache next to its oracle, are in test_gpu_kvcache.py.
"""
import math

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


# -- attention -----------------------------------------------------------------------------------------------------------

def whole_error(out, ref, extra):
    """Asserts that the error over all outputs is their type's rounding of `ref` and, independent of it, an error whose
    mean square is at most `extra` (5 % for the rounding of a few thousand other values than those of `ref`)."""
    rounded = torch.tensor(ref).to(out.dtype).double().numpy()
    bound = 1.05 * math.sqrt(((rounded - ref) ** 2).sum() + extra)
    off = math.sqrt(((out.double().cpu().numpy() - ref) ** 2).sum())
    assert off <= bound, off / bound


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("k_bits", [2, 4, 8])
@pytest.mark.parametrize("v_bits", [2, 4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_large_scores(gpu, d, k_bits, v_bits, dtype):
    """Scores of hundreds that lie within a few units, for calls with and without their logarithm: what is lost of a
    score is lost of a softmax weight, times the score."""
    c = Case(d, k_bits, v_bits, heads=2, lengths=(300, 40, 1), page_size=32, dtype=dtype)
    rng = np.random.default_rng(d)
    base = rng.standard_normal((2, d))
    for b, n in enumerate(c.lengths):
        k = torch.tensor(base + 0.1 * rng.standard_normal((n, 2, d))).to(c.dtype)
        c.append(c.slots(b, range(n)), np.arange(n, dtype=np.int32), k=k)
    q = torch.tensor(np.repeat(base, 3, 0) * 500 / math.sqrt(d) * (1 + 0.05 * rng.standard_normal((3, 6, 1)))).to(c.dtype)
    ref, rlse, sizes = O.attend(c.ref, c.kc, c.vc, q.double().numpy(), c.table, c.lengths, 1 / math.sqrt(d))
    # Scores, of up to 600: factors of 22 bits (2^-22 of the score) and sums in f32, of 2 d + 16 roundings of either sign
    # (2^-24 each): two standard deviations of their sum over all outputs, four for the worst of a few.  Weights and
    # values: 2^-11 of either for bf16, else 2^-22.
    deviation = math.sqrt((2 * d + 16) / 3) * 2.0 ** -24
    score = sizes[..., 0] * (2.0 ** -22 + 2 * deviation)
    half = 2.0 ** -11 if dtype == "bf16" else 2.0 ** -22
    extra = ((2 * score ** 2 + 2 * half ** 2) * sizes[..., 1] ** 2).sum()
    table, lengths = c.on_gpu()
    out = c.cache.attend(q.cuda(), table, lengths)
    whole_error(out, ref, extra)
    with_lse, lse = c.cache.attend(q.cuda(), table, lengths, return_lse=True)
    assert torch.equal(out, with_lse)
    assert (np.abs(lse.double().cpu().numpy() - rlse) <= 2 * score + 2.0 ** -20 + 2.0 ** -22 * np.abs(rlse)).all()


@pytest.mark.parametrize("d,k_bits,v_bits,heads,group,lengths", [(128, 4, 4, 2, 4, (1, 700, 0, 33)), (64, 4, 2, 4, 1, (900, 15)),
                                                                (256, 2, 2, 2, 16, (300, 2)), (80, 8, 8, 3, 5, (401,)),
                                                                (128, 8, 4, 2, 7, (3000,)), (200, 2, 8, 1, 9, (64, 63))])
def test_attend_bf16_whole_error(gpu, d, k_bits, v_bits, heads, group, lengths):
    """bf16 without the logarithm, the usual call: the output's own rounding, and 11 bits of weights and of values."""
    c = Case(d, k_bits, v_bits, heads=heads, lengths=lengths, page_size=64)
    q = torch.tensor(1.5 * c.rng.standard_normal((len(lengths), heads * group, d))).to(c.dtype)
    out = c.cache.attend(q.cuda(), *c.on_gpu())
    ref, _, sizes = O.attend(c.ref, c.kc, c.vc, q.double().numpy(), c.table, c.lengths, 1 / math.sqrt(d))
    # (relative to the outputs: weights' errors are independent, centroids' follow the centroids)
    whole_error(out, ref, 2 * 2.0 ** -22 * (ref ** 2).sum() + (sizes[..., 0] ** 2 * sizes[..., 1] ** 2 * 2.0 ** -40).sum())
    assert not out[torch.tensor(c.lengths == 0)].any()


def test_graph_accumulates(gpu):
    """A captured step of append and attend with accumulation: outputs, logarithms and weights of every replay."""
    c = Case(64, 4, 4, heads=2, lengths=(40, 7), page_size=16, slack=2)
    table, lengths = c.on_gpu()
    k, v, q = (torch.zeros(2, n, 64, device="cuda", dtype=torch.bfloat16) for n in (2, 2, 4))
    slots, position = torch.full((2,), -1, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")

    def step():
        c.cache.append(k, v, slots, position)
        return c.cache.attend(q, table, lengths, accumulate=True, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    c.cache.weights.copy_(torch.tensor(c.ref["weights"]))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = step()
    for i in range(4):
        kn, vn, qn = c.vectors(2), c.vectors(2), torch.tensor(c.rng.standard_normal((2, 4, 64))).bfloat16()
        new = np.array([c.slots(b, [n])[0] for b, n in enumerate(c.lengths)])
        O.append(c.ref, c.kc, c.vc, kn.float().numpy(), vn.float().numpy(), new, c.lengths.copy())
        for t, x in ((k, kn), (v, vn), (q, qn), (slots, torch.tensor(new)), (position, torch.tensor(c.lengths))):
            t.copy_(x)
        c.lengths += 1
        lengths.copy_(torch.tensor(c.lengths))
        g.replay()
        before = c.ref["weights"].astype(np.float64)
        ref, rlse, sizes = O.attend(c.ref, c.kc, c.vc, qn.double().numpy(), c.table, c.lengths, 1 / 8, accumulate=True)
        ds = sizes[..., 0] * (2.0 ** -22 + (2 * 64 + 16) * 2.0 ** -24)
        whole_error(out, ref, (2 * (ds ** 2 + 2.0 ** -22) * sizes[..., 1] ** 2).sum())
        assert (np.abs(lse.double().cpu().numpy() - rlse) <= ds + 2.0 ** -20 + 2.0 ** -22 * np.abs(rlse)).all()
        more = c.ref["weights"] - before
        err = np.abs(c.cache.weights.cpu().numpy() - c.ref["weights"])
        assert (err <= more * (np.expm1(2 * ds.max()) + 2.0 ** -20) + 2.0 ** -23 * c.ref["weights"]).all()
        c.ref["weights"] = c.cache.weights.cpu().numpy()
    c.check_pool()
