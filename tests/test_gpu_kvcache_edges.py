"""The key-value cache where it could go wrong.

The plain cases, and the helper that holds a cache next to its oracle, are in test_gpu_kvcache.py.
"""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from polarquant_b200 import KVCache, KVCodec
from test_gpu_kvcache import Case, codec

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


def with_norms(c, b, tokens, norms, side="v"):
    """Sets the stored norms of a sequence's tokens, for every head."""
    t = np.array(tokens)
    pg, off = c.table[b, t // c.page], t % c.page
    c.ref[side + "_norms"][pg, :, off] = np.asarray(norms, np.float32)[:, None]
    getattr(c.cache, side + "_norms").copy_(torch.tensor(c.ref[side + "_norms"]))


def check_weighted(c, q):
    """The outputs' error by the sum of p_j |v_j|, what was attended to, and not by the largest value."""
    d, scale = c.d, 1 / math.sqrt(c.d)
    ref = O.attend(c.ref, c.kc, c.vc, q.double().numpy(), c.table, c.lengths, scale)[0]
    size, score = np.zeros(ref.shape[:2]), np.zeros(ref.shape[:2])
    for b, h in np.ndindex(*size.shape):
        pg, off, _ = O.sequence(c.ref, c.table[b], c.lengths[b])
        at = (pg, h // (ref.shape[1] // c.heads), off)
        k = c.kc[2].astype(np.float64)[c.ref["k_codes"][at]] * c.ref["k_norms"][at].astype(np.float64)[:, None]
        v = c.vc[2].astype(np.float64)[c.ref["v_codes"][at]] * c.ref["v_norms"][at].astype(np.float64)[:, None]
        turned = c.kc[0].astype(np.float64) @ q[b, h].double().numpy()
        p = scale * (k @ turned)
        p = np.exp(p - p.max())
        size[b, h] = (p / p.sum() * np.sqrt((v ** 2).sum(-1))).sum()
        score[b, h] = scale * (np.abs(k) @ np.abs(turned))[p > 2.0 ** -60].max()  # of tokens that have weight
    out = c.cache.attend(q.cuda(), *c.on_gpu()).double().cpu().numpy()
    ds = score * (2.0 ** -22 + (2 * d + 16) * 2.0 ** -24)
    half = 2.0 ** -11 if c.dtype == torch.bfloat16 else 2.0 ** -22
    # weights off by their score's error, a rounding and an exponential (2^-22); values by a centroid's rounding; sums in f32
    bound = size * (np.expm1(2 * ds) + 2 * half + (4 * d + 64) * 2.0 ** -24)
    bound = bound + np.sqrt((ref ** 2).sum(-1)) * torch.finfo(c.dtype).eps / 2 + math.sqrt(d) * torch.finfo(c.dtype).tiny
    off = np.sqrt(((out - ref) ** 2).sum(-1))
    assert np.isfinite(out).all()
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,k_bits,v_bits", [(64, 4, 4), (128, 4, 2), (256, 2, 8)])
@pytest.mark.parametrize("log_norm", [12, 24, 30, 60, 99])
@pytest.mark.parametrize("first", [True, False])
def test_attend_unattended_large_value(gpu, d, k_bits, v_bits, dtype, log_norm, first):
    """Tokens without weight whose values are up to 2^99 times as long as the others', before and behind those: nothing is
    left of them, and nothing is lost of the others."""
    c = Case(d, k_bits, v_bits, heads=1, lengths=(300, 40), dtype=dtype, page_size=64)
    q = torch.zeros(2, 2, d)
    q[:, :, 0] = 30.0
    for b, n in enumerate(c.lengths):
        k = 0.3 * torch.tensor(c.rng.standard_normal((n, 1, d))).float()
        lost = [0, 1, 17] if first else [n - 1, n - 5]
        k[lost] = 0
        k[lost, :, 0] = -130 * math.sqrt(d) / 30  # a score of -130 or, of two bits, -110: weights below 2^-150
        c.append(c.slots(b, range(n)), np.arange(n, dtype=np.int32), k=k.to(c.dtype))
        with_norms(c, b, lost, np.full(len(lost), 2.0 ** log_norm))
    check_weighted(c, q.to(c.dtype))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_heads_of_different_tokens(gpu, dtype):
    """Two queries on one key head, one at values 2^40 times as long as the other's."""
    c = Case(64, 4, 4, heads=1, lengths=(400,), dtype=dtype, page_size=64)
    k = 0.2 * torch.tensor(c.rng.standard_normal((400, 1, 64))).float()
    k[:, :, 0] = torch.where(torch.arange(400) % 2 == 0, 20.0, -20.0)[:, None]
    c.append(c.slots(0, range(400)), np.arange(400, dtype=np.int32), k=k.to(c.dtype))
    with_norms(c, 0, range(400), np.where(np.arange(400) % 2 == 0, 2.0 ** -20, 2.0 ** 20) * np.exp(0.3 * c.rng.standard_normal(400)))
    q = torch.zeros(1, 2, 64)
    q[:, 0, 0], q[:, 1, 0] = 30.0, -30.0
    check_weighted(c, q.to(c.dtype))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_values_of_length_zero(gpu, dtype):
    """The token with all the weight has a value of 0, others' weights are 2^-40 of it; and all values 0."""
    c = Case(64, 4, 4, heads=1, lengths=(100, 30), dtype=dtype, page_size=32)
    q = torch.zeros(2, 2, 64)
    q[:, :, 0] = 16.0
    for b, n in enumerate(c.lengths):
        k = 0.1 * torch.tensor(c.rng.standard_normal((n, 1, 64))).float()
        k[3] = 0
        k[3, :, 0] = 14.0
        c.append(c.slots(b, range(n)), np.arange(n, dtype=np.int32), k=k.to(c.dtype))
        with_norms(c, b, range(n), np.where(np.arange(n) == 3, 0.0, 2.0 ** 30 if dtype != "f16" else 2.0 ** 34))
    check_weighted(c, q.to(c.dtype))
    with_norms(c, 1, range(30), np.zeros(30))
    check_weighted(c, q.to(c.dtype))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("log_norm", [99.9, -60.0])
def test_attend_values_of_extreme_lengths(gpu, dtype, log_norm):
    """Many tokens of one value near the largest length (a sum over them before the division by the weights' would
    overflow), and far below 1."""
    c = Case(64, 4, 4, heads=2, lengths=(500, 64, 3), dtype=dtype, page_size=64)
    for b, n in enumerate(c.lengths):
        v = torch.tensor(c.rng.standard_normal((1, 2, 64))).to(c.dtype).expand(n, 2, 64).contiguous()
        c.append(c.slots(b, range(n)), np.arange(n, dtype=np.int32), v=v)
        with_norms(c, b, range(n), np.full(n, 2.0 ** log_norm))
    check_weighted(c, torch.tensor(0.1 * c.rng.standard_normal((3, 4, 64))).to(c.dtype))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rising", [True, False])
def test_attend_scores_against_norms(gpu, dtype, rising):
    """Scores rise (fall) over the tokens as values get shorter (longer), so that the running maxima of the scores and of
    the products with the values come from different tokens all along."""
    n = 700
    c = Case(64, 4, 4, heads=1, lengths=(n,), dtype=dtype, page_size=64)
    t = np.arange(n) / n
    t = t if rising else t[::-1]
    k = 0.1 * torch.tensor(c.rng.standard_normal((n, 1, 64))).float()
    k[:, 0, 0] = torch.tensor(10.0 * t.copy()).float()
    c.append(c.slots(0, range(n)), np.arange(n, dtype=np.int32), k=k.to(c.dtype))
    with_norms(c, 0, range(n), 2.0 ** (-28 * t) * 2.0 ** 14)
    q = torch.zeros(1, 2, 64)
    q[:, 0, 0], q[:, 1, 0] = 16.0, 2.0
    check_weighted(c, q.to(c.dtype))


# -- codecs and reads ----------------------------------------------------------------------------------------------------

def test_codec_refuses_what_is_no_rotation(gpu):
    """Codes are exact, and read turns vectors back, for rotations (and reflections) alone."""
    _, (R, bounds, cent) = codec(64, 4)
    skew = R.copy()
    skew[3] = skew[4]
    for bad in (2 * R, 5 * np.eye(64), skew, np.zeros((64, 64)), np.full((64, 64), 1e20), R + 0.01):
        with pytest.raises(ValueError, match="rotation"):
            KVCodec(bad, bounds, cent)
    for good in (R, np.eye(64)[::-1], torch.tensor(R, device="cuda").bfloat16()):
        KVCodec(good, bounds, cent)
    KVCodec(np.array([[-1.0]]), bounds, cent)


def test_codec_keeps_its_own_tables(gpu):
    """A tensor that a codec was made of can be used for something else afterwards."""
    _, (R, bounds, cent) = codec(64, 4)
    given = [torch.tensor(x, device="cuda") for x in (R, bounds, cent)]
    cache = KVCache(KVCodec(*given), heads=1, pages=1, page_size=16)
    x = torch.randn(16, 1, 64, device="cuda")
    slots = torch.arange(16, device="cuda")
    cache.append(x, x, slots, slots.int())
    before = cache.read(slots)
    for t in given:
        t.zero_()
    for a, b in zip(cache.read(slots), before):
        assert torch.equal(a, b)


def test_codec_of_parameters(gpu):
    """Tables that require a gradient are constants to a codec."""
    _, tables = codec(64, 4)
    x = torch.randn(16, 1, 64, device="cuda")
    slots = torch.arange(16, device="cuda")
    got = []
    for t in (tables, [torch.nn.Parameter(torch.tensor(t, device="cuda")) for t in tables]):
        cache = KVCache(KVCodec(*t), heads=1, pages=1, page_size=16)
        cache.append(x, x, slots, slots.int())
        got.append(cache.read(slots)[0])
    assert not got[1].requires_grad and torch.equal(*got)


def test_scale_of_any_number(gpu):
    q, _ = codec(64, 4)
    cache = KVCache(q, heads=1, pages=1, page_size=16)
    x = torch.randn(16, 1, 64, device="cuda")
    slots = torch.arange(16, device="cuda")
    cache.append(x, x, slots, slots.int())
    table, lengths = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([16], dtype=torch.int32, device="cuda")
    got = [cache.attend(x[:1], table, lengths, scale=s) for s in (2.0, 2, np.float32(2), np.float64(2), torch.tensor(2.0))]
    assert all(torch.equal(t, got[0]) for t in got)
    for bad in (np.float32("inf"), torch.tensor(math.nan)):
        with pytest.raises(ValueError, match="scale"):
            cache.attend(x[:1], table, lengths, scale=bad)


def test_read_under_capture(gpu):
    """Reads of few and of very many rows are captured, and replayed on new contents; the many run while another stream
    turns as many rows by the encoder, in the same process and outside of the capture."""
    from polarquant_b200 import _lib
    from polarquant_b200.device import ptr, stream_ptr
    n, heads, d = 70000, 2, 16  # 140000 rows
    q, tables = codec(d, 4)
    cache = KVCache(q, heads=heads, pages=-(-n // 256), page_size=256)
    slots = torch.randperm(cache.pages * 256, device="cuda")[:n]
    few = slots[:33].clone()
    position = torch.zeros(n, dtype=torch.int32, device="cuda")
    x = [torch.randn(n, heads, d, device="cuda") for _ in range(2)]
    cache.append(x[0], x[0], slots, position)
    want = [cache.read(s, dtype=t) for s, t in ((slots, torch.float32), (few, torch.bfloat16))]
    # the encoder's own call, all of its buffers ready
    R = torch.tensor(tables[0], device="cuda").contiguous()
    nb = _lib.query("pq_rotation_planes_bytes", d)
    planes = torch.empty(nb, dtype=torch.uint8, device="cuda")
    _lib.call("pq_prepare_rotation", ptr(R), d, ptr(planes), nb, stream_ptr())
    ws = torch.empty(_lib.query("pq_encode_workspace_bytes", n * heads, d), dtype=torch.uint8, device="cuda")
    y = torch.empty_like(x[0])
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    turn = lambda: _lib.call("pq_rotate_tc", ptr(x[0]), n * heads, d, ptr(planes), ptr(y), ptr(ws), ws.numel(),  # noqa: E731
                             stream_ptr())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="relaxed"):
        got = [cache.read(slots), cache.read(few, dtype=torch.bfloat16)]
        with torch.cuda.stream(other):
            turn()
    other.synchronize()
    for new in x[::-1]:
        cache.append(new, new, slots, position)
        g.replay()
        if new is x[0]:
            for a, b in zip(got, want):
                assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        for a, (s, t) in zip(got, ((slots, torch.float32), (few, torch.bfloat16))):
            for z, eager in zip(a, cache.read(s, dtype=t)):
                assert torch.equal(z, eager)
    # the other stream's: factors of 22 bits, sums of d products in f32
    off = (y.view(-1, d).double() - x[0].view(-1, d).double() @ R.double().T).abs()
    assert (off <= (d + 2) * 2.0 ** -22 * x[0].view(-1, d).double().norm(dim=-1, keepdim=True)).all()


CONTEXTS = """
import ctypes, sys
sys.path.insert(0, {root!r})
import torch
from polarquant_b200 import _lib
rt = ctypes.CDLL("libcudart.so.12")  # torch's, loaded with it

def ok(code):
    assert code == 0, code

def device(values):
    p = ctypes.c_void_p()
    data = bytes(values)
    ok(rt.cudaMalloc(ctypes.byref(p), ctypes.c_size_t(len(data))))
    ok(rt.cudaMemcpy(p, data, ctypes.c_size_t(len(data)), 1))
    return p.value

def f32(*x):
    return bytes((ctypes.c_float * len(x))(*x))

def i32(*x):
    return bytes((ctypes.c_int32 * len(x))(*x))

d, page, pages, n = 64, 16, 320, 5000
for turn in range(2):
    eye = device(f32(*[float(i == j) for i in range(d) for j in range(d)]))
    bounds, cent = device(f32(-0.1, 0.0, 0.1)), device(f32(-0.2, -0.05, 0.05, 0.2))
    size = _lib.query("pq_kv_codec_bytes", d, 2)
    codec = device(size)
    _lib.call("pq_kv_prepare_codec", eye, bounds, cent, d, 2, codec, size, None)
    rows, norms = (device(pages * page * 16) for _ in range(2)), (device(f32(*[1.0] * (pages * page))) for _ in range(2))
    (kr, vr), (kn, vn) = rows, norms
    c = _lib.KVCacheDesc(k_rows=kr, v_rows=vr, k_norms=kn, v_norms=vn, positions=device(i32(*range(pages * page))),
                         weights=device(f32(*[float(i % 7) for i in range(pages * page)])), k_codec=codec, v_codec=codec,
                         k_ldb=16, v_ldb=16, pages=pages, heads=1, page_size=page, d=d, k_bits=2, v_bits=2)
    ref = ctypes.byref(c)
    table, lengths, slots = device(i32(*range(pages))), device(i32(n)), device(bytes((ctypes.c_int64 * n)(*range(n))))
    x, out = device(n * d * 4), device(d * 4)
    # an append of many rows, attention and an eviction: kernels of more than 48 KB of shared memory
    _lib.call("pq_kv_append", ref, x, x, 0, n, d, d, d, d, slots, device(i32(*range(n))), None, None)
    size = _lib.query("pq_kv_attend_workspace_bytes", ref, 1, 1, pages, 0)
    _lib.call("pq_kv_attend", ref, x, 0, d, d, table, pages, pages, lengths, 1, 1, 1.0, out, None, 0, device(size), size, None)
    new = device(4)
    size = _lib.query("pq_kv_evict_workspace_bytes", ref, 1, pages, 4999)
    _lib.call("pq_kv_evict", ref, table, pages, pages, lengths, 1, 4999, 0, 0, None, 0, 0, 0, new, device(size), size, None)
    left = ctypes.c_int32()
    ok(rt.cudaMemcpy(ctypes.byref(left), ctypes.c_void_p(new), ctypes.c_size_t(4), 2))
    assert left.value == 4999
    if turn == 0:
        ok(rt.cudaDeviceReset())
print("both contexts")
"""


def test_context_made_anew(gpu):
    """What a kernel is allowed in a context ends with it: calls go on in the next one."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CONTEXTS.format(root=root)], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "both contexts" in r.stdout, r.stderr
