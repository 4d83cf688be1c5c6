"""The compressed key-value cache on the GPU against the oracle's statement of it in 64 bits.

Codes, positions, lengths and moved rows have to be equal.  Attention is held to a bound made of the roundings that
the kernel makes: with 16-bit queries, factors of 11 bits (centroids and softmax weights; half a step is 2^-11 of
the value), with f32 queries factors of 22 bits and sums in f32.
"""
import math

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from polarquant_b200 import KVCache, KVCodec, Quantizer

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODECS = {}


def codec(d, bits, seed=42):
    if (d, bits, seed) not in CODECS:
        q = Quantizer(d, bits=bits, seed=seed)
        CODECS[d, bits, seed] = (q, (q.R, q.boundaries, q.centroids))
    return CODECS[d, bits, seed]


class Case:
    """A cache and its oracle with the same contents: random tokens on shuffled pages."""

    def __init__(self, d=64, k_bits=4, v_bits=4, heads=2, page_size=16, lengths=(33,), dtype="bf16", seed=0, spare=2,
                 slack=0):
        self.rng = np.random.default_rng(seed)
        self.d, self.heads, self.page, self.dtype = d, heads, page_size, TYPES[dtype]
        kq, self.kc = codec(d, k_bits)
        vq, self.vc = codec(d, v_bits, 43)
        need = [-(-n // page_size) + slack for n in lengths]
        self.pages = sum(need) + spare
        self.cache = KVCache(kq, vq, heads=heads, pages=self.pages, page_size=page_size)
        order = self.rng.permutation(self.pages)
        self.table = np.full((len(lengths), max(1, max(need, default=1))), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.lengths = np.array(lengths, np.int32)
        self.ref = O.empty(self.pages, heads, page_size, d)
        slots = np.concatenate([self.slots(b, range(n)) for b, n in enumerate(lengths)]).astype(np.int64)
        positions = np.concatenate([np.arange(n) for n in lengths]).astype(np.int32)
        if len(slots):
            self.append(slots, positions, weights=self.rng.random((len(slots), heads), np.float32))

    def slots(self, b, tokens):
        t = np.array(tokens, np.int64)
        return self.table[b, t // self.page].astype(np.int64) * self.page + t % self.page

    def vectors(self, n, size=1.0):
        x = self.rng.standard_normal((n, self.heads, self.d)) * np.exp(0.4 * self.rng.standard_normal((n, self.heads, 1)))
        return torch.tensor(size * x).to(self.dtype)

    def append(self, slots, positions, weights=None, k=None, v=None):
        k = self.vectors(len(slots)) if k is None else k
        v = self.vectors(len(slots), 0.5) if v is None else v
        self.cache.append(k.cuda(), v.cuda(), torch.tensor(slots).cuda(), torch.tensor(positions).cuda(),
                          None if weights is None else torch.tensor(weights).cuda())
        O.append(self.ref, self.kc, self.vc, k.float().numpy(), v.float().numpy(), slots, positions, weights)

    def on_gpu(self):
        return torch.tensor(self.table).cuda(), torch.tensor(self.lengths).cuda()

    def check_pool(self, weights=True):
        """Everything the pool holds, bit for bit."""
        every = torch.arange(self.pages * self.page).cuda()
        k, v = self.cache.read(every, rotated=True)
        rk, rv = O.values(self.ref, self.kc, self.vc, every.cpu().numpy())
        np.testing.assert_array_equal(k.cpu().numpy(), rk)
        np.testing.assert_array_equal(v.cpu().numpy(), rv)
        for name in ("k_norms", "v_norms", "positions") + (("weights",) if weights else ()):
            np.testing.assert_array_equal(getattr(self.cache, name).cpu().numpy(), self.ref[name])

    def check_attend(self, group=2, scale=None, accumulate=False, q=None, size=1.0, **kw):
        batch = len(self.lengths)
        if q is None:
            q = torch.tensor(size * self.rng.standard_normal((batch, self.heads * group, self.d))).to(self.dtype)
        table, lengths = self.on_gpu()
        before = self.ref["weights"].astype(np.float64)
        out, lse = self.cache.attend(q.cuda(), table, lengths, scale=scale, accumulate=accumulate, return_lse=True)
        assert out.dtype == self.dtype and out.shape == q.shape
        s = 1 / math.sqrt(self.d) if scale is None else scale
        ref, rlse, sizes = O.attend(self.ref, self.kc, self.vc, q.double().numpy(), self.table, self.lengths, s, accumulate)
        check_attention(out, lse, ref, rlse, sizes, self.dtype, self.d)
        if accumulate:
            more = self.ref["weights"] - before
            err = np.abs(self.cache.weights.cpu().numpy() - before - more)
            grow = score_error(sizes, self.dtype, self.d).max(initial=0)
            # a weight is off by its score's error and the sums' own: 2^-20 of what was added, 2^-23 of the sum
            assert (err <= more * (np.expm1(2 * grow) + 2.0 ** -20) + 2.0 ** -23 * (before + more)).all(), err.max()
            self.ref["weights"] = self.cache.weights.cpu().numpy()
        return out, lse


def score_error(sizes, dtype, d):
    """Bound on a score's error, from the sum of its terms' absolute values: a centroid off by half a step, and the sum
    in f32 with at most d/16 + 8 roundings of the products' matrix sums, the rotation's d roundings and the norm's."""
    half = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
    return sizes[..., 0] * (half + (2 * d + 16) * 2.0 ** -24)


def check_attention(out, lse, ref, rlse, sizes, dtype, d):
    half = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
    ds = score_error(sizes, dtype, d)
    lse, out = lse.double().cpu().numpy(), out.double().cpu().numpy()
    none = np.isneginf(rlse)
    assert (np.isneginf(lse) == none).all()
    off = np.abs(lse[~none] - rlse[~none])
    assert (off <= ds[~none] + 2.0 ** -20 + 2.0 ** -22 * np.abs(rlse[~none])).all()
    assert not out[none].any()
    # weights off by the scores' error and a rounding, values by a centroid's; sums in f32, turned back in f32;
    # then the type's rounding of each element
    bound = sizes[..., 1] * (np.expm1(2 * ds) + 2 * half + (4 * d + 64) * 2.0 ** -24)
    bound = bound + np.sqrt((ref ** 2).sum(-1)) * torch.finfo(dtype).eps / 2 + math.sqrt(d) * torch.finfo(dtype).tiny
    off = np.sqrt(((out - ref) ** 2).sum(-1))
    assert (off <= bound).all(), (off / bound).max()


# -- append and read ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,k_bits,v_bits", [(64, 4, 4), (128, 4, 2), (128, 8, 8), (80, 8, 4), (256, 2, 2), (1, 4, 2),
                                             (37, 2, 8), (255, 4, 4), (96, 2, 4)])
def test_append_and_read(gpu, d, k_bits, v_bits, dtype):
    c = Case(d, k_bits, v_bits, heads=3, lengths=(1, 37), dtype=dtype)
    c.check_pool()


def test_codes_next_to_boundaries(gpu):
    """Many rows at eight bits: every code equals the exact product's."""
    c = Case(128, 8, 8, heads=8, lengths=(4096,), page_size=256, dtype="bf16")
    c.check_pool()


def test_codes_are_the_quantizers(gpu):
    """append writes the rows that Quantizer.encode gives for the same vectors."""
    q, _ = codec(96, 4)
    x = np.random.default_rng(5).standard_normal((200, 96)).astype(np.float32)
    cache = KVCache(q, heads=1, pages=4, page_size=64)
    t = torch.tensor(x).cuda()[:, None]
    cache.append(t, t, torch.arange(200).cuda(), torch.arange(200, dtype=torch.int32).cuda())
    cv = q.encode(x)
    np.testing.assert_array_equal(cache.k_rows.view(256, -1)[:200, :48].cpu().numpy(), cv._device().rows_host())
    np.testing.assert_array_equal(cache.k_norms.view(-1)[:200].cpu().numpy(), cv.norms)
    back = cache.read(torch.arange(200).cuda())[0][:, 0].cpu().numpy()
    # two products of 22-bit factors and f32 sums, each within d + 2 roundings of the vector's size
    bound = 2 * (96 + 2) * 2.0 ** -22 * cv.norms[:, None]
    assert (np.abs(back - q.decode(cv)) <= bound).all()


def test_append_skips_and_overwrites(gpu):
    c = Case(64, 4, 4, lengths=(40,))
    slots = np.array([-1, c.slots(0, [3])[0], c.pages * 16, 1 << 40, c.slots(0, [39])[0], -(1 << 40)])
    c.append(slots, np.arange(6, dtype=np.int32) + 100)
    c.check_pool()


def test_append_strides(gpu):
    """Keys and values as views of one projection's output, at addresses of odd alignment, and expanded heads."""
    c = Case(64, 4, 4, heads=2, lengths=(32,))
    wide = torch.randn(5, 7, 200, dtype=torch.bfloat16)
    k, v = wide[:, 1:3, 3:67], wide[:, 4:6, 100:164]
    slots = c.slots(0, [0, 5, 9, 17, 31])
    table, lengths = c.on_gpu()
    g = wide.cuda()
    c.cache.append(g[:, 1:3, 3:67], g[:, 4:6, 100:164], torch.tensor(slots).cuda(),
                   torch.arange(5, dtype=torch.int32).cuda())
    O.append(c.ref, c.kc, c.vc, k.float().numpy(), v.float().numpy(), slots, np.arange(5))
    c.check_pool()
    one = torch.randn(3, 1, 64)
    c.cache.append(one.cuda().expand(3, 2, 64), one.cuda().expand(3, 2, 64), torch.tensor(slots[:3]).cuda(),
                   torch.arange(3, dtype=torch.int32).cuda())
    O.append(c.ref, c.kc, c.vc, one.expand(3, 2, 64).numpy(), one.expand(3, 2, 64).numpy(), slots[:3], np.arange(3))
    c.check_pool()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_zero_tiny_and_large_vectors(gpu, dtype):
    c = Case(64, 4, 4, heads=1, lengths=(16,), dtype=dtype)
    k = torch.randn(6, 1, 64).to(TYPES[dtype])
    k[0] = 0
    k[1] *= 1e-12
    k[2] *= 1e-30
    k[3] *= 1e15
    k[4] = 0
    k[4, 0, 7] = 3
    k[5, 0, 1:] *= 1e-6
    c.append(c.slots(0, range(6)), np.arange(6, dtype=np.int32), k=k, v=k.flip(0))
    c.check_pool()


def test_large_append(gpu):
    c = Case(128, 4, 4, heads=8, page_size=64, lengths=(700, 1, 0, 333), dtype="bf16")
    c.check_pool()


def encoded(x, R, boundaries):
    """Codes and norms of vectors on the GPU, the product in 64 bits."""
    x = x.float()
    norms = x.double().square().sum(-1).sqrt().float()
    unit = x / norms.clamp_min(1e-8)[..., None]
    R, edges = (torch.tensor(t, device="cuda").double() for t in (R, boundaries))
    turned = torch.cat([u.double() @ R.T for u in unit.flatten(0, 1).split(100000)])
    return torch.bucketize(turned, edges, out_int32=True).view(x.shape), norms


def check_rows(cache, codecs, k, v, slots):
    """Codes (as values) and norms of tokens that were appended in order."""
    page = cache.page_size
    got = cache.read(slots, rotated=True)
    for x, y, codec, norms in ((k, got[0], codecs[0], cache.k_norms), (v, got[1], codecs[1], cache.v_norms)):
        code, norm = encoded(x, codec[0], codec[1])
        assert torch.equal(norms[slots // page, :, slots % page], norm)
        assert torch.equal(y, torch.tensor(codec[2], device="cuda")[code] * norm[..., None])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,k_bits,v_bits", [(64, 4, 8), (128, 4, 4), (128, 8, 2), (256, 4, 8), (256, 2, 2), (96, 8, 4),
                                             (40, 4, 4), (200, 8, 8), (131, 4, 2), (7, 8, 8), (1, 2, 4)])
def test_append_many_rows(gpu, d, k_bits, v_bits, dtype):
    """Calls of many rows (more than 16 a multiprocessor) take another kernel than those of few."""
    (kq, kc), (vq, vc) = codec(d, k_bits), codec(d, v_bits, 43)
    n, heads = 1201, 5
    cache = KVCache(kq, vq, heads=heads, pages=1500 // 16, page_size=16)
    gen = torch.Generator(device="cuda").manual_seed(d)
    k, v = (torch.randn(2, n, heads, d, generator=gen, device="cuda") * 3).to(TYPES[dtype])
    k[5], v[17, 2] = 0, 0
    slots = torch.randperm(1500 // 16 * 16, generator=gen, device="cuda")[:n]
    before = [t.clone() for t in (cache.k_rows, cache.v_rows)]
    cache.append(k, v, slots, torch.arange(n, dtype=torch.int32, device="cuda"))
    check_rows(cache, (kc, vc), k, v, slots)
    assert torch.equal(cache.positions[slots // 16, :, slots % 16], torch.arange(n, dtype=torch.int32, device="cuda")[:, None].expand(n, heads))
    # rows of no token are as they were, and what is behind a row's codes is 0
    rest = torch.ones(cache.pages * 16, dtype=torch.bool, device="cuda")
    rest[slots] = False
    for t, b, bits in ((cache.k_rows, before[0], k_bits), (cache.v_rows, before[1], v_bits)):
        t, b = (x.transpose(1, 2).reshape(cache.pages * 16, heads, -1) for x in (t, b))
        assert torch.equal(t[rest], b[rest])
        used, odd = d * bits // 8, d * bits % 8
        assert not t[..., used + (odd > 0):].any()
        assert not odd or not (t[..., used] & (255 >> odd)).any()


def test_append_many_rows_strided_and_padded(gpu):
    (kq, kc), (vq, vc) = codec(64, 4), codec(64, 4, 43)
    cache = KVCache(kq, vq, heads=4, pages=100, page_size=16)
    wide = torch.randn(1000, 9, 150, device="cuda").bfloat16()
    for k, v in ((wide[:, 1:5, 3:67], wide[:, 5:9, 80:144]), (wide[:, :4, 64:128], wide[:, ::2, :64][:, :4])):
        slots = torch.randperm(1600, device="cuda")[:1000]
        slots[::7] = -1
        slots[3::7] = 1600
        cache.append(k, v, slots, torch.zeros(1000, dtype=torch.int32, device="cuda"))
        ok = (slots >= 0) & (slots < 1600)
        check_rows(cache, (kc, vc), k[ok], v[ok], slots[ok])


def test_append_of_zero_vectors_and_boundary_values(gpu):
    """Vectors all of whose coordinates are next to boundaries: more than a block lists."""
    d = 64
    q, c = codec(d, 4)
    R = c[0].astype(np.float64)
    heads, n = 8, 2000
    cache = KVCache(q, heads=heads, pages=n // 16 + 1, page_size=16)
    rng = np.random.default_rng(0)
    # unit vectors whose rotated coordinates are boundaries, up to the last, which makes the length 1
    edges = np.sort(np.abs(c[1][c[1] != 0]))
    y = rng.choice(edges[: len(edges) // 2], (n * heads, d)) * rng.choice([-1, 1], (n * heads, d))
    y[:, -1] = 0
    scale = 0.999 / np.maximum(np.linalg.norm(y, axis=1, keepdims=True), 0.999)
    y *= scale
    y[:, -1] = np.sqrt(np.maximum(0, 1 - (y ** 2).sum(1)))
    k = torch.tensor((y @ R).reshape(n, heads, d)).float().cuda()
    v = torch.zeros_like(k)
    slots = torch.arange(n, device="cuda")
    cache.append(k, v, slots, torch.zeros(n, dtype=torch.int32, device="cuda"))
    check_rows(cache, (c, c), k, v, slots)


@pytest.mark.parametrize("dtype,d,bits", [("bf16", 128, 8), ("f16", 256, 4), ("f32", 128, 2), ("bf16", 64, 8), ("f32", 256, 8),
                                          ("bf16", 80, 4)])
def test_append_of_equal_rows_on_boundaries(gpu, dtype, d, bits):
    """Many equal rows, the boundaries next to their own coordinates: a block's list is full after a few of them."""
    R = codec(d, 4)[1][0]
    rng = np.random.default_rng(d + bits)
    x = torch.tensor(rng.standard_normal((2, d))).to(TYPES[dtype])
    u = x.float().numpy()
    u = u / np.sqrt((u.astype(np.float64) ** 2).sum(-1, keepdims=True)).astype(np.float32)
    y = np.sort((u.astype(np.float64) @ R.astype(np.float64).T).ravel())
    levels = 1 << bits
    bounds = np.concatenate([y, np.linspace(y[-1] + 0.01, y[-1] + 0.5, levels)]) if len(y) < levels - 1 else y
    bounds = np.sort(rng.permutation(bounds)[: levels - 1]).astype(np.float32)
    c = (R, bounds, np.linspace(-1, 1, levels, dtype=np.float32))
    n, heads = 400, 8
    cache = KVCache(KVCodec(*c), heads=heads, pages=n // 16, page_size=16)
    k, v = (r.expand(n, heads, d).contiguous().cuda() for r in x)
    slots = torch.arange(n, device="cuda")
    cache.append(k, v, slots, torch.zeros(n, dtype=torch.int32, device="cuda"))
    check_rows(cache, (c, c), k, v, slots)


def test_append_in_several_launches(gpu):
    """More rows than one launch of the append of many rows takes."""
    q, c = codec(64, 8)
    n, heads = 60000, 8
    cache = KVCache(q, heads=heads, pages=n // 64 + 1, page_size=64)
    k, v = torch.randn(2, n, heads, 64, device="cuda").half()
    slots = torch.arange(n, device="cuda")
    cache.append(k, v, slots, torch.zeros(n, dtype=torch.int32, device="cuda"))
    check_rows(cache, (c, c), k, v, slots)


def test_codec_of_odd_tables(gpu):
    """Boundaries that coincide, or lie closer than the kernels' tables resolve."""
    d = 64
    R = codec(d, 4)[1][0]
    for edges in (np.zeros(15), np.repeat([-0.1, 0.0, 0.1], 5), np.linspace(-1e-4, 1e-4, 15),
                  np.r_[-1e30, np.linspace(-0.2, 0.2, 13), 1e30], np.r_[np.full(14, -0.0), 0.05]):
        c = (R, edges.astype(np.float32), np.linspace(-1, 1, 16).astype(np.float32))
        cache = KVCache(KVCodec(*c), heads=4, pages=100, page_size=16)
        for n in (3, 1500):
            k, v = torch.randn(2, n, 4, d, device="cuda")
            k[0] = 0
            slots = torch.arange(n, device="cuda")
            cache.append(k, v, slots, torch.zeros(n, dtype=torch.int32, device="cuda"))
            check_rows(cache, (c, c), k, v, slots)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_read_types(gpu, dtype):
    c = Case(80, 4, 8, lengths=(20,))
    slots = torch.tensor([5, -1, 3, 10 ** 9]).cuda()
    k, v = c.cache.read(slots, dtype=TYPES[dtype], rotated=True)
    rk, rv = O.values(c.ref, c.kc, c.vc, slots.cpu().numpy())
    assert torch.equal(k.cpu(), torch.tensor(rk).to(TYPES[dtype])) and torch.equal(v.cpu(), torch.tensor(rv).to(TYPES[dtype]))
    k, v = c.cache.read(slots, dtype=TYPES[dtype])
    rk, rv = O.values(c.ref, c.kc, c.vc, slots.cpu().numpy(), rotated=False)
    for x, r in ((k, rk), (v, rv)):
        size = np.sqrt((r ** 2).sum(-1, keepdims=True))
        bound = size * (80 + 2) * 2.0 ** -22 + np.abs(r) * torch.finfo(TYPES[dtype]).eps / 2 * (1 + 2.0 ** -10) \
            + torch.finfo(TYPES[dtype]).tiny
        assert (np.abs(x.double().cpu().numpy() - r) <= bound).all()


# -- attend ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k_bits", [2, 4, 8])
@pytest.mark.parametrize("v_bits", [2, 4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_bits(gpu, d, k_bits, v_bits, dtype):
    c = Case(d, k_bits, v_bits, heads=2, lengths=(70, 1, 0, 300), dtype=dtype, page_size=32)
    c.check_attend(group=3)


@pytest.mark.parametrize("d", [1, 8, 31, 63, 65, 80, 96, 100, 112, 127, 129, 160, 192, 250])
def test_attend_head_sizes(gpu, d):
    for dtype in ("f32", "bf16"):
        Case(d, 4, 8, heads=1, lengths=(45, 0, 16), dtype=dtype).check_attend(group=2)


@pytest.mark.parametrize("group", [1, 2, 5, 7, 8, 9, 12, 16, 17, 32, 71])
def test_attend_groups(gpu, group):
    for dtype in ("f32", "f16"):
        Case(64, 4, 2, heads=2, lengths=(50, 400, 0), dtype=dtype).check_attend(group=group)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1025, 2049])
def test_attend_lengths(gpu, n):
    Case(64, 4, 4, heads=1, lengths=(n,), page_size=16, slack=1).check_attend(group=4)
    Case(64, 4, 4, heads=2, lengths=(n, n - 1, 3), page_size=128, dtype="f16").check_attend(group=1)


@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256, 512, 1024])
def test_attend_pages(gpu, page_size):
    Case(128, 4, 4, heads=2, lengths=(page_size * 2 + 5, page_size, page_size - 1, 0, 1), page_size=page_size).check_attend()


def test_attend_many_short(gpu):
    rng = np.random.default_rng(3)
    Case(64, 4, 4, heads=4, lengths=tuple(rng.integers(0, 90, 120)), page_size=16).check_attend(group=2)


def test_attend_one_long(gpu):
    Case(64, 4, 4, heads=2, lengths=(40001,), page_size=64, dtype="f16").check_attend(group=2)


def test_attend_empty_batch_and_all_empty(gpu):
    c = Case(64, lengths=(0, 0))
    out, lse = c.check_attend()
    assert not out.any() and torch.isneginf(lse).all()
    table, lengths = c.on_gpu()
    out = c.cache.attend(torch.zeros(0, 2, 64, device="cuda"), table[:0], lengths[:0])
    assert out.shape == (0, 2, 64)
    none = KVCache(codec(64, 4)[0], heads=1, pages=0)
    out, lse = none.attend(torch.randn(2, 3, 64, device="cuda"), torch.zeros(2, 0, dtype=torch.int32, device="cuda"),
                           torch.tensor([0, 7], dtype=torch.int32, device="cuda"), return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_concentrated_and_flat(gpu, dtype):
    """Scores hundreds apart in both directions, and all equal."""
    c = Case(128, 4, 4, heads=2, lengths=(300, 17), dtype=dtype)
    c.check_attend(size=30.0)
    c.check_attend(scale=-0.5)
    c.check_attend(scale=0.0)
    q = torch.zeros(2, 4, 128, dtype=c.dtype)
    c.check_attend(q=q)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_growing_scores(gpu, dtype):
    """The running maximum rises at almost every token, slowly and by leaps; values' norms span many octaves."""
    for step in (0.05, 3.0):
        c = Case(64, 4, 4, heads=1, lengths=(400,), dtype=dtype, page_size=64)
        q = torch.zeros(1, 2, 64)
        q[:, 0, 0], q[:, 1, 0] = 4.0, -4.0
        k = torch.zeros(400, 1, 64)
        k[:, 0, 0] = torch.arange(400) * step
        v = c.vectors(400) * torch.exp(4 * torch.randn(400, 1, 1))
        c.append(c.slots(0, range(400)), np.arange(400, dtype=np.int32), k=k.to(c.dtype), v=v.to(c.dtype))
        c.check_attend(q=q.to(c.dtype), group=2)


def test_attend_stale_slots_and_bad_pages(gpu):
    """What lies behind a sequence's end is not read into it, whatever it is; tokens on pages outside the pool are not there."""
    c = Case(64, 4, 4, heads=2, lengths=(21, 40), page_size=16, slack=1)
    for name in ("k_norms", "v_norms"):
        pool = getattr(c.cache, name)
        for b, n in enumerate(c.lengths):
            for t in range(n, c.table.shape[1] * 16):
                pg = c.table[b, t // 16]
                if pg >= 0:
                    pool[int(pg), :, t % 16] = float("nan") if t % 2 else float("inf")
    c.check_attend()
    for bad in (-1, c.pages, 2 ** 31 - 1, -2 ** 31):
        c.table[1, 1] = bad
        c.check_attend()
    c.table[0, :] = -7
    c.check_attend()
    c.lengths[:] = (2 ** 31 - 1, -5)
    c.table[0] = c.table[0].max()
    q = torch.randn(2, 2, 64, device="cuda")
    out, lse = c.cache.attend(q, *c.on_gpu(), return_lse=True)
    assert torch.isneginf(lse).all() and not out.any()


def test_attend_strides(gpu):
    c = Case(64, 4, 4, heads=2, lengths=(33, 70))
    wide = torch.randn(2, 9, 100, dtype=torch.bfloat16)
    q = wide[:, 1:9:2, 3:67]
    table, lengths = c.on_gpu()
    tw = torch.full((4, table.shape[1] + 3), 10 ** 6, dtype=torch.int32, device="cuda")
    tw[::2, 1:-2] = table
    out, lse = c.cache.attend(wide.cuda()[:, 1:9:2, 3:67], tw[::2, 1:-2], lengths, return_lse=True)
    ref, rlse, sizes = O.attend(c.ref, c.kc, c.vc, q.double().numpy(), c.table, c.lengths, 1 / 8)
    check_attention(out, lse, ref, rlse, sizes, torch.bfloat16, 64)
    one = torch.randn(1, 1, 64, dtype=torch.bfloat16)
    out, lse = c.cache.attend(one.cuda().expand(2, 4, 64), table, lengths, return_lse=True)
    ref, rlse, sizes = O.attend(c.ref, c.kc, c.vc, one.expand(2, 4, 64).double().numpy(), c.table, c.lengths, 1 / 8)
    check_attention(out, lse, ref, rlse, sizes, torch.bfloat16, 64)


@pytest.mark.parametrize("dtype,d,bits,heads,lengths", [("f16", 242, 2, 3, (4000, 37)), ("f16", 64, 8, 8, (1700,)),
                                                        ("f16", 128, 4, 2, (9, 300)), ("f32", 167, 4, 4, (3500,)),
                                                        ("f32", 64, 8, 8, (30000,)), ("f32", 128, 2, 3, (1633, 5))])
def test_attend_whole_error(gpu, dtype, d, bits, heads, lengths):
    """The error over all outputs.  f16: the output's own rounding, at most 2^-11 of an element and 0.42 times that in
    the mean, leaves no room for another of 11 bits (tokens share the centroids, so theirs would not average).  f32:
    three roundings (2^-24) of scores in units of log 2, of up to 11 here, 2^-22 of an exponential and of each pair of
    factors: 2^-19 if all had one sign, and no drift over thousands of sums."""
    c = Case(d, bits, bits, heads=heads, lengths=lengths, page_size=64, dtype=dtype)
    q = torch.tensor(1.5 * c.rng.standard_normal((len(lengths), heads * 2, d))).to(c.dtype)
    out = c.cache.attend(q.cuda(), *c.on_gpu()).double().cpu().numpy()
    ref, _, _ = O.attend(c.ref, c.kc, c.vc, q.double().numpy(), c.table, c.lengths, 1 / math.sqrt(d), False)
    assert np.sqrt(((out - ref) ** 2).sum() / (ref ** 2).sum()) <= (2.0 ** -11 if dtype == "f16" else 2.0 ** -19)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [1, 3, 8, 11])
def test_accumulate(gpu, dtype, group):
    c = Case(64, 4, 4, heads=2, lengths=(70, 0, 1, 600), page_size=16, dtype=dtype)
    c.check_attend(group=group, accumulate=True)
    c.check_attend(group=group, accumulate=True)


def test_accumulate_shared_pages(gpu):
    """Two sequences on the same pages: each adds its own."""
    c = Case(64, 4, 4, heads=1, lengths=(40,))
    c.table, c.lengths = np.repeat(c.table, 3, 0), np.array([40, 16, 25], np.int32)
    c.check_attend(accumulate=True)


def test_same_call_same_bits(gpu):
    c = Case(128, 4, 4, heads=4, lengths=(5000, 77, 900), page_size=64)
    q = torch.randn(3, 16, 128, device="cuda").bfloat16()
    table, lengths = c.on_gpu()
    a, la = c.cache.attend(q, table, lengths, return_lse=True)
    for _ in range(5):
        b, lb = c.cache.attend(q, table, lengths, return_lse=True)
        assert torch.equal(a, b) and torch.equal(la, lb)
    # a longer table, another batch order: the same sums of the same tokens up to the kernel's own roundings
    out, _ = c.cache.attend(q.flip(0), table.flip(0), lengths.flip(0), return_lse=True)
    assert (out.flip(0).float() - a.float()).abs().max() <= 2 ** -7 * a.float().abs().max()


# -- evict -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("lengths,budget", [((50,), 20), ((50, 20, 19, 21, 0, 1), 20), ((300, 1000), 1), ((33,), 0),
                                            ((64, 65), 64), ((2000, 40), 1900), ((5000,), 77)])
def test_evict(gpu, lengths, budget, prompt):
    c = Case(64, 4, 2, heads=3, lengths=lengths, page_size=16)
    w = c.rng.random((len(lengths), 3, max(lengths)), np.float32) if prompt else None
    for recent, sinks in ((0, 0), (budget // 3, min(2, budget // 2))):
        new = c.cache.evict(*c.on_gpu(), budget, recent=recent, sinks=sinks,
                            weights=None if w is None else torch.tensor(w).cuda())
        ref = O.evict(c.ref, c.table, c.lengths, budget, recent, sinks, w)
        assert new.dtype == torch.int32
        np.testing.assert_array_equal(new.cpu().numpy(), ref)
        c.check_pool()


def test_evict_ties_and_odd_weights(gpu):
    c = Case(32, 4, 4, heads=4, lengths=(200,), page_size=16)
    w = c.ref["weights"]
    pg, off, _ = O.sequence(c.ref, c.table[0], 200)
    w[pg, 0, off] = 1.0
    w[pg, 1, off] = np.where(np.arange(200) % 3 == 0, 0.0, -0.0)
    w[pg, 2, off] = np.array([np.nan, np.inf, -np.inf, 1e-45, -1e-45, 3.0, 3.0, np.float32(3e38)])[np.arange(200) % 8]
    w[pg, 3, off] = -c.rng.random(200)
    c.cache.weights.copy_(torch.tensor(w))
    new = c.cache.evict(*c.on_gpu(), 90, recent=7, sinks=3)
    np.testing.assert_array_equal(new.cpu().numpy(), O.evict(c.ref, c.table, c.lengths, 90, 7, 3))
    c.check_pool()


def test_evict_more_protected_than_budget(gpu):
    c = Case(32, 4, 4, heads=2, lengths=(100, 40), page_size=16)
    new = c.cache.evict(*c.on_gpu(), 10, recent=60, sinks=30)
    np.testing.assert_array_equal(new.cpu().numpy(), O.evict(c.ref, c.table, c.lengths, 10, 60, 30))
    c.check_pool()
    new = c.cache.evict(*c.on_gpu(), 9, recent=2 ** 31 - 1, sinks=2 ** 31 - 1)
    np.testing.assert_array_equal(new.cpu().numpy(), O.evict(c.ref, c.table, c.lengths, 9, 2 ** 31 - 1, 2 ** 31 - 1))
    c.check_pool()


def test_evict_long(gpu):
    c = Case(16, 4, 4, heads=1, lengths=(70001, 3), page_size=256)
    new = c.cache.evict(*c.on_gpu(), 9000, recent=500, sinks=4)
    np.testing.assert_array_equal(new.cpu().numpy(), O.evict(c.ref, c.table, c.lengths, 9000, 500, 4))
    c.check_pool()


@pytest.mark.parametrize("prompt", [False, True])
def test_evict_many_rows(gpu, prompt):
    """More heads than clusters fit on the device, of lengths that one block's shared memory just holds, and a longer one."""
    c = Case(16, 2, 2, heads=57, lengths=(9000, 7000), page_size=256)
    w = c.rng.random((2, 57, 9000), np.float32) if prompt else None
    for n in (9000, 5000):
        c.lengths[0] = n
        new = c.cache.evict(*c.on_gpu(), 4500, recent=300, sinks=4, weights=None if w is None else torch.tensor(w).cuda())
        np.testing.assert_array_equal(new.cpu().numpy(), O.evict(c.ref, c.table, c.lengths, 4500, 300, 4, w))
        c.lengths = new.cpu().numpy()
        c.check_pool()


def test_evict_bad_pages(gpu):
    """Tokens on pages outside the pool count as the lightest; other pages' tokens stay whole."""
    c = Case(32, 4, 4, heads=2, lengths=(64, 32), page_size=16)
    c.table[0, 3] = c.pages + 5
    c.cache.evict(*c.on_gpu(), 48)
    c.check_pool()  # the 48 tokens before the budget are all that exist
    before = {n: getattr(c.cache, n).clone() for n in ("k_rows", "v_rows", "k_norms", "v_norms", "positions", "weights")}
    c.table[0, 0] = -3
    new = c.cache.evict(*c.on_gpu(), 48)
    assert new.tolist() == [48, 32]
    for n, t in before.items():
        assert torch.equal(t, getattr(c.cache, n))


# -- together ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_generation(gpu, dtype):
    """Prompts, then steps of append, attend with accumulation, eviction at the budget and attention over what is left."""
    c = Case(64, 4, 4, heads=2, lengths=(60, 9, 30), page_size=16, dtype=dtype, slack=4)
    budget, position = 32, np.array([60, 9, 30], np.int32)
    for step in range(12):
        slots = np.array([c.slots(b, [n])[0] for b, n in enumerate(c.lengths)])
        c.append(slots, position)
        c.lengths += 1
        position += 1
        c.check_attend(group=2, accumulate=True)
        if step % 3 == 2:
            new = c.cache.evict(*c.on_gpu(), budget, recent=8, sinks=2)
            np.testing.assert_array_equal(new.cpu().numpy(), O.evict(c.ref, c.table, c.lengths, budget, 8, 2))
            c.lengths = new.cpu().numpy()
            c.check_pool()


def test_graph(gpu):
    """A decoding step captured once and replayed as the sequences grow, next to another graph and eager calls."""
    c = Case(64, 4, 4, heads=2, lengths=(40, 7), page_size=16, slack=2)
    d = Case(64, 4, 4, heads=2, lengths=(300,), page_size=16, seed=9)
    table, lengths = c.on_gpu()
    td, ld = d.on_gpu()
    k, v, q = (torch.zeros(2, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    qd = torch.randn(1, 2, 64, device="cuda").bfloat16()
    slots = torch.zeros(2, dtype=torch.int64, device="cuda")
    position = torch.zeros(2, dtype=torch.int32, device="cuda")

    def step():
        c.cache.append(k, v, slots, position)
        return c.cache.attend(q, table, lengths, accumulate=True)

    other = lambda: d.cache.attend(qd, td, ld)  # noqa: E731
    eager = other()
    slots.fill_(-1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        other()
    torch.cuda.current_stream().wait_stream(side)
    c.ref["weights"] = c.cache.weights.cpu().numpy()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out = step()
    with torch.cuda.graph(g2):
        out2 = other()
    for i in range(4):
        kn, vn, qn = c.vectors(2), c.vectors(2), c.vectors(2)
        new = np.array([c.slots(b, [n])[0] for b, n in enumerate(c.lengths)])
        O.append(c.ref, c.kc, c.vc, kn.float().numpy(), vn.float().numpy(), new, c.lengths.copy())
        for t, x in ((k, kn), (v, vn), (q, qn), (slots, torch.tensor(new)), (position, torch.tensor(c.lengths))):
            t.copy_(x)
        c.lengths += 1
        lengths.copy_(torch.tensor(c.lengths))
        g1.replay()
        g2.replay()
        ref, rlse, sizes = O.attend(c.ref, c.kc, c.vc, qn.double().numpy(), c.table, c.lengths, 1 / 8, accumulate=True)
        lse = torch.tensor(rlse)
        check_attention(out, lse, ref, rlse, sizes, torch.bfloat16, 64)
        assert torch.equal(out2, eager) and torch.equal(other(), eager)
        c.ref["weights"] = c.cache.weights.cpu().numpy()


def test_graph_of_eviction(gpu):
    c = Case(64, 4, 4, heads=2, lengths=(90, 30), page_size=16)
    table, lengths = c.on_gpu()
    g = torch.cuda.CUDAGraph()
    state = {n: getattr(c.cache, n).clone() for n in ("k_rows", "v_rows", "k_norms", "v_norms", "positions", "weights")}
    c.cache.evict(table, lengths, 25, recent=4)
    with torch.cuda.graph(g):
        new = c.cache.evict(table, lengths, 25, recent=4)
    for n, t in state.items():
        getattr(c.cache, n).copy_(t)
    g.replay()
    np.testing.assert_array_equal(new.cpu().numpy(), O.evict(c.ref, c.table, c.lengths, 25, 4))
    c.check_pool()


def test_streams(gpu):
    """Two streams attend over one cache at the same time."""
    c = Case(128, 4, 4, heads=4, lengths=(3000, 1200), page_size=64)
    q = torch.randn(2, 16, 128, device="cuda").bfloat16()
    table, lengths = c.on_gpu()
    want = [c.cache.attend(x, table, lengths) for x in (q, -q)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, (s, x) in enumerate(zip(streams, (q, -q))):
            with torch.cuda.stream(s):
                got[i].append(c.cache.attend(x, table, lengths))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_buffers(gpu):
    """A pool of the caller's own, saved and taken up again by another cache."""
    c = Case(64, 4, 2, heads=2, lengths=(50,))
    names = ("k_rows", "v_rows", "k_norms", "v_norms", "positions", "weights")
    copy = {n: getattr(c.cache, n).clone() for n in names}
    other = KVCache(KVCodec(*c.kc), KVCodec(*c.vc), heads=2, page_size=16, buffers=copy)
    assert other.pages == c.pages and other.nbytes == c.cache.nbytes
    table, lengths = c.on_gpu()
    q = torch.randn(1, 4, 64, device="cuda")
    assert torch.equal(other.attend(q, table, lengths), c.cache.attend(q, table, lengths))
    assert other.k_rows.data_ptr() == copy["k_rows"].data_ptr()


def test_quality(gpu):
    """Attention over eight bits is near attention over the vectors themselves: eight-bit codes carry a vector to
    about 1 % (their mean squared error at 256 levels is below 1e-4 of its square)."""
    c = Case(128, 8, 8, heads=1, lengths=(200,), dtype="f32")
    k, v = c.vectors(200), c.vectors(200)
    c.append(c.slots(0, range(200)), np.arange(200, dtype=np.int32), k=k, v=v)
    q = c.vectors(1)
    table, lengths = c.on_gpu()
    out = c.cache.attend(q.cuda(), table, lengths).cpu().double()[0, 0]
    p = torch.softmax(k[:, 0].double() @ q[0, 0].double() / math.sqrt(128), 0)
    want = p @ v[:, 0].double()
    assert (out - want).norm() <= 0.05 * want.norm()


# -- refusals --------------------------------------------------------------------------------------------------------------

def test_refusals(gpu):
    c = Case(64, 4, 4, heads=2, lengths=(20, 3))
    cache = c.cache
    table, lengths = c.on_gpu()
    q = torch.zeros(2, 4, 64, device="cuda")
    k = torch.zeros(3, 2, 64, device="cuda")
    slots, pos = torch.arange(3, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    bad = [
        lambda: cache.attend(q.cpu(), table, lengths), lambda: cache.attend(q[:1], table, lengths),
        lambda: cache.attend(q[:, :3], table, lengths), lambda: cache.attend(q[..., :63], table, lengths),
        lambda: cache.attend(q[:, :0], table, lengths), lambda: cache.attend(q[0], table, lengths),
        lambda: cache.attend(q.mT.contiguous().mT, table, lengths), lambda: cache.attend(q, table.cpu(), lengths),
        lambda: cache.attend(q, table, lengths[:1]), lambda: cache.attend(q, table[0], lengths),
        lambda: cache.attend(q, table.t().contiguous().t(), lengths), lambda: cache.attend(q, table, lengths, scale=math.inf),
        lambda: cache.attend(q, table, lengths, scale=math.nan), lambda: cache.attend(q.requires_grad_(), table, lengths),
        lambda: cache.append(k, k[:2], slots, pos), lambda: cache.append(k, k, slots[:2], pos),
        lambda: cache.append(k, k, slots, pos[:2]), lambda: cache.append(k[:, :1], k[:, :1], slots, pos),
        lambda: cache.append(k, k, slots[None], pos), lambda: cache.append(k, k, slots, pos, torch.zeros(3, 1, device="cuda")),
        lambda: cache.append(k.cpu(), k, slots, pos), lambda: cache.append(k, k, slots.cpu(), pos),
        lambda: cache.append(k, k, slots, torch.zeros(6, dtype=torch.int32, device="cuda")[::2]),
        lambda: cache.read(slots[None]), lambda: cache.read(torch.arange(6, device="cuda")[::2]),
        lambda: cache.evict(table, lengths, -1), lambda: cache.evict(table, lengths, 2.5),
        lambda: cache.evict(table, lengths, 1, recent=-1), lambda: cache.evict(table, lengths, 1, sinks=1 << 31),
        lambda: cache.evict(table, lengths, 1, weights=torch.zeros(2, 2, device="cuda")),
        lambda: cache.evict(table, lengths, 1, weights=torch.zeros(2, 3, 9, device="cuda")),
        lambda: cache.evict(table, lengths, 1, weights=torch.zeros(2, 2, 9, device="cpu")),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    for i, f in enumerate([
        lambda: cache.attend(q.double(), table, lengths), lambda: cache.attend(q, table.long(), lengths),
        lambda: cache.attend(q, table, lengths.long()), lambda: cache.append(k.double(), k.double(), slots, pos),
        lambda: cache.append(k, k.half(), slots, pos), lambda: cache.append(k, k, slots.int(), pos),
        lambda: cache.append(k, k, slots, pos.long()), lambda: cache.read(slots, dtype=torch.float64),
        lambda: cache.read(slots.int()), lambda: cache.append(k, k, slots, pos, torch.zeros(3, 2, device="cuda").half()),
        lambda: cache.evict(table, lengths, 1, weights=torch.zeros(2, 2, 9, device="cuda").half()),
    ]):
        with pytest.raises(TypeError):
            f()
            pytest.fail(f"call {i} was not refused")
    kc = cache.key
    for f in (lambda: KVCache(kc, heads=0, pages=1), lambda: KVCache(kc, heads=1, pages=-1), lambda: KVCache(kc, heads=1),
              lambda: KVCache(kc, heads=1, pages=1, page_size=24), lambda: KVCache(kc, heads=1, pages=1, page_size=8),
              lambda: KVCache(kc, heads=1, pages=1, page_size=2048), lambda: KVCache(kc, codec(32, 4)[0], heads=1, pages=1),
              lambda: KVCache(Quantizer(64, bits=3), heads=1, pages=1), lambda: KVCache(Quantizer(64, bits=1), heads=1, pages=1),
              lambda: KVCache(kc, heads=1, pages=1 << 27, page_size=16), lambda: KVCache(kc, heads=2, page_size=16, buffers={}),
              lambda: KVCache(kc, heads=2, page_size=16, buffers={"k_rows": cache.k_rows}),
              lambda: KVCodec(np.eye(257), np.zeros(15), np.zeros(16)), lambda: KVCodec(np.eye(4), np.zeros(15), np.zeros(8)),
              lambda: KVCodec(np.eye(4), np.arange(14), np.zeros(16)), lambda: KVCodec(np.eye(4), -np.arange(15), np.zeros(16)),
              lambda: KVCodec(np.zeros((3, 4)), np.arange(15), np.zeros(16))):
        with pytest.raises(ValueError):
            f()
            pytest.fail("was not refused")
    with pytest.raises(TypeError):
        KVCache(codec(64, 4)[1], heads=1, pages=1)
    c.check_pool()
