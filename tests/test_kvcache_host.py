"""Host-side checks of the key-value cache that need no GPU: the C ABI's refusals and sizes, and the oracle's own."""
import ctypes

import numpy as np
import pytest

from oracle import kv_oracle as O


@pytest.fixture(scope="module")
def lib():
    from polarquant_b200 import build, _lib
    build.build()
    return _lib.load()


def desc(**kw):
    from polarquant_b200 import _lib
    p = 4096
    f = dict(k_rows=p, v_rows=p, k_norms=p, v_norms=p, positions=p, weights=p, k_codec=p, v_codec=p, k_ldb=32, v_ldb=32,
             pages=4, heads=2, page_size=16, d=64, k_bits=4, v_bits=4)
    f.update(kw)
    return _lib.KVCacheDesc(**f)


BAD_CACHES = [
    (dict(d=0), b"d must"), (dict(d=257), b"d must"), (dict(k_bits=3), b"bits"), (dict(v_bits=1), b"bits"),
    (dict(heads=0), b"heads"), (dict(pages=-1), b"pages"), (dict(page_size=24), b"page_size"), (dict(page_size=8), b"page_size"),
    (dict(page_size=2048), b"page_size"), (dict(pages=1 << 27), b"2^31"), (dict(pages=1 << 20, heads=1 << 12), b"2^31"),
    (dict(k_ldb=24), b"ldb"), (dict(v_ldb=16), b"ldb"), (dict(k_ldb=48), b"ldb"), (dict(pages=1 << 20, heads=1 << 8), b"2^32"), (dict(k_codec=0), b"codec"), (dict(k_rows=0), b"pool"),
    (dict(weights=0), b"pool"), (dict(v_rows=4100), b"aligned"),
]


@pytest.mark.parametrize("kw,word", BAD_CACHES)
def test_abi_refuses_bad_caches(lib, kw, word):
    c = ctypes.byref(desc(**kw))
    for rc in (lib.pq_kv_append(c, 16, 16, 0, 1, 1, 1, 1, 1, 16, 16, 0, None), lib.pq_kv_read(c, 16, 1, 16, 16, 0, None),
               lib.pq_kv_attend(c, 16, 0, 1, 1, 16, 4, 4, 16, 1, 2, 1.0, 16, 0, 0, 16, 1 << 30, None),
               lib.pq_kv_evict(c, 16, 4, 4, 16, 1, 5, 0, 0, 0, 0, 0, 0, 16, 16, 1 << 30, None)):
        assert rc == -1 and word in lib.pq_last_error()
    assert lib.pq_kv_append(None, 16, 16, 0, 1, 1, 1, 1, 1, 16, 16, 0, None) == -1


def test_abi_refuses_bad_arguments(lib):
    c = ctypes.byref(desc())
    big = 1 << 30
    bad = [
        (lib.pq_kv_append, (c, 16, 16, 3, 1, 1, 1, 1, 1, 16, 16, 0, None), b"dtype"),
        (lib.pq_kv_append, (c, 16, 16, 0, -1, 1, 1, 1, 1, 16, 16, 0, None), b"rows"),
        (lib.pq_kv_append, (c, 16, 16, 0, 1 << 30, 1, 1, 1, 1, 16, 16, 0, None), b"rows"),
        (lib.pq_kv_append, (c, 0, 16, 0, 1, 1, 1, 1, 1, 16, 16, 0, None), b"null"),
        (lib.pq_kv_append, (c, 16, 16, 0, 1, 1, 1, 1, 1, 0, 16, 0, None), b"null"),
        (lib.pq_kv_read, (c, 16, 1, 16, 16, -1, None), b"dtype"),
        (lib.pq_kv_read, (c, 0, 1, 16, 16, 0, None), b"null"),
        (lib.pq_kv_attend, (c, 16, 9, 1, 1, 16, 4, 4, 16, 1, 2, 1.0, 16, 0, 0, 16, big, None), b"dtype"),
        (lib.pq_kv_attend, (c, 16, 0, 1, 1, 16, 4, 4, 16, 1, 3, 1.0, 16, 0, 0, 16, big, None), b"q_heads"),
        (lib.pq_kv_attend, (c, 16, 0, 1, 1, 16, 4, 4, 16, 1, 0, 1.0, 16, 0, 0, 16, big, None), b"q_heads"),
        (lib.pq_kv_attend, (c, 16, 0, 1, 1, 16, 4, 4, 16, -1, 2, 1.0, 16, 0, 0, 16, big, None), b"batch"),
        (lib.pq_kv_attend, (c, 16, 0, 1, 1, 0, 4, 4, 16, 1, 2, 1.0, 16, 0, 0, 16, big, None), b"null"),
        (lib.pq_kv_attend, (c, 16, 0, 1, 1, 16, 4, 4, 0, 1, 2, 1.0, 16, 0, 0, 16, big, None), b"null"),
        (lib.pq_kv_attend, (c, 16, 0, 1, 1, 16, 4, 4, 16, 1, 2, float("nan"), 16, 0, 0, 16, big, None), b"finite"),
        (lib.pq_kv_attend, (c, 16, 0, 1, 1, 16, 4, -1, 16, 1, 2, 1.0, 16, 0, 0, 16, big, None), b"2^30"),
        (lib.pq_kv_attend, (c, 16, 0, 1, 1, 16, 4, 1 << 27, 16, 1, 2, 1.0, 16, 0, 0, 16, big, None), b"2^30"),
        (lib.pq_kv_attend, (c, 16, 0, 1, 1, 16, 4, 1 << 26, 16, 64, 32, 1.0, 16, 0, 0, 16, big, None), b"2^31"),
        (lib.pq_kv_evict, (c, 16, 4, 4, 16, 1, -1, 0, 0, 0, 0, 0, 0, 16, 16, big, None), b"budget"),
        (lib.pq_kv_evict, (c, 16, 4, 4, 16, 1, 5, -1, 0, 0, 0, 0, 0, 16, 16, big, None), b"recent"),
        (lib.pq_kv_evict, (c, 16, 4, 4, 16, 1, 5, 0, 0, 16, 0, 0, -1, 16, 16, big, None), b"prompt_width"),
        (lib.pq_kv_evict, (c, 16, 4, 4, 16, 1, 5, 0, 0, 0, 0, 0, 0, 0, 16, big, None), b"null"),
        (lib.pq_kv_prepare_codec, (16, 16, 16, 300, 4, 16, big, None), b"d must"),
        (lib.pq_kv_prepare_codec, (16, 16, 16, 64, 3, 16, big, None), b"bits"),
        (lib.pq_kv_prepare_codec, (0, 16, 16, 64, 4, 16, big, None), b"null"),
    ]
    for f, args, word in bad:
        assert f(*args) == -1 and word in lib.pq_last_error(), (f, args, lib.pq_last_error())
    assert lib.pq_kv_prepare_codec(16, 16, 16, 64, 4, 16, 8, None) == -3
    for ws, n in ((0, big), (16, 8)):
        assert lib.pq_kv_attend(c, 16, 0, 1, 1, 16, 4, 4, 16, 1, 2, 1.0, 16, 0, 0, ws, n, None) == -3
        assert lib.pq_kv_evict(c, 16, 4, 4, 16, 1, 5, 0, 0, 0, 0, 0, 0, 16, ws, n, None) == -3


def test_abi_takes_empty_calls(lib):
    c = ctypes.byref(desc(pages=0, k_rows=0, v_rows=0, k_norms=0, v_norms=0, positions=0, weights=0))
    assert lib.pq_kv_append(c, 0, 0, 0, 0, 1, 1, 1, 1, 0, 0, 0, None) == 0
    assert lib.pq_kv_read(c, 0, 0, 0, 0, 0, None) == 0
    assert lib.pq_kv_attend(c, 0, 0, 1, 1, 16, 4, 4, 16, 0, 2, 1.0, 0, 0, 0, 0, 0, None) == 0
    assert lib.pq_kv_evict(c, 16, 4, 4, 16, 0, 5, 0, 0, 0, 0, 0, 0, 0, 0, 0, None) == 0


def test_workspaces_grow_with_the_call(lib):
    c = ctypes.byref(desc())
    small = lib.pq_kv_attend_workspace_bytes(c, 1, 2, 4, 0)
    assert 0 < small < lib.pq_kv_attend_workspace_bytes(c, 1, 2, 4, 1)
    assert lib.pq_kv_attend_workspace_bytes(c, 64, 32, 4096, 1) >= 64 * 32 * 4096 * 16 * 4
    # holes and movers: at most the smaller of the budget and what may lie behind it, twice, a sequence and head
    assert lib.pq_kv_evict_workspace_bytes(c, 3, 100, 500) >= 3 * 2 * 2 * 500 * 4
    assert lib.pq_kv_evict_workspace_bytes(c, 3, 100, 1600) < 1 << 12
    assert lib.pq_kv_codec_bytes(64, 3) == 0 and lib.pq_kv_codec_bytes(300, 4) == 0
    assert lib.pq_kv_codec_bytes(64, 4) >= 2 * 64 * 64 * 4


def test_oracle_attends_as_softmax_attention():
    """The oracle against attention over the vectors that its codes stand for, written out in model coordinates."""
    from polarquant_b200 import Quantizer
    rng = np.random.default_rng(0)
    kq, vq = Quantizer(32, bits=4), Quantizer(32, bits=2, seed=7)
    kc, vc = (kq.R, kq.boundaries, kq.centroids), (vq.R, vq.boundaries, vq.centroids)
    cache = O.empty(4, 2, 16, 32)
    k, v = rng.standard_normal((2, 20, 2, 32)).astype(np.float32)
    slots = np.array([3 * 16 + i if i < 16 else 16 + i - 16 for i in range(20)])
    O.append(cache, kc, vc, k, v, slots, np.arange(20))
    q = rng.standard_normal((1, 4, 32))
    out, lse, _ = O.attend(cache, kc, vc, q, np.array([[3, 1]]), [20], 0.3)
    kh, vh = O.values(cache, kc, vc, slots, rotated=False)
    # values() rounds each product to f32 (2^-24), and R's f32 entries leave R R^T off the identity by at most
    # sqrt(32) 2^-24 < 6 * 2^-24: scores agree within 8 * 2^-24 of |q||k| scale, weights within twice that, values
    # within 8 * 2^-24 of their size
    for h in range(4):
        keys, vals = kh[:, h // 2], vh[:, h // 2]
        s = 0.3 * keys @ q[0, h]
        p = np.exp(s - s.max())
        off = 0.3 * np.linalg.norm(q[0, h]) * np.linalg.norm(keys, axis=1).max() * 8 * 2.0 ** -24
        size = np.linalg.norm(vals, axis=1).max()
        assert np.linalg.norm(out[0, h] - p @ vals / p.sum()) <= size * (2 * off + 8 * 2.0 ** -24)
        assert abs(lse[0, h] - np.log(np.exp(s).sum())) <= off


def test_oracle_evicts_by_weight():
    cache = O.empty(2, 1, 16, 4)
    cache["weights"][0, 0, :6] = [5, 1, 4, 0, 3, 9]
    cache["positions"][0, 0, :6] = [0, 1, 2, 3, 4, 5]
    new = O.evict(cache, np.array([[0]]), [6], 3)
    assert new.tolist() == [3]
    assert cache["positions"][0, 0, :3].tolist() == [0, 5, 2]  # token 5 into token 1's place
    new = O.evict(cache, np.array([[0]]), [3], 2, recent=1, sinks=1)
    assert sorted(cache["positions"][0, 0, :2].tolist()) == [0, 5]


def test_types_and_sizes_are_the_headers():
    from polarquant_b200 import _lib
    assert ctypes.sizeof(_lib.KVCacheDesc) == 8 * 8 + 2 * 8 + 6 * 4


@pytest.mark.parametrize("lengths,new,batch", [(4096, 4096, 1), (4096, 4100, 2), (4100, 4096, 2), (4096, 4096 + 4 * 9, 10)])
def test_evict_refuses_new_lengths_over_lengths(lib, lengths, new, batch):
    """Blocks of one sequence's heads read its length while one of them writes the new one."""
    c = ctypes.byref(desc())
    assert lib.pq_kv_evict(c, 16, 4, 4, lengths, batch, 5, 0, 0, 0, 0, 0, 0, new, 1 << 16, 1 << 30, None) == -1
    assert b"overlap" in lib.pq_last_error()
