"""The compressed key-value cache's operators from their definitions, in NumPy and 64 bits.

A cache is a dict of arrays: ``k_codes`` / ``v_codes`` (pages, heads, page_size, d) uint8, ``k_norms`` /
``v_norms`` f32, ``positions`` int32 and ``weights`` f32 (pages, heads, page_size).  A codec is
(R, boundaries, centroids).  Sequences are given by a page table and lengths, as the package takes them.
"""
import numpy as np


def empty(pages, heads, page_size, d):
    pool = (pages, heads, page_size)
    return {"k_codes": np.zeros(pool + (d,), np.uint8), "v_codes": np.zeros(pool + (d,), np.uint8),
            "k_norms": np.zeros(pool, np.float32), "v_norms": np.zeros(pool, np.float32),
            "positions": np.zeros(pool, np.int32), "weights": np.zeros(pool, np.float32)}


def encode(x, codec):
    """(codes, norms) of vectors along the last axis: Quantizer.encode with the product in f64."""
    R, boundaries, _ = codec
    x = np.asarray(x, np.float32)
    norms = np.sqrt((x.astype(np.float64) ** 2).sum(-1)).astype(np.float32)
    unit = x / np.maximum(norms, np.float32(1e-8))[..., None]
    turned = unit.astype(np.float64) @ R.astype(np.float64).T
    return np.searchsorted(boundaries.astype(np.float64), turned).astype(np.uint8), norms


def append(cache, kc, vc, k, v, slots, positions, weights=None):
    page = cache["positions"].shape[2]
    for i, slot in enumerate(np.asarray(slots)):
        if not 0 <= slot < cache["positions"].shape[0] * page:
            continue
        at = (slot // page, slice(None), slot % page)
        for name, x, codec in (("k", k, kc), ("v", v, vc)):
            cache[name + "_codes"][at], cache[name + "_norms"][at] = encode(x[i], codec)
        cache["positions"][at] = positions[i]
        cache["weights"][at] = 0 if weights is None else weights[i]


def sequence(cache, table, length):
    """(pages, offsets) of a sequence's tokens that lie on a page of the pool, and their indices."""
    pages, _, page = cache["positions"].shape
    t = np.arange(max(0, min(int(length), len(table) * page)))
    pg = np.asarray(table)[t // page]
    ok = (pg >= 0) & (pg < pages)
    return pg[ok], (t % page)[ok], t[ok]


def attend(cache, kc, vc, q, table, lengths, scale, accumulate=False):
    """out (f64), lse (f64), and for every row what its error bounds go by: the largest sum of the scores' absolute
    terms and the largest value norm."""
    q = np.asarray(q, np.float64)
    batch, hq, d = q.shape
    heads = cache["positions"].shape[1]
    group = hq // heads
    out, lse = np.zeros((batch, hq, d)), np.full((batch, hq), -np.inf)
    size = np.zeros((batch, hq, 2))
    weights = cache["weights"].astype(np.float64)
    for b in range(batch):
        pg, off, _ = sequence(cache, table[b], lengths[b])
        if not len(pg):
            continue
        for h in range(hq):
            j = h // group
            kh = kc[2].astype(np.float64)[cache["k_codes"][pg, j, off]] * cache["k_norms"][pg, j, off].astype(np.float64)[:, None]
            vh = vc[2].astype(np.float64)[cache["v_codes"][pg, j, off]] * cache["v_norms"][pg, j, off].astype(np.float64)[:, None]
            turned = kc[0].astype(np.float64) @ q[b, h]
            s = scale * (kh @ turned)
            m = s.max()
            p = np.exp(s - m)
            lse[b, h] = m + np.log(p.sum())
            p /= p.sum()
            out[b, h] = (p @ vh) @ vc[0].astype(np.float64)
            size[b, h] = abs(scale) * (np.abs(kh) @ np.abs(turned)).max(), np.sqrt((vh ** 2).sum(-1)).max()
            if accumulate:
                np.add.at(weights, (pg, j, off), p)
    if accumulate:
        cache["weights"] = weights
    return out, lse, size


def evict(cache, table, lengths, budget, recent=0, sinks=0, prompt=None):
    """New lengths; the cache is changed in place."""
    heads, page = cache["positions"].shape[1:]
    new = []
    for b, length in enumerate(lengths):
        length = max(0, min(int(length), len(table[b]) * page))
        new.append(min(length, budget))
        pg, off, tok = sequence(cache, table[b], length)  # the tokens that are there
        for h in range(heads):
            at = (pg, h, off)
            w = (cache["weights"][at] if prompt is None else prompt[b, h, tok]).astype(np.float32).copy()
            pos = cache["positions"][at].copy() if prompt is None else tok.astype(np.int32)
            first = tok < budget  # places that the kept tokens take
            source = np.arange(first.sum())
            if length > budget and len(source):
                last = int(pos.max()) if prompt is None else length - 1
                safe = (pos < sinks) | (pos.astype(np.int64) > last - recent)
                nan = np.isnan(w)
                order = np.lexsort((tok, -np.where(nan | safe, 0, w), nan & ~safe, ~safe))
                kept = np.zeros(len(tok), bool)
                kept[order[:len(source)]] = True
                source[~kept[first]] = np.flatnonzero(kept & ~first)
            to, fr = (pg[:len(source)], h, off[:len(source)]), (pg[source], h, off[source])
            for name in ("k_codes", "v_codes", "k_norms", "v_norms"):
                cache[name][to] = cache[name][fr].copy()
            cache["positions"][to], cache["weights"][to] = pos[source], w[source]
    return np.array(new, np.int32)


def values(cache, kc, vc, slots, rotated=True):
    """(k, v) f32 vectors of slots: norm * centroid, in rotated coordinates or turned back (then f64)."""
    pages, _, page = cache["positions"].shape
    slots = np.asarray(slots)
    ok = (slots >= 0) & (slots < pages * page)
    at = (np.where(ok, slots, 0) // page, slice(None), np.where(ok, slots, 0) % page)
    result = []
    for name, codec in (("k", kc), ("v", vc)):
        x = codec[2][cache[name + "_codes"][at]] * cache[name + "_norms"][at][..., None] * ok[:, None, None].astype(np.float32)
        result.append(x if rotated else x.astype(np.float64) @ codec[0].astype(np.float64))
    return result
