"""Workloads of the compressed key-value cache: writing tokens into it, attending over it, evicting from it.

A cache holds, for every token and key-value head, the key and the value as packed Lloyd-Max codes of their rotated
unit vectors (the rows that Quantizer.encode writes) and an f32 norm each, in pages of `page` tokens. Here are the
cases, their inputs, the operators in plain torch, and the same results in 64 bits.
"""
import functools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # One user's next token after a short prompt: a handful of kilobytes per head, launch latency is all.
        dict(name="attend-one-short", op="attend", batch=1, heads=8, group=4, d=128, k_bits=4, v_bits=4, dtype="bf16",
             page=16, longest=1000, ragged=False, accumulate=False, lse=False),
        # One head of queries per key head, small heads, keys finer than values, a ragged batch with an empty row.
        dict(name="attend-mha-ragged", op="attend", batch=24, heads=16, group=1, d=64, k_bits=4, v_bits=2, dtype="fp16",
             page=32, longest=2049, ragged=True, accumulate=False, lse=True),
        # A serving batch that keeps score of what was attended to, for eviction.
        dict(name="attend-accumulate", op="attend", batch=16, heads=8, group=8, d=128, k_bits=4, v_bits=4, dtype="bf16",
             page=64, longest=8192, ragged=True, accumulate=True, lse=False),
        # One long document, few heads: the work has to be split over the length.
        dict(name="attend-one-long", op="attend", batch=1, heads=4, group=7, d=128, k_bits=8, v_bits=4, dtype="bf16",
             page=64, longest=131071, ragged=False, accumulate=False, lse=False),
        # Many query heads on few key heads, wide heads at two bits.
        dict(name="attend-wide-2bit", op="attend", batch=6, heads=4, group=16, d=256, k_bits=2, v_bits=2, dtype="bf16",
             page=128, longest=20011, ragged=True, accumulate=False, lse=False),
        # Full precision in and out, a head size that fills no power of two, eight bits.
        dict(name="attend-f32-odd", op="attend", batch=5, heads=3, group=5, d=80, k_bits=8, v_bits=8, dtype="f32",
             page=16, longest=4001, ragged=True, accumulate=False, lse=True),
        # The largest: a full serving batch of long contexts.
        dict(name="attend-batch-long", op="attend", batch=16, heads=8, group=4, d=128, k_bits=4, v_bits=4, dtype="bf16",
             page=64, longest=32768, ragged=True, accumulate=False, lse=False),
        # One new token of each sequence of a serving batch.
        dict(name="append-tokens", op="append", tokens=32, heads=8, d=128, k_bits=4, v_bits=4, dtype="bf16", page=64,
             padded=False),
        # A prompt chunk of full precision, padded tokens in it, odd head size.
        dict(name="append-f32-padded", op="append", tokens=1777, heads=5, d=96, k_bits=8, v_bits=2, dtype="f32", page=16,
             padded=True),
        # Prompts of a whole batch.
        dict(name="append-prompts", op="append", tokens=24576, heads=8, d=128, k_bits=4, v_bits=4, dtype="bf16", page=64,
             padded=False),
        # Generations at their budget: a page of new tokens comes in, as many of the least attended ones go.
        dict(name="evict-page", op="evict", batch=4, heads=8, d=64, k_bits=4, v_bits=4, page=64, longest=2112,
             budget=2048, recent=256, sinks=4, ragged=False, prompt=False),
        # A prompt cut down to its heavy tokens by the column sums that its attention handed over.
        dict(name="evict-prompt", op="evict", batch=6, heads=8, d=128, k_bits=4, v_bits=2, page=64, longest=65536,
             budget=4096, recent=512, sinks=4, ragged=True, prompt=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attend", "attend", "append", "evict"))
    d = rng.choice((64, 128, 128, 256, rng.randrange(16, 257)))
    bits = rng.choice(((4, 4), (4, 4), (8, 8), (2, 2), (8, 4), (4, 2), (8, 2)))
    case = dict(op=op, heads=rng.randrange(1, 17), d=d, k_bits=bits[0], v_bits=bits[1],
                page=rng.choice((16, 32, 64, 128)))
    if op == "attend":
        # Up to about the largest listed cases' codes and products.
        group = rng.choice((1, 2, 4, 5, 7, 8, 12, 16))
        case["heads"] = max(1, min(case["heads"], 64 // group))
        row = d * (bits[0] + bits[1]) / 8 + 8
        most = min(200e6 / (row * case["heads"]), 2.5e9 / (case["heads"] * group * d))
        batch = _log(rng, 1, min(64, most / 32))
        longest = _log(rng, 1, min(200000, most / batch))
        case.update(batch=batch, group=group, dtype=rng.choice(("bf16", "bf16", "fp16", "f32")), longest=max(1, longest),
                    ragged=batch > 2 and rng.random() < 0.7, accumulate=rng.random() < 0.3, lse=rng.random() < 0.3)
    elif op == "append":
        dtype = rng.choice(("bf16", "bf16", "fp16", "f32"))
        most = 24576 * 8 * 128 * (0.45 if dtype == "f32" else 0.7) / (case["heads"] * max(d, 64) * (2 if d > 128 else 1))
        case.update(tokens=_log(rng, 1, most), dtype=dtype, padded=rng.random() < 0.4)
    else:
        batch, prompt = _log(rng, 1, 8), rng.random() < 0.5
        rows = batch * case["heads"]
        longest = _log(rng, 2, min(100000, (2e6 if prompt else 8e4) / rows))
        budget = max(1, min(longest, int(longest * rng.uniform(0.02, 0.98)), int(8e4 / rows)))
        if not prompt:  # the new tokens cost as an append does
            budget = max(budget, longest - int(2e4 / rows) - 1)
        case.update(batch=batch, longest=longest, budget=budget, recent=rng.randrange(0, budget + 1) // 4,
                    sinks=min(4, budget // 2), ragged=prompt and batch > 2 and rng.random() < 0.6, prompt=prompt)
    return case


def _lengths(case):
    """The rows' lengths: all the longest, or spread below it with an empty row and a row of one token."""
    n, top = case["batch"], case["longest"]
    if not case["ragged"]:
        return [top] * n
    spread = [max(1, int(top * ((i * 0.6180339887498949) % 1.0))) for i in range(n)]
    spread[0] = top
    spread[-1] = 0
    if n > 3:
        spread[-2] = 1
    return spread


def _row_bytes(d, bits):
    return (d * bits + 7) // 8


def work(case):
    h, d = case["heads"], case["d"]
    row = _row_bytes(d, case["k_bits"]) + _row_bytes(d, case["v_bits"]) + 8  # codes and norms of one token and head
    if case["op"] == "attend":
        tokens, size, b = sum(_lengths(case)), BYTES[case["dtype"]], case["batch"]
        hq = h * case["group"]
        moved = tokens * h * (row + (8 if case["accumulate"] else 0)) + 2 * b * hq * d * size
        moved += sum(-(-n // case["page"]) for n in _lengths(case)) * 4 + 4 * b + (4 * b * hq if case["lse"] else 0)
        return {"bytes": moved, "flops": 4 * tokens * hq * d + 4 * b * hq * d * d}
    if case["op"] == "append":
        n = case["tokens"]
        rows = n * h
        # vectors in, codes, norms, position and weight out; then codes and norms in, values out
        return {"bytes": rows * (2 * row + 8 + 4 * d * BYTES[case["dtype"]]) + 16 * n, "flops": 4 * rows * d * d}
    over = [n for n in _lengths(case) if n > case["budget"]]
    scored = sum(over) * h
    moved = sum(case["budget"] * (1 - case["budget"] / n) for n in over) * h
    back = sum(min(n, case["budget"]) for n in _lengths(case)) * h
    if case["prompt"]:
        return {"bytes": int(4 * scored + moved * (2 * row + 8) + back * (row + 4 * d)), "flops": scored}
    new = sum(over) * h - case["budget"] * len(over) * h  # tokens that come in, and whose rows are moved to the holes
    return {"bytes": int(8 * scored + new * (4 * d + row + 8) + new * 2 * (row + 8) + back * (row + 4 * d)),
            "flops": scored + 4 * new * d * d}


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _levels(d, bits):
    """Lloyd-Max boundaries and centroids of a coordinate of a random unit vector, N(0, 1/d)."""
    s = 1 / math.sqrt(d)
    pdf = lambda x: torch.exp(-0.5 * (x / s) ** 2) / (s * math.sqrt(2 * math.pi))  # noqa: E731
    cdf = lambda x: 0.5 * torch.special.erfc(-x / (s * math.sqrt(2)))  # noqa: E731
    c = torch.linspace(-3 * s, 3 * s, 1 << bits, dtype=torch.float64)
    ends = torch.tensor([math.inf], dtype=torch.float64)
    for _ in range(200):
        edge = torch.cat([-ends, (c[1:] + c[:-1]) / 2, ends])
        mass = cdf(edge[1:]) - cdf(edge[:-1])
        c = torch.where(mass > 1e-15, s * s * (pdf(edge[:-1]) - pdf(edge[1:])) / mass.clamp_min(1e-300), c)
    return ((c[1:] + c[:-1]) / 2).float(), c.float()


def _codec(d, bits, gen):
    g = torch.randn(d, d, generator=gen, device="cuda", dtype=torch.float64)
    rotation, r = torch.linalg.qr(g)
    rotation = (rotation * torch.sign(torch.diagonal(r))).float().contiguous()
    boundaries, centroids = _levels(d, bits)
    return dict(rotation=rotation, boundaries=boundaries.cuda(), centroids=centroids.cuda(), bits=bits, d=d)


def _stride(d, bits):
    """Bytes from one packed row to the next."""
    return max(16, -(-_row_bytes(d, bits) // 16) * 16)


def _pack(codes, bits):
    """[..., d] codes -> packed rows of `_stride` bytes, the first code in the highest bits."""
    d = codes.shape[-1]
    per = 8 // bits
    out = torch.zeros(*codes.shape[:-1], _stride(d, bits) * per, dtype=torch.uint8, device=codes.device)
    out[..., :d] = codes
    out = out.view(*codes.shape[:-1], -1, per)
    row = out[..., 0] << (8 - bits)
    if per > 1:
        row = row | out[..., 1] << (8 - 2 * bits)
    if per > 2:
        row = row | out[..., 2] << (8 - 3 * bits) | out[..., 3]
    return row


def _random_pool(shape, codec, gen):
    """Rows as encoded random vectors have them: codes of normal coordinates."""
    rows = torch.empty(*shape, _stride(codec["d"], codec["bits"]), dtype=torch.uint8, device="cuda")
    flat, edges = rows.view(-1, rows.shape[-1]), codec["boundaries"] * math.sqrt(codec["d"])
    step = max(1, (1 << 27) // codec["d"])
    for at in range(0, flat.shape[0], step):
        part = flat[at:at + step]
        x = torch.randn(part.shape[0], codec["d"], generator=gen, device="cuda")
        part.copy_(_pack(torch.bucketize(x, edges, out_int32=True).to(torch.uint8), codec["bits"]))
    return rows


def _tables(case, gen):
    """Pages in no order, as a pool in use hands them out; entries behind a sequence's end name no page."""
    need = [-(-n // case["page"]) for n in _lengths(case)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    at = torch.tensor(need, device="cuda")
    col = torch.arange(max(1, -(-case["longest"] // case["page"])), device="cuda")
    first = torch.cumsum(at, 0) - at
    table = torch.where(col < at[:, None], order[(first[:, None] + col).clamp_max(pages - 1)], -1).to(torch.int32)
    return pages, table, torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    h, d, page = case["heads"], case["d"], case["page"]
    kc, vc = _codec(d, case["k_bits"], gen), _codec(d, case["v_bits"], gen)
    s = dict(case=case, kc=kc, vc=vc)
    if case["op"] == "append":
        n = case["tokens"]
        pages = -(-n // page) + 5
        dtype = DTYPES[case["dtype"]]
        size = torch.exp(0.4 * randn(2, n, h, 1)) * torch.tensor([1.0, 0.3], device="cuda").view(2, 1, 1, 1)
        kv = (randn(2, n, h, d) * size).to(dtype)
        slots = torch.randperm(pages, generator=gen, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
        s.update(k=kv[0], v=kv[1], slots=slots.view(-1)[:n].contiguous(),
                 positions=torch.arange(n, dtype=torch.int32, device="cuda"))
        if case["padded"]:
            s["slots"][torch.rand(n, generator=gen, device="cuda") < 0.1] = -1
        s.update(k_rows=torch.zeros(pages, h, page, _stride(d, kc["bits"]), dtype=torch.uint8, device="cuda"),
                 v_rows=torch.zeros(pages, h, page, _stride(d, vc["bits"]), dtype=torch.uint8, device="cuda"),
                 k_norms=torch.zeros(pages, h, page, device="cuda"), v_norms=torch.zeros(pages, h, page, device="cuda"),
                 cache_positions=torch.zeros(pages, h, page, dtype=torch.int32, device="cuda"),
                 weights=torch.zeros(pages, h, page, device="cuda"))
        return s
    pages, table, lengths = _tables(case, gen)
    s.update(table=table, lengths=lengths, k_rows=_random_pool((pages, h, page), kc, gen),
             v_rows=_random_pool((pages, h, page), vc, gen),
             k_norms=math.sqrt(d) * torch.exp(0.3 * randn(pages, h, page)),
             v_norms=0.3 * math.sqrt(d) * torch.exp(0.5 * randn(pages, h, page)),
             weights=torch.rand(pages, h, page, generator=gen, device="cuda") ** 8)
    where = torch.zeros(pages, page, dtype=torch.int32, device="cuda")  # each token's position, the same for all heads
    at = torch.arange(table.shape[1] * page, dtype=torch.int32, device="cuda").view(1, -1, page).expand(*table.shape, page)
    where[table[table >= 0].long()] = at[table >= 0]
    s["cache_positions"] = where[:, None].expand(pages, h, page).contiguous()
    if case["op"] == "attend":
        s["q"] = (1.5 * randn(case["batch"], h * case["group"], d)).to(DTYPES[case["dtype"]])
    else:
        s["given"] = torch.rand(case["batch"], h, case["longest"], generator=gen, device="cuda") ** 8 \
            if case["prompt"] else None
        if not case["prompt"]:
            at = torch.arange(case["budget"], case["longest"], device="cuda")
            s.update(new_slots=(table.long()[:, at // page] * page + at % page).view(-1),
                     new_positions=at.to(torch.int32).repeat(case["batch"]))
            s["k"], s["v"] = (randn(2, len(s["new_slots"]), h, d) * math.sqrt(0.3)).bfloat16()
        first = torch.arange(case["budget"], device="cuda")
        slots = table.long()[:, first // page] * page + first % page
        s["slots"] = torch.where(first < lengths[:, None], slots, -1).view(-1).contiguous()
    return s


# ---------------------------------------------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------------------------------------------

def _values(rows, norms, codec):
    """Packed rows and norms -> the vectors they stand for, in rotated coordinates."""
    d, bits = codec["d"], codec["bits"]
    rows = rows[..., :_row_bytes(d, bits)]
    if bits == 4:
        rows = torch.stack([rows >> 4, rows & 15], -1).flatten(-2)
    elif bits == 2:
        rows = torch.stack([rows >> 6, rows >> 4 & 3, rows >> 2 & 3, rows & 3], -1).flatten(-2)
    return codec["centroids"][rows[..., :d].int()] * norms[..., None]


def _encode(x, codec):
    x = x.float()
    norm = x.double().square().sum(-1).sqrt().float()
    unit = x / norm.clamp_min(1e-8)[..., None]
    turned = unit.double() @ codec["rotation"].double().T  # 64 bits: coordinates next to a boundary
    return _pack(torch.bucketize(turned, codec["boundaries"].double(), out_int32=True).to(torch.uint8), codec["bits"]), norm


def _plain_append(s, slots, positions):
    page = s["case"]["page"]
    held = slots >= 0
    slots = slots[held]
    for x, rows, norms, codec in ((s["k"], s["k_rows"], s["k_norms"], s["kc"]), (s["v"], s["v_rows"], s["v_norms"], s["vc"])):
        packed, norm = _encode(x[held], codec)
        rows[slots // page, :, slots % page] = packed
        norms[slots // page, :, slots % page] = norm
    s["cache_positions"][slots // page, :, slots % page] = positions[held][:, None]
    s["weights"][slots // page, :, slots % page] = 0


def _plain_read(s, slots, dtype):
    page, held = s["case"]["page"], (slots >= 0)[:, None, None]
    at = slots.clamp_min(0)
    k = _values(s["k_rows"][at // page, :, at % page], s["k_norms"][at // page, :, at % page], s["kc"])
    v = _values(s["v_rows"][at // page, :, at % page], s["v_norms"][at // page, :, at % page], s["vc"])
    return torch.where(held, k, 0.0).to(dtype), torch.where(held, v, 0.0).to(dtype)


def _paged(pool, table):
    """[pages, heads, page, ...] -> [batch, heads, tokens, ...]"""
    return pool[table.clamp_min(0).long()].transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    case, q, table, lengths = s["case"], s["q"], s["table"], s["lengths"]
    b, h, d = case["batch"], case["heads"], case["d"]
    turned = q.float() @ s["kc"]["rotation"].T
    k = _values(_paged(s["k_rows"], table), _paged(s["k_norms"], table), s["kc"])
    scores = turned.view(b, h, -1, d) @ k.transpose(-1, -2) / math.sqrt(d)
    del k
    inside = torch.arange(scores.shape[-1], device=q.device) < lengths[:, None, None, None]
    scores = torch.where(inside, scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    p = p / total.clamp_min(1e-30)
    lse = (top + torch.log(total)).view(b, -1)
    out = p @ _values(_paged(s["v_rows"], table), _paged(s["v_norms"], table), s["vc"])
    out = (out.view(b, -1, d) @ s["vc"]["rotation"]).to(q.dtype)
    if case["accumulate"]:
        slot = torch.arange(scores.shape[-1], device=q.device)
        page = table.clamp_min(0).long()[:, slot // case["page"]]
        s["weights"].index_put_((page[:, None], torch.arange(h, device=q.device)[None, :, None],
                                 (slot % case["page"])[None, None]), p.sum(2), accumulate=True)
    return out, lse


def _plain_evict(s):
    case, table, lengths = s["case"], s["table"].long().clamp_min(0), s["lengths"]
    page, budget, h = case["page"], case["budget"], case["heads"]
    slot = torch.arange(case["longest"], device=table.device)
    at = (table[:, slot // page][:, None], torch.arange(h, device=table.device)[None, :, None], (slot % page)[None, None])
    inside = slot < lengths[:, None, None]
    prompt = s["given"] is not None  # a prompt's tokens lie in order, with the weights that came with them
    weight = s["given"] if prompt else s["weights"][at]
    position = torch.where(inside, slot.to(torch.int32) if prompt else s["cache_positions"][at], -1)
    safe = (position < case["sinks"]) | (position > position.amax(-1, keepdim=True) - case["recent"])
    key = torch.where(inside, torch.where(safe, math.inf, weight), -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(inside.expand_as(key)).scatter(-1, order[..., :budget], True) & inside
    hole, mover = inside & ~kept & (slot < budget), kept & (slot >= budget)
    if prompt:
        held = kept & (slot < budget)
        place = [x.expand_as(key)[held] for x in at]
        s["weights"][place[0], place[1], place[2]] = weight[held]
        s["cache_positions"][place[0], place[1], place[2]] = position.expand_as(key)[held]
    to, fr = ([x.expand_as(key)[m] for x in at] for m in (hole, mover))  # the first hole takes the first mover's token
    for pool in (s["k_rows"], s["v_rows"], s["k_norms"], s["v_norms"]):
        pool[to[0], to[1], to[2]] = pool[fr[0], fr[1], fr[2]]
    s["cache_positions"][to[0], to[1], to[2]] = position.expand_as(key)[mover]
    s["weights"][to[0], to[1], to[2]] = weight[mover]
    return lengths.clamp_max(budget)


def _handle(s):
    """The cache over the buffers in `s`, as a serving program holds it from its start on."""
    if "cache" not in s:
        from polarquant_b200 import KVCache, KVCodec
        kc, vc = (KVCodec(c["rotation"], c["boundaries"], c["centroids"]) for c in (s["kc"], s["vc"]))
        s["cache"] = KVCache(kc, vc, heads=s["case"]["heads"], page_size=s["case"]["page"], buffers=dict(
            k_rows=s["k_rows"], v_rows=s["v_rows"], k_norms=s["k_norms"], v_norms=s["v_norms"],
            positions=s["cache_positions"], weights=s["weights"]))
    return s["cache"]


def run(s):
    case = s["case"]
    if case["op"] == "attend":
        if own:
            out = _handle(s).attend(s["q"], s["table"], s["lengths"], accumulate=case["accumulate"], return_lse=case["lse"])
            out, lse = out if case["lse"] else (out, None)
        else:
            out, lse = _plain_attend(s)
        return {"out": out, "lse": lse if case["lse"] else None, "weights": s["weights"] if case["accumulate"] else None}
    if case["op"] == "append":
        if own:
            cache = _handle(s)
            cache.append(s["k"], s["v"], s["slots"], s["positions"])
            k, v = cache.read(s["slots"], dtype=s["k"].dtype, rotated=True)
        else:
            _plain_append(s, s["slots"], s["positions"])
            k, v = _plain_read(s, s["slots"], s["k"].dtype)
        return {"k": k, "v": v, "k_norms": s["k_norms"], "v_norms": s["v_norms"], "positions": s["cache_positions"],
                "weights": s["weights"]}
    if own:
        cache = _handle(s)
        if not case["prompt"]:
            cache.append(s["k"], s["v"], s["new_slots"], s["new_positions"])
        lengths = cache.evict(s["table"], s["lengths"], case["budget"], recent=case["recent"], sinks=case["sinks"],
                              weights=s["given"])
        k, v = cache.read(s["slots"], dtype=torch.bfloat16, rotated=True)
    else:
        if not case["prompt"]:
            _plain_append(s, s["new_slots"], s["new_positions"])
        lengths = _plain_evict(s)
        k, v = _plain_read(s, s["slots"], torch.bfloat16)
    if not case["prompt"]:
        s["new_positions"].add_(case["longest"] - case["budget"])  # the next page's tokens
    return {"lengths": lengths, "positions": s["cache_positions"], "weights": s["weights"], "k": k, "v": v}


# ---------------------------------------------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def _exact_rows(rows, norms, codec):
    bits, per = codec["bits"], 8 // codec["bits"]
    value = torch.empty(*rows.shape[:-1], rows.shape[-1] * per, dtype=torch.float64, device=rows.device)
    for i in range(per):
        value[..., i::per] = codec["centroids"].double()[(rows >> (8 - bits * (i + 1)) & ((1 << bits) - 1)).int()]
    return value[..., :codec["d"]] * norms.double()[..., None]


def _exact_code(x, codec):
    """(values in rotated coordinates, norms) of encoded vectors."""
    norm = torch.linalg.vector_norm(x.double(), dim=-1)
    unit = (x.float() / norm.float().clamp_min(1e-8)[..., None]).double()
    turned = torch.einsum("nhi,ji->nhj", unit, codec["rotation"].double())
    code = torch.zeros_like(turned, dtype=torch.int32)
    for edge in codec["boundaries"].double():
        code += turned > edge
    return codec["centroids"].double()[code] * norm[..., None], norm


def exact(case, seed):
    s = prepare(case, seed)
    h, d, page = case["heads"], case["d"], case["page"]
    if case["op"] == "append":
        result, there = {}, s["slots"] >= 0
        for name, codec in (("k", s["kc"]), ("v", s["vc"])):
            value, norm = _exact_code(s[name], codec)
            norms = torch.zeros_like(s["k_norms"], dtype=torch.float64).transpose(1, 2).reshape(-1, h)
            norms[s["slots"][there]] = norm[there]
            result[name] = value * there[:, None, None]
            result[name + "_norms"] = norms.view(-1, page, h).transpose(1, 2).contiguous()
        return {**result, "positions": None, "weights": torch.zeros_like(s["weights"], dtype=torch.float64)}
    if case["op"] == "attend":
        outs, lses, weights = [], [], s["weights"].double()
        for b, n in enumerate(_lengths(case)):
            turned = s["q"][b].double().view(h, -1, d) @ s["kc"]["rotation"].double().T
            pages = s["table"][b, :-(-n // page)].long()
            rows = lambda x: x[pages].transpose(0, 1).flatten(1, 2)[:, :n]  # noqa: E731, B023
            scores = turned @ _exact_rows(rows(s["k_rows"]), rows(s["k_norms"]), s["kc"]).mT / d ** 0.5
            p = torch.softmax(scores, -1) if n else scores
            out = p @ _exact_rows(rows(s["v_rows"]), rows(s["v_norms"]), s["vc"])
            outs.append(out.reshape(-1, d) @ s["vc"]["rotation"].double())
            lses.append(torch.logsumexp(scores, -1).flatten() if n else torch.full((h * case["group"],), -math.inf,
                                                                                   dtype=torch.float64, device="cuda"))
            if case["accumulate"] and n:
                more = torch.zeros(h, len(pages) * page, dtype=torch.float64, device="cuda")
                more[:, :n] = p.sum(1)
                weights[pages] += more.view(h, -1, page).transpose(0, 1)
        return {"out": torch.stack(outs), "lse": torch.stack(lses) if case["lse"] else None,
                "weights": weights if case["accumulate"] else None}
    budget, positions, weights = case["budget"], s["cache_positions"].clone(), s["weights"].double()
    new = {}
    if not case["prompt"]:
        at = (s["new_slots"] // page, slice(None), s["new_slots"] % page)
        positions[at], weights[at] = s["new_positions"][:, None], 0
        new = {n: _exact_code(s[n], s[n + "c"])[0].view(case["batch"], -1, h, d) for n in "kv"}
    back = {n: torch.zeros(case["batch"], budget, h, d, dtype=torch.float64, device="cuda") for n in "kv"}
    for b, n in enumerate(_lengths(case)):
        slot = torch.arange(n, device="cuda")
        pg, off = s["table"][b].long()[slot // page], slot % page
        for j in range(h):
            weight = s["given"][b, j, :n].double() if case["prompt"] else weights[pg, j, off]
            source = slot[:budget].clone()
            if n > budget:
                where = slot if case["prompt"] else positions[pg, j, off]
                safe = (where < case["sinks"]) | (where > int(where.max()) - case["recent"])
                order = torch.argsort(torch.where(safe, math.inf, weight), descending=True, stable=True)
                kept = torch.zeros(n, dtype=torch.bool, device="cuda")
                kept[order[:budget]] = True
                source[~kept[:budget]] = slot[budget:][kept[budget:]]
            weights[pg[:budget], j, off[:budget]] = weight[source]
            for name in "kv":
                back[name][b, :len(source), j] = _exact_rows(s[name + "_rows"][pg[source], j, off[source]],
                                                             s[name + "_norms"][pg[source], j, off[source]], s[name + "c"])
                if new:
                    fresh = source >= budget
                    back[name][b, fresh.nonzero()[:, 0], j] = new[name][b, source[fresh] - budget, j]
    return {"lengths": None, "positions": None, "weights": weights, "k": back["k"].view(-1, h, d), "v": back["v"].view(-1, h, d)}
