"""Serving cases: a key and value cache in 8 bits, in pages, and what a serving step does with it.

Three operators, each through its public entry point:

  slots   `pmkl_amd.cache_slots`: from the requests' lengths and the list of free pages, the block table's new entries
          and the slot of every new token
  append  `pmkl_amd.cache_append`: the new tokens' keys and values into the cache's pages, as e4m3 codes with a
          power-of-two scale for each page and head
  attend  `pmkl_amd.cache_attn_fwd`: attention of the new tokens over their requests' pages

The cache: `k_cache` [pages, kv_heads, page, dim] and `v_cache` [pages, kv_heads, dim, page], both float8_e4m3fn, with
`k_scale` and `v_scale` [pages, kv_heads]. A request's lengths are part of its case, so that its work is known; what the
tensors hold, and which pages a request has, comes from the seed.
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
LEAST_SCALE = 2.0 ** -126

# The most that a drawn case may cost, of the largest listed ones: bytes of a cache that a decoding step reads,
# multiply-adds x 2 of a step with chunks of a prompt, bytes that an append moves.
MAX_CACHE_BYTES = 1 << 30
MAX_FLOPS = 4 * 512 * 32 * 3840 * 128 * 4
MAX_APPEND_BYTES = 8192 * 8 * 128 * 6


def _attend(name, dtype, batch, heads, kv_heads, dim, page, context, ragged=False, chunk=0, chunks=0):
    """`chunks` of the requests bring `chunk` new tokens each, the others one; contexts count the new tokens."""
    return {"name": name, "kind": "attend", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "context": context, "ragged": ragged, "chunk": chunk, "chunks": chunks}


def _append(name, dtype, batch, kv_heads, dim, page, context, new):
    """`batch` requests bring `new` tokens each to contexts of up to `context` tokens; 0: lengths from 1 to 2 pages."""
    return {"name": name, "kind": "append", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "dim": dim,
            "page": page, "context": context, "new": new}


def _slots(name, batch, page, context, new):
    return {"name": name, "kind": "slots", "batch": batch, "page": page, "context": context, "new": new}


def listed():
    return [
        # One request, one token, a short float32 context with the heads of the smallest benchmark shape: pure latency.
        _attend("attend_f32_1x128", "fp32", 1, 4, 4, 64, 16, 128),
        # One request decoding at the end of a long context, as many key heads as query heads.
        _attend("attend_bf16_1x16k", "bf16", 1, 16, 16, 128, 16, 16384),
        # A small batch decoding in a large decoder layer, four query heads to a key head.
        _attend("attend_bf16_4x4k", "bf16", 4, 32, 8, 128, 16, 4096),
        # A batch whose contexts differ widely, smaller heads, larger pages.
        _attend("attend_f16_64_ragged", "fp16", 64, 16, 4, 64, 32, 4095, ragged=True),
        # A full server: the most that a decoding step reads.
        _attend("attend_bf16_128_ragged", "bf16", 128, 32, 8, 128, 64, 16384, ragged=True),
        # Chunks of four prompts over what is cached of them: bound by the products.
        _attend("attend_bf16_chunks", "bf16", 4, 32, 8, 128, 16, 4096, chunk=512, chunks=4),
        # A step that mixes one chunk of a prompt with requests that decode.
        _attend("attend_f16_mixed", "fp16", 32, 16, 4, 64, 16, 2049, ragged=True, chunk=333, chunks=1),
        # A decoding step's tokens, one to a request, into pages that are partly filled.
        _append("append_bf16_decode", "bf16", 256, 8, 128, 16, 4096, 1),
        # Chunks of prompts: whole pages and their ends.
        _append("append_bf16_prompts", "bf16", 4, 8, 128, 16, 4096, 2048),
        # Short odd runs in float32 and large pages.
        _append("append_f32_odd", "fp32", 24, 4, 64, 64, 1000, 0),
        # The tables of a decoding step.
        _slots("slots_decode", 64, 16, 4096, 1),
        # The tables of many prompts at once.
        _slots("slots_prompts", 512, 16, 4096, 256),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choices(["attend", "append", "slots"], [0.6, 0.25, 0.15])[0]
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "slots":
        new = rng.choice([1, 1, _log_int(rng, 2, 1024)])
        return {"kind": kind, "batch": _log_int(rng, 1, min(2048, 131072 // new)), "page": page,
                "context": _log_int(rng, 1, 8192), "new": new}
    dtype = rng.choices(["fp32", "fp16", "bf16"], [0.2, 0.35, 0.45])[0]
    dim = rng.choice([32, 64, 128, 128])
    if kind == "append":
        kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
        most = MAX_APPEND_BYTES // (2 * kv_heads * dim * (DTYPES[dtype].itemsize + 1))   # tokens
        new = rng.choice([0, 1, 1, _log_int(rng, 2, min(4096, most))])
        return {"kind": kind, "dtype": dtype, "batch": _log_int(rng, 1, min(256, most // (new or 2 * page))),
                "kv_heads": kv_heads, "dim": dim, "page": page, "context": _log_int(rng, 1, 8192), "new": new}
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 16])
    group = rng.choice([1, 1, 2, 4, 4, 7, 8, 16])
    context = _log_int(rng, 16, 16384)
    most = min(256, MAX_CACHE_BYTES // (2 * context * kv_heads * dim))
    chunk = 0
    if rng.random() < 0.25:    # the plain form computes every request at the longest chunk
        pairs = MAX_FLOPS // (4 * dim * kv_heads * group * context)
        chunk = _log_int(rng, 2, min(context, 1024, pairs))
        most = min(most, pairs // chunk)
    batch = _log_int(rng, 1, most)
    return {"kind": kind, "dtype": dtype, "batch": batch, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "page": page, "context": context, "ragged": rng.random() < 0.6, "chunk": chunk,
            "chunks": rng.randint(1, batch) if chunk else 0}


def _lengths(case):
    """(tokens cached before the step, new tokens) of each request: they follow from the case alone."""
    rng = random.Random("%(kind)s %(batch)d %(context)d %(page)d" % case)
    batch, context = case["batch"], case["context"]
    if case["kind"] == "attend":
        total = [_log_int(rng, max(1, context // 32), context) if case["ragged"] else context for _ in range(batch)]
        if case["ragged"]:
            total[0] = context
        new = [min(total[b], case["chunk"]) if b < case["chunks"] else 1 for b in range(batch)]
        return [t - n for t, n in zip(total, new)], new
    new = [case["new"] or rng.randint(1, 2 * case["page"]) for _ in range(batch)]
    if case["kind"] == "slots" and case["new"] > 1:
        new = [rng.randint(0, case["new"]) for _ in range(batch)]
    return [rng.randint(0, context) for _ in range(batch)], new


def _pages(length, page):
    return -(-length // page)


def _normal(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _cache(gen, pages, kv_heads, page, dim):
    """A cache of normal keys and values: e4m3 codes under scales that put a page's largest value near 448, with pages
    whose values are a few times larger or smaller among them."""
    codes = []
    for shape in ((pages, kv_heads, page, dim), (pages, kv_heads, dim, page)):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
        codes.append(x.mul_(100.0).clamp_(-E4M3_MAX, E4M3_MAX).to(E4M3))
        del x
    steps = torch.randint(-8, -5, (2, pages, kv_heads), generator=gen, device="cuda")
    scales = torch.ldexp(torch.ones((), device="cuda"), steps)
    return {"k_cache": codes[0], "v_cache": codes[1], "k_scale": scales[0].clone(), "v_scale": scales[1].clone()}


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(lengths, page, width, order):
    """Block table [requests, width] for requests of these lengths, pages taken in `order`, -1 where there is none."""
    counts = torch.tensor([_pages(n, page) for n in lengths])
    has = torch.arange(width) < counts[:, None]
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    table[has] = order[:int(counts.sum())].to(torch.int32)
    return table.to("cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cached, new = _lengths(case)
    page, batch = case["page"], case["batch"]
    total = [c + n for c, n in zip(cached, new)]
    tokens = sum(new)
    width = max(_pages(t, page) for t in total)
    needed = sum(_pages(t, page) for t in total)
    pages = needed + 16
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    state = {"case": case, "page": page, "tokens": tokens}
    if case["kind"] == "slots":
        width += 2
        held = sum(_pages(c, page) for c in cached)
        return state | {"cached_lens": _int32(cached), "new_lens": _int32(new),
                        "block_table": _table(cached, page, width, order),
                        "free_pages": order[held:].to(torch.int32).to("cuda"), "free_head": _int32([0])}
    kv_heads, dim = case["kv_heads"], case["dim"]
    state |= _cache(gen, pages, kv_heads, page, dim)
    table = _table(total, page, width, order)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    if case["kind"] == "attend":
        return state | {"q": _normal(gen, DTYPES[case["dtype"]], tokens, case["heads"], dim), "block_table": table,
                        "seq_lens": _int32(total), "query_start": _int32(starts), "longest": max(total),
                        "most_new": max(new)}
    request = torch.repeat_interleave(torch.arange(batch), torch.tensor(new)).to("cuda")
    at = torch.arange(tokens, device="cuda") - torch.tensor(starts, device="cuda")[request]
    at += torch.tensor(cached, device="cuda")[request]
    state["slots"] = table[request, at // page].long() * page + at % page
    packed = _normal(gen, DTYPES[case["dtype"]], tokens, 3, kv_heads, dim)   # one projection's output, as layers write it
    return state | {"k": packed[:, 1], "v": packed[:, 2]}


def run(state):
    return {"slots": _run_slots, "append": _run_append, "attend": _run_attend}[state["case"]["kind"]](state)


def _run_slots(state):
    names = ("cached_lens", "new_lens", "block_table", "free_pages", "free_head")
    cached, new, table, free, head = (state[n] for n in names)
    page, tokens = state["page"], state["tokens"]
    if own:
        import pmkl_amd

        seq_lens, query_start, slots, head = pmkl_amd.cache_slots(cached, new, table, free, head, page, tokens)
    else:
        seq_lens = cached + new
        first, last = ((n + page - 1) // page for n in (cached, seq_lens))
        count = last - first
        start = head + count.cumsum(0) - count
        column = torch.arange(table.shape[1], device="cuda")
        taken = start[:, None] + column - first[:, None]
        fresh = (column >= first[:, None]) & (column < last[:, None])
        table.copy_(torch.where(fresh, free[taken.clamp(0, free.shape[0] - 1)], table))
        query_start = torch.cat([new.new_zeros(1), new.cumsum(0)]).to(torch.int32)
        token = torch.arange(tokens, device="cuda")
        request = torch.repeat_interleave(torch.arange(new.shape[0], device="cuda"), new, output_size=tokens)
        at = cached[request] + token - query_start[request]
        slots = table[request, at // page].long() * page + at % page
        head = (head + count.sum()).to(torch.int32)
    return {"seq_lens": seq_lens, "query_start": query_start, "slots": slots, "free_head": head, "block_table": table}


def _scale_for(largest):
    """The least power of two, from 2^-126 on, under which `largest` is at most 448."""
    mantissa, exponent = torch.frexp(largest.clamp(min=E4M3_MAX * LEAST_SCALE) / E4M3_MAX)
    return torch.ldexp(torch.ones_like(largest), exponent - (mantissa == 0.5).to(exponent.dtype))


def _run_append(state):
    caches = {n: state[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    if own:
        import pmkl_amd

        pmkl_amd.cache_append(state["k"], state["v"], state["slots"], **caches)
        return caches
    slot, size = state["slots"], state["page"]
    page, offset = slot // size, slot % size
    first = torch.full(caches["k_scale"].shape[:1], size, device="cuda").scatter_reduce(0, page, offset, "amin")
    old_token = torch.arange(size, device="cuda") < first[:, None]
    for name, x in (("k", state["k"]), ("v", state["v"])):
        x = x.float()
        cache, scale = caches[name + "_cache"], caches[name + "_scale"]
        largest = torch.zeros_like(scale).index_reduce(0, page, x.abs().amax(-1), "amax")
        grown = torch.maximum(torch.where(first[:, None] > 0, scale, 0.0), _scale_for(largest))
        grown = torch.where(first[:, None] < size, grown, scale)
        codes = cache.float()
        if name == "v":
            codes = codes.transpose(2, 3)
        codes = torch.where(old_token[:, None, :, None], codes * (scale / grown)[..., None, None], codes)
        codes[page, :, offset] = x / grown[page][..., None]
        cache.copy_((codes.transpose(2, 3) if name == "v" else codes).to(E4M3))
        scale.copy_(grown)
    return caches


def _gather(cache, scale, table):
    """[requests, kv_heads, pages of the table, ...] values in 32 bits."""
    codes = cache.view(torch.uint8)[table].view(E4M3).float()
    return (codes * scale[table][..., None, None]).transpose(1, 2)


def _run_attend(state):
    case = state["case"]
    q, table, seq_lens, query_start = (state[n] for n in ("q", "block_table", "seq_lens", "query_start"))
    caches = {n: state[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    if own:
        import pmkl_amd

        out, m, l = pmkl_amd.cache_attn_fwd(q, **caches, block_table=table, seq_lens=seq_lens,
                                            query_start=query_start)
        return {"out": out, "m": m, "l": l}
    tokens, heads, dim = q.shape
    batch, kv_heads, most = case["batch"], case["kv_heads"], state["most_new"]
    pages = table[:, :_pages(state["longest"], state["page"])].long().clamp(min=0)
    k = _gather(caches["k_cache"], caches["k_scale"], pages).flatten(2, 3)
    v = _gather(caches["v_cache"], caches["v_scale"], pages).transpose(3, 4).flatten(2, 3)
    new = query_start[1:] - query_start[:-1]
    token = (query_start[:-1, None] + torch.arange(most, device="cuda")).clamp(max=tokens - 1)
    rows = q.float()[token].view(batch, most, kv_heads, -1, dim).transpose(1, 2).flatten(2, 3)
    s = torch.matmul(rows, k.transpose(2, 3).contiguous()) / math.sqrt(dim)
    position = (seq_lens - new)[:, None] + torch.arange(most, device="cuda")
    seen = torch.arange(k.shape[2], device="cuda") <= torch.minimum(position, seq_lens[:, None] - 1)[..., None]
    s = s.view(batch, kv_heads, most, -1, k.shape[2]).masked_fill(~seen[:, None, :, None], -math.inf)
    m = s.amax(-1)
    p = (s - m[..., None]).exp()
    l = p.sum(-1)
    out = torch.matmul(p.flatten(2, 3), v.contiguous()).view(batch, kv_heads, most, -1, dim) / l[..., None]
    request = torch.repeat_interleave(torch.arange(batch, device="cuda"), new, output_size=tokens)
    at = torch.arange(tokens, device="cuda") - query_start[request]
    out, m, l = (x.transpose(1, 2).flatten(2, 3)[request, at] for x in (out, m, l))
    return {"out": out.to(q.dtype), "m": m, "l": l}


def work(case):
    cached, new = _lengths(case)
    tokens, page = sum(new), case["page"]
    if case["kind"] == "slots":   # lengths read, lengths and starts written, a slot for each token, the new table entries
        fresh = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
        return {"bytes": 16 * case["batch"] + 8 * tokens + 8 * fresh, "flops": 0}
    kv_heads, dim = case["kv_heads"], case["dim"]
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "append":
        return {"bytes": 2 * tokens * kv_heads * dim * (size + 1) + 8 * tokens, "flops": 0}
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, new))
    cache = sum(2 * (c + n) * kv_heads * dim + 8 * _pages(c + n, page) * kv_heads for c, n in zip(cached, new))
    return {"bytes": cache + tokens * case["heads"] * (2 * dim * size + 8), "flops": 4 * dim * case["heads"] * pairs}


def _round_e4m3(x):
    """Nearest e4m3 value of each float64 value of magnitude 448 at most, ties to even: four significant bits, from 2^-6 on
    downwards steps of 2^-9."""
    step = torch.exp2((torch.frexp(x)[1] - 4).clamp(min=-9).double())
    return torch.round(x / step) * step


def exact(case, seed):
    if case["kind"] == "slots":
        return None    # whole numbers
    state = prepare(case, seed)
    cached, new = _lengths(case)
    page = case["page"]
    result = {n: state[n].double() for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    if case["kind"] == "append":
        at = 0
        slots = state["slots"].tolist()
        while at < len(slots):
            p, first = divmod(slots[at], page)
            count = 1
            while at + count < len(slots) and slots[at + count] == slots[at] + count and first + count < page:
                count += 1
            for name in "kv":
                x = state[name][at:at + count].double()
                scale = result[name + "_scale"][p]
                need = torch.exp2(torch.ceil(torch.log2(x.abs().amax((0, 2)) / E4M3_MAX)).clamp(min=-126))
                grown = torch.maximum(scale, need) if first else need
                codes = result[name + "_cache"][p]
                codes = codes.transpose(1, 2) if name == "v" else codes
                codes[:, :first] = _round_e4m3(codes[:, :first] * (scale / grown)[:, None, None])
                codes[:, first:first + count] = _round_e4m3((x / grown[:, None]).transpose(0, 1))
                scale.copy_(grown)
            at += count
        return result
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    outs = []
    at = 0
    for b in range(case["batch"]):
        n, length = new[b], cached[b] + new[b]
        pages = state["block_table"][b, :_pages(length, page)].long()
        k = state["k_cache"].view(torch.uint8)[pages].view(E4M3).double() * result["k_scale"][pages][..., None, None]
        v = state["v_cache"].view(torch.uint8)[pages].view(E4M3).double() * result["v_scale"][pages][..., None, None]
        k = k.permute(1, 0, 2, 3).reshape(kv_heads, -1, dim)[:, :length]
        v = v.permute(1, 0, 3, 2).reshape(kv_heads, -1, dim)[:, :length]
        q = state["q"][at:at + n].double().view(n, kv_heads, heads // kv_heads, dim)
        s = torch.stack([q[:, h] @ k[h].T for h in range(kv_heads)], 1) * dim ** -0.5
        future = torch.arange(length, device="cuda") > (cached[b] + torch.arange(n, device="cuda"))[:, None]
        s.masked_fill_(future[:, None, None], -math.inf)
        m = s.amax(-1)
        p = torch.exp(s - m[..., None])
        l = p.sum(-1)
        out = torch.stack([p[:, h] @ v[h] for h in range(kv_heads)], 1) / l[..., None]
        outs.append((out.reshape(n, heads, dim), m.reshape(n, heads), l.reshape(n, heads)))
        at += n
    return dict(zip(("out", "m", "l"), (torch.cat(x) for x in zip(*outs))))
