"""Operators of a paged cache of bounded size, in their plain form and as calls of this package.

A case is a dict of plain values; ``op`` names the operator:

  sinks    attention in which a query sees the last ``window`` keys and the first ``sinks``
           ones, over the paged cache: rows of one token, or of a chunk of tokens
  weights  attention that also adds each key's softmax weight, summed over the call's
           queries and the heads of its group, to the weights kept per key and KV head
           (keys of the call's own tokens start at 0)
  evict    per sequence, layer and KV head the first ``sinks``, the last ``recent`` and, of
           the other tokens, the heaviest stay, ``keep`` in all; codes, scales and weights
           move to the front of other pages, in order

Lengths come from the case alone; values, page tables and row numbers from the seed.
Histories hold N(0, 1) keys and values quantized to the cache's format.
"""

import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

BLOCK = 16
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
FORMATS = {"int8": (torch.int8, 127.0), "fp8_e4m3fn": (torch.float8_e4m3fn, 448.0),
           "fp8_e5m2": (torch.float8_e5m2, 57344.0)}

BASE = {"op": "sinks", "rows": 1, "lo": 1, "hi": 1, "chunk_lo": 1, "chunk_hi": 1, "q_heads": 32,
        "kv_heads": 8, "dim": 128, "dtype": "bfloat16", "format": "int8", "window": 0, "sinks": 0,
        "padding": 0.0, "layers": 1, "keep": 0, "recent": 0, "mix": 0}

# (visible keys x KV heads x head dim) of a decode call, scores of a chunk call and K/V codes
# of an eviction: the largest listed case's
MOST_KV = 16 * 32768 * 8 * 128
MOST_SCORES = 32 * 512 * 16512
MOST_TOKENS = 8 * 9000 * 16 * 8 * 128


def _case(name, **values):
    return {"name": name, **BASE, **values}


def listed():
    return [
        # one user alone on the card, far into a long chat with a sliding-window model
        _case("sink_decode_one", lo=8192, hi=8192, window=1024, sinks=4),
        # the smallest call: four short chats of a small fp32 model
        _case("sink_decode_fp32", rows=4, lo=17, hi=300, q_heads=4, kv_heads=4, dim=64,
              dtype="float32", window=100, sinks=5, mix=1),
        # a sliding-window model over an FP8 cache, long chats, fp16
        _case("sink_decode_fp8", rows=48, lo=500, hi=9000, q_heads=32, kv_heads=4,
              dtype="float16", format="fp8_e4m3fn", window=1024, sinks=4, mix=2),
        # the ordinary full batch with a wide window
        _case("sink_decode_batch", rows=128, lo=64, hi=9000, window=4096, sinks=64, mix=3),
        # the next chunk of one long prompt
        _case("sink_chunk", lo=16000, hi=16000, chunk_lo=512, chunk_hi=512, window=4096, sinks=16,
              mix=4),
        # ragged prompts of a head-dim 64 model over an FP8 cache
        _case("sink_chunks_fp8", rows=12, lo=0, hi=700, chunk_lo=33, chunk_hi=900, q_heads=16,
              kv_heads=8, dim=64, dtype="float16", format="fp8_e4m3fn", window=256, sinks=3, mix=5),
        # a bounded cache: the decode step of a single sequence
        _case("weights_decode_one", op="weights", lo=8192, hi=8192, mix=6),
        # ... and of 64 chats of mixed lengths
        _case("weights_decode_batch", op="weights", rows=64, lo=128, hi=4096, mix=7),
        # long documents before their first eviction
        _case("weights_decode_long", op="weights", rows=16, lo=32768, hi=32768, q_heads=64, mix=8),
        # a new prompt
        _case("weights_prompt", op="weights", lo=0, hi=0, chunk_lo=2000, chunk_hi=2000, mix=9),
        # one sequence of a four-layer decoder back to its budget
        _case("evict_one", op="evict", lo=1100, hi=1100, layers=4, kv_heads=4, keep=1024, sinks=4,
              recent=128, mix=10),
        # prompts of mixed lengths cut to the budget, 16 layers
        _case("evict_prompts", op="evict", rows=8, lo=1500, hi=9000, layers=16, keep=1024, sinks=4,
              recent=256, mix=11),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["sinks", "sinks", "sinks", "weights", "weights", "weights", "evict", "evict"])
    kv_heads = rng.choice([2, 4, 8, 8])
    group = rng.choice([1, 2, 4, 4, 8])
    case = {**BASE, "op": op, "dim": rng.choice([64, 128, 128, 128, 256]), "kv_heads": kv_heads,
            "q_heads": kv_heads * group, "dtype": rng.choice(["bfloat16", "bfloat16", "float16"]),
            "format": rng.choice(["int8", "int8", "fp8_e4m3fn", "fp8_e5m2"]),
            "padding": rng.choice([0.0, 0.0, 0.0, 0.1]), "mix": rng.randrange(1 << 20)}
    if op == "evict":
        case["layers"] = _log(rng, 1, 16)
        case["keep"] = _log(rng, 16, 2048)
        case["sinks"] = rng.choice([0, 4, min(16, case["keep"] // 4)])
        case["recent"] = rng.randrange(case["keep"] // 2 + 1)
        case["lo"] = _log(rng, 16, 4096)
        case["hi"] = case["lo"] + _log(rng, 1, 8192)
        case["rows"] = _log(rng, 1, 32)
        while case["rows"] > 1 and case["rows"] * case["hi"] * case["layers"] * kv_heads \
                * case["dim"] > MOST_TOKENS:
            case["rows"] //= 2
        while case["layers"] > 1 and case["hi"] * case["layers"] * kv_heads * case["dim"] > MOST_TOKENS:
            case["layers"] //= 2
        return case
    if op == "sinks":
        case["window"] = _log(rng, 16, 4096)
        case["sinks"] = _log(rng, 1, 64)
    case["lo"] = _log(rng, 1, 8192)
    case["hi"] = case["lo"] + _log(rng, 1, 8192)
    if rng.random() < 0.65:  # decode
        case["dtype"] = rng.choice([case["dtype"], case["dtype"], "float32"])
        case["rows"] = _log(rng, 1, 256)
        while case["rows"] > 1 and case["rows"] * case["hi"] * kv_heads * case["dim"] > MOST_KV:
            case["rows"] //= 2
        return case
    case["lo"] = rng.choice([0, case["lo"] // 2])
    case["hi"] = case["lo"] + rng.randrange(1, 2048)
    case["chunk_lo"] = _log(rng, 2, 512)
    case["chunk_hi"] = case["chunk_lo"] + rng.randrange(1, 512)
    case["rows"] = _log(rng, 1, 16)
    while case["rows"] * case["chunk_hi"] * (case["hi"] + case["chunk_hi"]) * case["q_heads"] \
            > MOST_SCORES and case["chunk_hi"] > 8:
        if case["rows"] > 1:
            case["rows"] //= 2
        else:
            case["chunk_hi"] = max(8, case["chunk_hi"] // 2)
            case["chunk_lo"] = min(case["chunk_lo"], case["chunk_hi"])
    return case


# ---- shapes (from the case alone) ------------------------------------------------------


def _shape(case):
    """(context lengths, query tokens) per row; ``lo`` to ``hi`` are the lengths of a row of one
    token and those before a chunk."""
    rng = np.random.default_rng(case["mix"])
    prior = rng.integers(case["lo"], case["hi"], size=case["rows"], endpoint=True)
    queries = rng.integers(case["chunk_lo"], case["chunk_hi"], size=case["rows"], endpoint=True)
    lens = prior + (queries if case["chunk_hi"] > 1 else 0)
    return lens.astype(np.int32), queries.astype(np.int32)


def work(case):
    """Codes and scales of every key some query sees, queries in, outputs out, page ids; a
    key's weight in and out; 4 q_heads dim operations per visible (query, key) pair, and half
    as many again where a chunk's weights need the scores under the final sums. Evictions:
    the weights in, the kept rows and weights in and out."""
    lens, queries = _shape(case)
    row = 2 * case["dim"] + 8
    if case["op"] == "evict":
        kept = np.minimum(lens, case["keep"])
        heads = case["layers"] * case["kv_heads"]
        return {"bytes": int(heads * (4 * lens.sum() + (2 * row + 8) * kept.sum())), "flops": 0}
    window = case["window"] or 1 << 30
    first = np.maximum(lens - queries - window + 1, 0)
    keys = int((lens - first + np.minimum(first, case["sinks"])).sum())
    pairs = 0
    for length, n in zip(lens.tolist(), queries.tolist()):
        pos = np.arange(length - n, length)
        start = np.maximum(pos + 1 - window, 0)
        pairs += int((pos + 1 - start + np.minimum(start, case["sinks"])).sum())
    item = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    moved = keys * case["kv_heads"] * row + 2 * int(queries.sum()) * case["q_heads"] * case["dim"] * item \
        + keys // 4
    flops = 4 * case["q_heads"] * case["dim"] * pairs
    if case["op"] == "weights":
        moved += 8 * keys * case["kv_heads"]
        if case["chunk_hi"] > 1:
            flops += flops // 2
    return {"bytes": moved, "flops": flops}


# ---- values ----------------------------------------------------------------------------


def _history(case, blocks, gen):
    """Codes (as bytes) ``[blocks, layers, 2, kv_heads, 16, dim]`` and scales of full pages."""
    dtype, most = FORMATS[case["format"]]
    shape = (case["layers"], 2, case["kv_heads"], BLOCK, case["dim"])
    codes = torch.empty((blocks, *shape), dtype=torch.int8, device="cuda")
    scales = torch.empty((blocks, *shape[:-1]), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // math.prod(shape))
    for at in range(0, blocks, step):
        n = min(step, blocks - at)
        x = torch.randn((n, *shape), generator=gen, device="cuda", dtype=torch.float32)
        amax = x.abs().amax(-1)
        scales[at:at + n] = amax / most
        units = (x / scales[at:at + n][..., None]).clamp(-most, most)
        codes[at:at + n] = (units.round() if case["format"] == "int8" else units).to(dtype).view(torch.int8)
    return codes, scales


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng([case["mix"], seed])
    lens, queries = _shape(case)
    own_pages = -(-lens // BLOCK)
    kept_pages = -(-case["keep"] // BLOCK)
    extra = case["rows"] * kept_pages
    perm = rng.permutation(int(own_pages.sum()) + extra + 16).astype(np.int32)
    tables = np.zeros((case["rows"], max(1, int(own_pages.max()))), dtype=np.int32)
    at = 0
    for r, n in enumerate(own_pages.tolist()):
        tables[r, :n] = perm[at:at + n]
        at += n
    x = SimpleNamespace(case=case, lens_host=lens, queries_host=queries, blocks=len(perm),
                        most=int(lens.max()), most_queries=int(queries.max()))
    x.tables = torch.from_numpy(tables).cuda()
    x.lens = torch.from_numpy(lens).cuda()
    x.codes, x.scales = _history(case, x.blocks, gen)
    x.valid = None
    if case["padding"]:
        x.valid = torch.rand((x.blocks, BLOCK), generator=gen, device="cuda") >= case["padding"]
    if case["op"] == "evict":
        x.dst = torch.from_numpy(perm[at:at + extra].reshape(case["rows"], kept_pages)).cuda()
    else:
        total = int(queries.sum())
        x.query = torch.randn((total, case["q_heads"], case["dim"]), generator=gen, device="cuda",
                              dtype=torch.float32).to(DTYPES[case["dtype"]])
        starts = np.concatenate([[0], np.cumsum(queries)]).astype(np.int32)
        x.starts = torch.from_numpy(starts).cuda() if case["chunk_hi"] > 1 else None
    if case["op"] != "sinks":
        # what the keys have gathered so far (over some four steps, or many before an eviction):
        # most little, some much, some nothing
        x.capacity = -(-max(x.most, case["keep"]) // BLOCK) * BLOCK
        numbers = rng.permutation(2 * case["rows"] + 2)
        x.from_rows, x.to_rows = numbers[:case["rows"]].tolist(), numbers[case["rows"]:2 * case["rows"]].tolist()
        shape = (len(numbers), case["layers"], case["kv_heads"], x.capacity)
        u = torch.rand(shape, generator=gen, device="cuda")
        much = 40.0 if case["op"] == "evict" else 36.0 * case["q_heads"] / case["kv_heads"] / x.most
        x.weights = torch.where(u < 0.05, 0.0, u.pow(8) * much)
    return x


def prepare(case, seed):
    s = _inputs(case, seed)
    s.at = torch.tensor(s.from_rows, device="cuda") if case["op"] != "sinks" else None
    s.to = torch.tensor(s.to_rows, device="cuda") if case["op"] == "evict" else None
    if own:  # the cache and the row numbers that a user's program keeps
        from aster_amd import KeyWeights, KVQuantization, PagedKVCache

        s.cache = PagedKVCache(num_blocks=s.blocks, num_layers=case["layers"],
                               num_kv_heads=case["kv_heads"], head_dim=case["dim"], device="cuda:0",
                               quantization=KVQuantization(case["format"]))
        s.cache.codes.copy_(s.codes)
        s.cache.scales.copy_(s.scales)
        s.codes = s.scales = None
        if s.valid is not None:
            s.cache.write_key_valid(torch.arange(s.blocks * BLOCK, device="cuda"), s.valid.reshape(-1))
        if case["op"] != "sinks":
            s.key_weights = KeyWeights(s.cache, rows=len(s.weights), capacity=s.capacity)
            s.key_weights.values.copy_(s.weights)
            s.weights = None
            s.rows = s.key_weights.select(s.from_rows)
            s.into = s.key_weights.select(s.to_rows)
    return s


# ---- one pass --------------------------------------------------------------------------


def run(s):
    case = s.case
    if case["op"] == "evict":
        return _run_evict(s)
    if own:
        if case["op"] == "sinks":
            return {"out": s.cache.paged_attention(
                0, s.query, s.tables, s.lens, max_context_len=s.most, window=case["window"],
                sinks=case["sinks"], query_start_loc=s.starts,
                max_query_len=s.most_queries if s.starts is not None else None)}
        out = s.cache.paged_attention_weights(
            0, s.query, s.tables, s.lens, s.rows, max_context_len=s.most, query_start_loc=s.starts,
            max_query_len=s.most_queries if s.starts is not None else None)
        return {"out": out, "weights": s.key_weights.values}
    if s.starts is None and case["op"] == "sinks":
        return {"out": _plain_sink_rows(s)}
    out, seen, weights = _plain_attention(s)
    if case["op"] == "sinks":
        return {"out": out}
    # [rows, queries, heads, keys] -> per key and KV head; the call's own keys start at 0
    rows, n, heads, keys = weights.shape
    new = weights.view(rows, n, case["kv_heads"], -1, keys).sum((1, 3))
    position = torch.arange(keys, device="cuda")
    fresh = position >= (s.lens - _query_counts(s))[:, None]
    old = s.weights[s.at, 0, :, :keys]
    inside = (position < s.lens[:, None])[:, None]
    s.weights[s.at, 0, :, :keys] = torch.where(inside, torch.where(fresh[:, None], 0.0, old) + new, old)
    return {"out": out, "weights": s.weights}


def _query_counts(s):
    return s.starts[1:] - s.starts[:-1] if s.starts is not None else torch.ones_like(s.lens)


def _dequantized(s, positions, layer=0):
    """K and V ``[rows, kv_heads, positions, dim]`` of per-row positions, in 32 bits."""
    page = s.tables.gather(1, positions // BLOCK).long()
    slot = positions % BLOCK
    codes = s.codes[page, layer, :, :, slot].view(FORMATS[s.case["format"]][0]).float()
    x = codes * s.scales[page, layer, :, :, slot][..., None]  # [rows, positions, 2, heads, dim]
    real = s.valid[page, slot] if s.valid is not None else None
    return x[:, :, 0].transpose(1, 2), x[:, :, 1].transpose(1, 2), real


def _softmax(scores, seen):
    """Weights of masked scores; a row that sees nothing has weights 0."""
    top = scores.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(top.isfinite(), top, 0.0)).masked_fill(~seen, 0.0)
    return w / w.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)


def _plain_sink_rows(s):
    """Rows of one token: only the positions that they can see are read."""
    case = s.case
    last = (s.lens - 1).long()[:, None]
    tail = last - torch.arange(min(case["window"], s.most), device="cuda")
    head = torch.arange(min(case["sinks"], s.most), device="cuda").expand(case["rows"], -1)
    positions = torch.cat([head, tail], 1)
    seen = torch.cat([head < (last + 1 - case["window"]).clamp_min(0), tail >= 0], 1)
    k, v, real = _dequantized(s, positions.clamp_min(0))
    if real is not None:
        seen = seen & real
    q = s.query.float().view(case["rows"], case["kv_heads"], -1, case["dim"])
    w = _softmax(q @ k.transpose(2, 3) * case["dim"] ** -0.5, seen[:, None, None])
    return (w @ v).view_as(s.query).to(s.query.dtype)


def _plain_attention(s):
    """Every row padded to the longest: outputs packed, and weights [rows, queries, heads, keys]."""
    case, kv = s.case, s.case["kv_heads"]
    n, rows = s.most_queries, case["rows"]
    counts = _query_counts(s).long()
    first = s.starts[:-1].long() if s.starts is not None else torch.arange(rows, device="cuda")
    index = first[:, None] + torch.arange(n, device="cuda")
    used = torch.arange(n, device="cuda") < counts[:, None]
    index = index.clamp_max(len(s.query) - 1)
    q = s.query[index].float().view(rows, n, kv, -1, case["dim"])
    keys = torch.arange(s.most, device="cuda")
    k, v, real = _dequantized(s, keys.expand(rows, -1))
    pos = (s.lens.long() - counts)[:, None] + torch.arange(n, device="cuda")
    seen = (keys <= pos[..., None]) & used[..., None]
    if case["window"]:
        seen &= (keys > pos[..., None] - case["window"]) | (keys < case["sinks"])
    if real is not None:
        seen &= real[:, None]
    # [rows, kv, queries x group, keys]
    q = q.permute(0, 2, 1, 3, 4).reshape(rows, kv, -1, case["dim"])
    scores = (q @ k.transpose(2, 3) * case["dim"] ** -0.5).view(rows, kv, n, -1, s.most)
    w = _softmax(scores, seen[:, None, :, None])
    out = (w.view(rows, kv, -1, s.most) @ v).view(rows, kv, n, -1, case["dim"])
    out = out.permute(0, 2, 1, 3, 4).reshape(rows, n, -1, case["dim"])[used].to(s.query.dtype)
    return out, seen, w.permute(0, 2, 1, 3, 4).reshape(rows, n, -1, s.most)


def _run_evict(s):
    case = s.case
    if own:
        got = s.cache.evict(s.tables, s.lens, s.rows, keep=case["keep"], recent=case["recent"],
                            sinks=case["sinks"], max_context_len=s.most, dst_tables=s.dst,
                            into=s.into)
        return {"kept": got.kept, "lengths": got.lengths, "codes": s.cache.code_view(s.cache.codes),
                "scales": s.cache.scales, "weights": s.key_weights.values}
    keys = torch.arange(s.most, device="cuda")
    real = (keys < s.lens[:, None])
    if s.valid is not None:
        real &= s.valid[s.tables.gather(1, (keys // BLOCK).expand(case["rows"], -1)).long(), keys % BLOCK]
    rank = real.long().cumsum(1) - 1  # among the real tokens
    count = real.long().sum(1, keepdim=True)
    fixed = real & ((rank < case["sinks"]) | (rank >= count - case["recent"]))
    w = s.weights[s.at, :, :, :s.most]
    order = torch.where(fixed[:, None, None], math.inf, torch.where(real[:, None, None], w, -math.inf))
    order = order.sort(dim=-1, descending=True, stable=True).indices[..., :case["keep"]]
    lengths = count[:, 0].clamp_max(case["keep"])
    slot = torch.arange(order.shape[-1], device="cuda")
    there = (slot < lengths[:, None])[:, None, None]
    kept = order.masked_fill(~there, s.most).sort(-1).values
    there = there.expand_as(kept)
    row, layer, head, to = there.nonzero(as_tuple=True)
    at = kept[there]
    page, dst = s.tables[row, at // BLOCK].long(), s.dst[row, to // BLOCK].long()
    codes, scales = s.codes[page, layer, :, head, at % BLOCK], s.scales[page, layer, :, head, at % BLOCK]
    s.codes[dst, layer, :, head, to % BLOCK] = codes
    s.scales[dst, layer, :, head, to % BLOCK] = scales
    s.weights[s.to[row], layer, head, to] = w[row, layer, head, at]
    if s.valid is not None:
        s.valid[dst, to % BLOCK] = True
    full = torch.full((*kept.shape[:3], case["keep"]), -1, dtype=torch.int32, device="cuda")
    full[..., :kept.shape[-1]] = torch.where(there, kept, -1)
    return {"kept": full, "lengths": lengths.to(torch.int32),
            "codes": s.codes.view(FORMATS[case["format"]][0]), "scales": s.scales, "weights": s.weights}


# ---- 64-bit results --------------------------------------------------------------------


def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "evict":
        weights = x.weights.double()
        scales = x.scales.double()
        for r, n in enumerate(x.lens_host.tolist()):
            pages = x.tables[r].long()
            tokens = torch.arange(n, device="cuda")
            if x.valid is not None:
                tokens = tokens[x.valid[pages[tokens // BLOCK], tokens % BLOCK]]
            keep = min(case["keep"], len(tokens))
            if not keep:
                continue
            must = torch.zeros(len(tokens), dtype=torch.bool, device="cuda")
            must[:case["sinks"]] = True
            must[max(0, len(tokens) - case["recent"]):] = True
            for layer in range(case["layers"]):
                w = weights[x.from_rows[r], layer][:, tokens]
                best = torch.argsort(torch.where(must, math.inf, w), dim=-1, descending=True, stable=True)
                chosen = tokens[best[:, :keep].sort(-1).values]  # [kv_heads, keep]
                heads = torch.arange(case["kv_heads"], device="cuda")[:, None]
                place = torch.arange(keep, device="cuda")
                dst = x.dst[r].long()[place // BLOCK]
                for which in range(2):
                    scales[dst, layer, which, heads, place % BLOCK] = \
                        scales[pages[chosen // BLOCK], layer, which, heads, chosen % BLOCK]
                weights[x.to_rows[r], layer, heads, place] = weights[x.from_rows[r], layer, heads, chosen]
        return {"kept": None, "lengths": None, "codes": None, "scales": scales, "weights": weights}
    outs, at = [], 0
    weights = x.weights.double() if case["op"] == "weights" else None
    group = case["q_heads"] // case["kv_heads"]
    for r, (length, n) in enumerate(zip(x.lens_host.tolist(), x.queries_host.tolist())):
        pages = x.tables[r, :-(-length // BLOCK)].long()
        keys = torch.arange(length, device="cuda")
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        seen = keys <= pos
        if case["window"]:
            seen = seen & ((pos - keys < case["window"]) | (keys < case["sinks"]))
        if x.valid is not None:
            seen = seen & x.valid[pages].reshape(-1)[:length]
        if weights is not None:
            weights[x.from_rows[r], 0, :, length - n:length] = 0.0
        out = torch.empty((n, case["q_heads"], case["dim"]), dtype=torch.float64, device="cuda")
        for head in range(case["kv_heads"]):
            kv = x.codes[pages, 0, :, head].view(FORMATS[case["format"]][0]).double() \
                * x.scales[pages, 0, :, head].double()[..., None]
            k, v = (kv[:, i].reshape(-1, case["dim"])[:length].contiguous() for i in range(2))
            for g in range(head * group, head * group + group):
                score = (x.query[at:at + n, g].double() @ k.t().contiguous()) / math.sqrt(case["dim"])
                p = torch.nan_to_num(torch.softmax(score.masked_fill(~seen, -math.inf), -1))
                out[:, g] = p @ v
                if weights is not None:
                    weights[x.from_rows[r], 0, head, :length] += p.sum(0)
        outs.append(out)
        at += n
    result = {"out": torch.cat(outs)}
    return result if weights is None else {**result, "weights": weights}
