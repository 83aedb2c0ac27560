"""What is measured of the serving-step operators over the paged 4- / 8-bit cache: their cases, their plain forms, and
the calls a user makes.

    rope     rotary positions of a step's q and k rows (Ops.rotary, Ops.rope)
    decode   one token per sequence over the cache with a sliding window and sink tokens (Ops.decode(window=, sinks=))
    chunk    several new rows per sequence over the cached history and themselves (Ops.attend_chunk)

A cache is a pool of page records [blocks, H, record bytes]: P tokens x D channels as K codes, V codes, fp16 K scale and
bias per channel, fp16 V scale and bias per token (x = code * scale + bias); an int4 byte j of a token row holds channel
j (low nibble) and channel j + D/2 (high).  The last, unfinished page of a sequence keeps its exact K rows in tail_k.
"""
import functools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------- cases
def _rope(name, rows, heads, kv_heads, dim, rotary_dim, dtype, interleaved=False, scaling="none", max_pos=8192,
          packed=True):
    return {"name": name, "op": "rope", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary_dim": rotary_dim, "dtype": dtype, "interleaved": interleaved, "scaling": scaling,
            "max_pos": max_pos, "packed": packed}


def _decode(name, seqs, kv_heads, group, dim, bits, page, dtype, min_len, max_len, window, sinks):
    return {"name": name, "op": "decode", "seqs": seqs, "kv_heads": kv_heads, "group": group, "dim": dim, "bits": bits,
            "page": page, "dtype": dtype, "min_len": min_len, "max_len": max_len, "window": window, "sinks": sinks}


def _chunk(name, seqs, kv_heads, group, dim, bits, page, dtype, min_ctx, max_ctx, min_new, max_new, window=0, sinks=0):
    return {"name": name, "op": "chunk", "seqs": seqs, "kv_heads": kv_heads, "group": group, "dim": dim, "bits": bits,
            "page": page, "dtype": dtype, "min_ctx": min_ctx, "max_ctx": max_ctx, "min_new": min_new,
            "max_new": max_new, "window": window, "sinks": sinks}


def listed():
    return [
        # one decoded token of one sequence: the launch itself
        _rope("rope one token", 1, 32, 8, 128, 128, "bf16"),
        # a decode batch, part of the head rotated in the interleaved layout, positions stretched linearly
        _rope("rope batch partial", 253, 28, 4, 128, 64, "fp16", True, "linear", 32768),
        # exact rows of a far context in fp32, frequencies scaled by band
        _rope("rope far fp32", 1000, 12, 12, 64, 64, "fp32", False, "llama3", 1 << 20, False),
        # a prefill step of q and k inside packed q|k|v rows, scaled for a long context
        _rope("rope prefill", 16384, 32, 8, 128, 128, "bf16", False, "yarn", 131072),
        # one long conversation: a window of 8192 tokens and 4 sinks
        _decode("window one sequence", 1, 8, 4, 128, 4, 32, "bf16", 131072, 131072, 8192, 4),
        # a ragged batch in 8 bits, one sequence still empty, some shorter than the window
        _decode("window ragged int8", 61, 4, 7, 128, 8, 32, "fp16", 0, 6001, 1000, 5),
        # a serving batch at 16-token pages
        _decode("window batch", 256, 8, 4, 128, 4, 16, "bf16", 3000, 32768, 4096, 64),
        # the first short turn of a conversation
        _chunk("chunk short turn", 1, 8, 4, 128, 4, 32, "bf16", 500, 500, 17, 17),
        # verification of 5 drafted tokens for a batch
        _chunk("chunk verify batch", 64, 8, 4, 128, 4, 16, "bf16", 4000, 8192, 5, 5),
        # prompts of many lengths together, some with history
        _chunk("chunk ragged prefill", 6, 4, 7, 128, 4, 32, "bf16", 0, 2000, 1, 3001),
        # two chunks of long documents under a sliding window, 8-bit cache
        _chunk("chunk window int8", 2, 8, 4, 128, 8, 16, "fp16", 12000, 13000, 1501, 1600, 4096, 16),
        # a chunk of a long prompt over its history
        _chunk("chunk long", 1, 8, 4, 128, 4, 32, "bf16", 30001, 30001, 2048, 2048),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    dim = rng.choice([64, 128, 128, 128, 128, 256])
    op = rng.choice(["rope", "decode", "decode", "chunk", "chunk"])
    heads, group = rng.choice([(8, 4), (4, 7), (8, 1), (2, 8), (1, 5), (4, 12), (16, 2)])
    if op == "rope":
        rows = _spread(rng, 1, 16384 * 40 * 128 * 2 // (heads * (group + 1) * dim * 4))
        case = _rope("", rows, heads * group, heads, dim, rng.choice([dim, dim, dim // 2, dim // 4, 20]), dtype,
                     rng.random() < 0.4, rng.choice(["none", "linear", "ntk", "yarn", "llama3"]),
                     _spread(rng, 1000, 1 << 20), rng.random() < 0.5)
    else:
        bits, page = rng.choice([4, 4, 8]), rng.choice([16, 32])
        if op == "decode":
            window, sinks = _spread(rng, 1, 8192), rng.choice([0, 1, 4, 5, 33, 64, 200])
            cap = max(1, 256 * 8 * 4160 * 128 // (heads * dim * (window + sinks + 64)))
            seqs = _spread(rng, 1, min(300, cap))
            longest = _spread(rng, 1, 100000)
            case = _decode("", seqs, heads, group, dim, bits, page, dtype, rng.choice([0, longest // 2, longest]), longest,
                           window, sinks)
        else:
            # pairs of rows and tokens of the whole padded batch: at most the longest listed one's, fewer where the
            # arithmetic is in 32 bits or the head is wide
            pairs = (2048 * 8 * 4 * 32000 if dtype != "fp32" and dim < 256 else 2048 * 4 * 4000) // (heads * group)
            new = _spread(rng, 1, 3000 if dtype != "fp32" and dim < 256 else 300)
            ctx = rng.choice([0, 1, 2, 2, 2])
            ctx = ctx and _spread(rng, 1, max(1, min(30000, pairs // new - new)))
            held = 64 * 8192 * 8 * 128 // (heads * dim * (ctx + new))
            seqs = _spread(rng, 1, max(1, min(64, held, pairs // (new * (ctx + new)))))
            window, sinks = (0, 0) if rng.random() < 0.6 else (_spread(rng, 1, 8192), rng.choice([0, 1, 4, 70]))
            case = _chunk("", seqs, heads, group, dim, bits, page, dtype, rng.choice([0, ctx]), ctx,
                          rng.choice([1, new]), new, window, sinks)
    del case["name"]
    return case


def _lengths(n, lo, hi):
    """n lengths spread over [lo, hi], both ends among them: what a ragged batch looks like, the same for every seed."""
    got = [lo + int((hi - lo + 1) * ((i * 0.6180339887498949 + 0.5) % 1.0)) for i in range(n)]
    if n > 1:
        got[n // 2], got[n - 1] = lo, hi
    else:
        got[0] = hi
    return got


def _plan(case):
    """(tokens in the cache, new rows) of each sequence."""
    if case["op"] == "decode":
        return _lengths(case["seqs"], case["min_len"], case["max_len"]), [1] * case["seqs"]
    return (_lengths(case["seqs"], case["min_ctx"], case["max_ctx"]),
            _lengths(case["seqs"], case["min_new"], case["max_new"])[::-1])


def _seen(cached, first, window, sinks):
    """Which of `cached` tokens a query at position `first`, or a later one, sees: (sink tokens, first window token)."""
    if not window:
        return 0, 0
    lo = min(cached, max(0, first - window + 1))
    return min(sinks, lo), lo


# ---------------------------------------------------------------------------------------------------- rotary frequencies
SCALINGS = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 4.0},
    "ntk": {"rope_type": "ntk", "factor": 4.0},
    "yarn": {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 8192, "beta_fast": 32.0,
             "beta_slow": 1.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192},
}
THETA = 500000.0


def _frequencies(rotary_dim, name, device):
    """(radians per position of each pair, factor of the cosines and sines), in 64 bits."""
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    freq = THETA ** (-i / rotary_dim)
    c = SCALINGS[name]
    if name == "linear":
        return freq / c["factor"], 1.0
    if name == "ntk":
        return (THETA * c["factor"] ** (rotary_dim / (rotary_dim - 2))) ** (-i / rotary_dim), 1.0
    if name == "yarn":
        # pairs that turn more than beta_fast times over the original context keep their frequency, those that turn less
        # than beta_slow times are stretched, a ramp over the pair's index between
        at = [rotary_dim * math.log(c["original_max_position_embeddings"] / (b * 2 * math.pi)) / (2 * math.log(THETA))
              for b in (c["beta_fast"], c["beta_slow"])]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary_dim - 1)
        keep = 1 - ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return freq / c["factor"] * (1 - keep) + freq * keep, 0.1 * math.log(c["factor"]) + 1.0
    if name == "llama3":
        turns = c["original_max_position_embeddings"] * freq / (2 * math.pi)
        keep = ((turns - c["low_freq_factor"]) / (c["high_freq_factor"] - c["low_freq_factor"])).clamp(0, 1)
        return freq / c["factor"] * (1 - keep) + freq * keep, 1.0
    return freq, 1.0


# ---------------------------------------------------------------------------------------------------- inputs
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _records(gen, pages, heads, dim, bits, page):
    """`pages` blocks of quantized keys (channel offsets and two outlier channels per head, as keys have) and values."""
    levels, half = 2 ** bits - 1, 2 ** (bits - 1)
    offset = 2 * _normal(gen, heads, 1, dim)
    offset[:, :, :2] += 15.0
    out = []
    for start in range(0, pages, 8192):
        n = min(8192, pages - start)
        rows, scales = [], []
        for x, over in ((_normal(gen, n, heads, page, dim) + offset, 2), (_normal(gen, n, heads, page, dim), 3)):
            lo, hi = torch.aminmax(x, dim=over, keepdim=True)
            s = ((hi - lo) / levels).half()
            b = (lo + s.float() * half).half()
            c = ((x - b.float()) / s.float()).round_().clamp_(-half, half - 1).to(torch.int16)
            if bits == 4:
                c = (c[..., :dim // 2] & 15) | ((c[..., dim // 2:] & 15) << 4)
            rows.append((c & 255).to(torch.uint8).reshape(n, heads, -1))
            scales += [s.reshape(n, heads, -1), b.reshape(n, heads, -1)]
        out.append(torch.cat(rows + [t.contiguous().view(torch.uint8) for t in scales], dim=-1))
    return torch.cat(out)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, dim = DTYPES[case["dtype"]], case["dim"]
    s = dict(case)
    if case["op"] == "rope":
        rows, hq, hk = case["rows"], case["heads"], case["kv_heads"]
        if case["packed"]:                                  # q and k are parts of the projection's q|k|v rows
            qkv = _normal(gen, rows, (hq + 2 * hk) * dim).to(dtype)
            s["q"], s["k"] = (t.view(rows, -1, dim) for t in (qkv[:, :hq * dim], qkv[:, hq * dim:(hq + hk) * dim]))
        else:
            s["q"], s["k"] = _normal(gen, rows, hq, dim).to(dtype), _normal(gen, rows, hk, dim).to(dtype)
        first = torch.randint(0, case["max_pos"], (1,), generator=gen, device="cuda")
        s["positions"] = (first + torch.arange(rows, device="cuda")) % case["max_pos"]
        s["q_out"], s["k_out"] = (torch.empty(t.shape, dtype=dtype, device="cuda") for t in (s["q"], s["k"]))
        return s
    heads, page, window, sinks = case["kv_heads"], case["page"], case["window"], case["sinks"]
    cached, new = _plan(case)
    seqs, rows = len(cached), sum(new)
    # a step keeps the pages that a query may see; the pages that the window has left behind were given back
    kept = []
    for n in cached:
        ns, lo = _seen(n, n - 1 if case["op"] == "decode" else n, window, sinks)
        kept.append([p for p in range(-(-n // page)) if p * page < ns or (p + 1) * page > lo])
    blocks = sum(len(p) for p in kept)
    s["cache"] = _records(gen, max(1, blocks), heads, dim, case["bits"], page)
    order = torch.randperm(max(1, blocks), generator=gen, device="cuda").tolist()
    table, at = [[-1] * max(1, -(-max(cached) // page)) for _ in cached], 0
    for i, pages in enumerate(kept):
        for p in pages:
            table[i][p] = order[at]
            at += 1
    s["block_table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
    s["tail_k"] = (_normal(gen, seqs, heads, page, dim) + 2 * _normal(gen, 1, heads, 1, dim)).to(dtype)
    s["tail_idx"] = torch.randperm(seqs, generator=gen, device="cuda").to(torch.int32)
    s["q"] = _normal(gen, rows, heads * case["group"], dim).to(dtype)
    s["out"] = torch.empty_like(s["q"])
    s["max_cached"], s["max_new"] = max(cached), max(new)
    if case["op"] == "decode":
        s["seq_lens"] = torch.tensor(cached, dtype=torch.int32, device="cuda")
    else:
        s["k"] = (_normal(gen, rows, heads, dim) + 2 * _normal(gen, 1, heads, dim)).to(dtype)
        s["v"] = _normal(gen, rows, heads, dim).to(dtype)
        s["seq_lens"] = torch.tensor([c + n for c, n in zip(cached, new)], dtype=torch.int32, device="cuda")
        s["query_start_loc"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    return s


# ---------------------------------------------------------------------------------------------------- the user's calls
@functools.lru_cache(None)
def _ops(dim, bits, group, dtype, page):
    from kushkash_b200 import Ops
    return Ops(torch.device("cuda"), dim, bits, group, DTYPES[dtype], page)


@functools.lru_cache(None)
def _rotary(dim, rotary_dim, dtype, interleaved, scaling):
    return _ops(dim, 4, 1, dtype, 32).rotary(rotary_dim, THETA, interleaved=interleaved, scaling=SCALINGS[scaling])


@functools.lru_cache(None)
def _workspace(n):
    return torch.empty(n, dtype=torch.float32, device="cuda")


def _call(s):
    if s["op"] == "rope":
        ops = _ops(s["dim"], 4, 1, s["dtype"], 32)
        rotary = _rotary(s["dim"], s["rotary_dim"], s["dtype"], s["interleaved"], s["scaling"])
        return ops.rope(s["q"], s["k"], s["positions"], rotary, s["q_out"], s["k_out"])
    ops = _ops(s["dim"], s["bits"], s["group"], s["dtype"], s["page"])
    heads, window, sinks, scale = s["kv_heads"], s["window"] or None, s["sinks"], s["dim"] ** -0.5
    if s["op"] == "decode":
        n = ops.splits(s["seqs"], heads, s["max_cached"] // s["page"], window=window, sinks=sinks)
        work = _workspace(ops.work_size(s["seqs"], heads, n)) if n > 1 else None
        ops.decode(s["q"], s["out"], s["cache"], s["block_table"], s["seq_lens"], s["tail_idx"], s["tail_k"], scale, n, work,
                   window=window, sinks=sinks)
    else:
        rows = s["q"].shape[0]
        n = ops.chunk_splits(rows, s["seqs"], heads, s["max_cached"] + s["max_new"], window=window, sinks=sinks)
        work = _workspace(ops.chunk_work_size(rows, heads, n)) if n > 1 else None
        ops.attend_chunk(s["q"], s["k"], s["v"], s["out"], s["query_start_loc"], s["seq_lens"], s["tail_idx"], s["cache"],
                         s["block_table"], s["tail_k"], scale, n, work, window=window, sinks=sinks)
    return s["out"]


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_rope(s):
    r, dtype = s["rotary_dim"], s["q"].dtype
    freq, factor = _frequencies(r, s["scaling"], s["positions"].device)
    angle = s["positions"].double()[:, None, None] * freq            # 64 bits: a far position times a frequency
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()

    def turned(x):
        x = x.float()
        y = x.clone()
        if s["interleaved"]:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = x[..., :r // 2], x[..., r // 2:r]
            y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
        return y.to(dtype)

    return turned(s["q"]), turned(s["k"])


def _plain_history(s, cached, first):
    """Keys and values of the cached tokens that queries from position `first` on may see, by pages: ([S, pages, P] token
    positions, -1 where there is none; K; V [S, pages, P, H, D]), with the unfinished page's keys from tail_k."""
    page, dim, heads, bits = s["page"], s["dim"], s["kv_heads"], s["bits"]
    pool, table, dev = s["cache"], s["block_table"].long(), s["cache"].device
    lo = (first - s["window"] + 1).clamp(min=0).minimum(cached) if s["window"] else torch.zeros_like(cached)
    sink_pages = torch.minimum(torch.full_like(lo, (s["sinks"] + page - 1) // page), lo // page)
    count = sink_pages + (cached + page - 1) // page - lo // page
    width = min(s["max_cached"] // page + 1, (s["window"] + s["sinks"]) // page + 4) if s["window"] else s["max_cached"] // page + 1
    i = torch.arange(width, device=dev)[None]
    at = torch.where(i < sink_pages[:, None], i, i - sink_pages[:, None] + (lo // page)[:, None])
    real = i < count[:, None]
    block = torch.where(real, table.gather(1, at.clamp(max=table.shape[1] - 1)), 0)
    record = pool[block.clamp(min=0)]                                 # [S, pages, H, bytes]
    width_c = dim if bits == 8 else dim // 2

    def codes(raw):
        raw = raw.unflatten(-1, (page, width_c))
        if bits == 8:
            return raw.view(torch.int8).float()
        low, high = raw & 15, raw >> 4
        both = torch.cat([low, high], dim=-1).to(torch.int8)
        return torch.where(both > 7, both - 16, both).float()

    cuts = [0, page * width_c, 2 * page * width_c]
    cuts += [cuts[2] + 2 * dim, cuts[2] + 4 * dim, cuts[2] + 4 * dim + 2 * page, cuts[2] + 4 * dim + 4 * page]
    part = [record[..., a:b].contiguous() for a, b in zip(cuts, cuts[1:])]
    ks, kb, vs, vb = (p.view(torch.float16).float() for p in part[2:])
    k = codes(part[0]) * ks[..., None, :] + kb[..., None, :]
    v = codes(part[1]) * vs[..., None] + vb[..., None]
    unfinished = (at == (cached // page)[:, None])[..., None, None, None]
    k = torch.where(unfinished, s["tail_k"][s["tail_idx"].long()].float()[:, None], k)
    token = at[..., None] * page + torch.arange(page, device=dev)
    token = torch.where(real[..., None] & (token < cached[:, None, None]), token, -1)
    return token, k.transpose(2, 3), v.transpose(2, 3)


def _plain_attention(q, k, v, seen):
    """q [S, T, H, G, D], k and v [S, N, H, D] in fp32, seen [S, T, N]: softmax(q k) v; 0 for a row that sees nothing."""
    score = torch.einsum("sthgd,snhd->shgtn", q, k)
    seen = seen[:, None, None]
    top = score.masked_fill_(~seen, -math.inf).amax(-1, keepdim=True)
    weight = score.sub_(top.clamp(min=-1e30)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.einsum("shgtn,snhd->sthgd", weight, torch.where(seen[:, 0, 0].any(1)[..., None, None], v, 0.0))
    return out / total.clamp(min=1e-30).permute(0, 3, 1, 2, 4)


def _visible(s, token, position):
    """token [S, N] (-1: none), position [S, T] -> [S, T, N]."""
    token, position = token[:, None, :], position[:, :, None]
    seen = (token >= 0) & (token <= position)
    return seen & ((token > position - s["window"]) | (token < s["sinks"])) if s["window"] else seen


def _plain_decode(s):
    n = s["seq_lens"].long()
    token, k, v = _plain_history(s, n, n - 1)
    q = s["q"].float().view(s["seqs"], 1, s["kv_heads"], s["group"], s["dim"]) * s["dim"] ** -0.5
    out = _plain_attention(q, k.flatten(1, 2), v.flatten(1, 2), _visible(s, token.flatten(1), (n - 1)[:, None]))
    return out.reshape(s["q"].shape).to(s["q"].dtype)


def _plain_chunk(s):
    start = s["query_start_loc"].long()
    new = start[1:] - start[:-1]
    cached = s["seq_lens"].long() - new
    token, k, v = _plain_history(s, cached, cached)
    t = torch.arange(s["max_new"], device=start.device)[None]
    real = t < new[:, None]
    row = (start[:-1, None] + t).clamp(max=s["q"].shape[0] - 1)        # [S, T], rows of a padded batch
    position = cached[:, None] + t
    q = s["q"][row].float().unflatten(2, (s["kv_heads"], s["group"])) * s["dim"] ** -0.5
    token = torch.cat([token.flatten(1), torch.where(real, position, -1)], dim=1)
    k = torch.cat([k.flatten(1, 2), s["k"][row].float()], dim=1)
    v = torch.cat([v.flatten(1, 2), s["v"][row].float()], dim=1)
    out = _plain_attention(q, k, v, _visible(s, token, position) & real[..., None])
    back = torch.empty_like(s["q"])
    back[row[real]] = out.flatten(2, 3)[real].to(back.dtype)
    return back


def run(state):
    if own:
        return _call(state)
    return {"rope": _plain_rope, "decode": _plain_decode, "chunk": _plain_chunk}[state["op"]](state)


# ---------------------------------------------------------------------------------------------------- floors
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rope":
        n = case["rows"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["dim"] * size + 8 * case["rows"], "flops": 3 * n * case["rotary_dim"]}
    heads, group, dim, page = case["kv_heads"], case["group"], case["dim"], case["page"]
    window, sinks = case["window"], case["sinks"]
    code = dim if case["bits"] == 8 else dim // 2
    data, pairs, rows = 0, 0, 0
    for n, t in zip(*_plan(case)):
        ns, lo = _seen(n, n - 1 if case["op"] == "decode" else n, window, sinks)
        tail = min(n % page, ns + n - lo)
        tokens, pages = ns + n - lo, (n // page - lo // page) + (min(ns, lo // page * page) + page - 1) // page
        data += heads * (tokens * (2 * code + 4) + pages * 4 * dim + tail * (size * dim - code)) + 4 * pages
        rows += t
        if case["op"] == "decode":
            pairs += tokens
        else:
            data += 2 * t * heads * dim * size
            for p in range(n, n + t):
                pairs += p + 1 if not window else min(p + 1, window) + min(sinks, max(0, p + 1 - window))
    return {"bytes": data + 2 * rows * heads * group * dim * size, "flops": 4 * dim * heads * group * pairs}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _exact_rope(s):
    r = s["rotary_dim"]
    freq, factor = _frequencies(r, s["scaling"], "cuda")
    turn = torch.polar(torch.full_like(freq, factor)[None], s["positions"].double()[:, None] * freq)[:, None]
    got = []
    for x in (s["q"].double(), s["k"].double()):
        head, rest = x[..., :r], x[..., r:]
        pair = head.unflatten(-1, (r // 2, 2)) if s["interleaved"] else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z if s["interleaved"] else z.transpose(-1, -2)
        got.append(torch.cat([z.reshape(head.shape), rest], dim=-1))
    return tuple(got)


def _exact_tokens(s, i, n, seen):
    """K and V [tokens, H, D] of sequence i's cached tokens `seen` (a sorted list of positions below n), in 64 bits."""
    page, dim, heads = s["page"], s["dim"], s["kv_heads"]
    at = torch.tensor(seen, device="cuda")
    pages, index = torch.unique(at // page, return_inverse=True)
    raw = s["cache"][s["block_table"][i].long()[pages]]
    width = dim * s["bits"] // 8
    scale = raw[..., 2 * page * width:].contiguous().view(torch.float16).double()
    got = []
    for kind in (0, 1):
        c = raw[..., kind * page * width:(kind + 1) * page * width].reshape(len(pages), heads, page, width).to(torch.int32)
        if s["bits"] == 4:
            c = torch.cat([(c << 28) >> 28, (c << 24) >> 28], dim=-1)
        else:
            c = (c << 24) >> 24
        if kind == 0:
            x = c.double() * scale[..., None, :dim] + scale[..., None, dim:2 * dim]
        else:
            x = c.double() * scale[..., 2 * dim:2 * dim + page, None] + scale[..., 2 * dim + page:, None]
        got.append(x.transpose(1, 2)[index, at % page])
    exact = at >= n // page * page
    got[0][exact] = s["tail_k"][int(s["tail_idx"][i])].double().transpose(0, 1)[(at % page)[exact]]
    return at, got[0], got[1]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s)
    cached, new = _plan(case)
    heads, group, dim = case["kv_heads"], case["group"], case["dim"]
    out, row = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (n, t) in enumerate(zip(cached, new)):
        first = n - 1 if case["op"] == "decode" else n
        ns, lo = _seen(n, first, case["window"], case["sinks"])
        seen = list(range(ns)) + list(range(lo, n))
        q = s["q"][row:row + t].double().view(t, heads, group, dim)
        at, k, v = _exact_tokens(s, i, n, seen) if seen else (torch.zeros(0, dtype=torch.long, device="cuda"), None, None)
        if case["op"] == "chunk":
            at = torch.cat([at, n + torch.arange(t, device="cuda")])
            k, v = ([] if x is None else [x] for x in (k, v))
            k, v = torch.cat(k + [s["k"][row:row + t].double()]), torch.cat(v + [s["v"][row:row + t].double()])
        if len(at):
            gap = (first + torch.arange(t, device="cuda"))[:, None] - at[None]
            dark = gap < 0
            if case["window"]:
                dark |= (gap >= case["window"]) & (at >= case["sinks"])[None]
            for h in range(heads):
                for g in range(group):
                    logit = (q[:, h, g] @ k[:, h].T / math.sqrt(dim)).masked_fill(dark, -math.inf)
                    out[row:row + t, h * group + g] = torch.softmax(logit, dim=-1) @ v[:, h]
        row += t
    return out
