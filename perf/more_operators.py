"""Performance cases of the 4-bit paged cache and of attention with further forms of its scores.

A serving program that keeps its cache in 4 bits appends to it (``paged_kv_append_int4``), attends it
(``paged_attention_int4``) and takes tokens out of it again (``paged_kv_read``, of any cache). Models whose
scores are capped, lose with the distance of the token, or whose first tokens are seen by all rows attend
with ``biased_paged_attention``, over any of the caches. ``own`` selects the framework's calls; otherwise
``run`` computes the same from elementary torch operations in 32 bits.

Keys and values in 4 bits: groups of 32 elements of a token's head (the last may be shorter), each with a
scale and a lowest value in f16; the value of a code is lowest + scale * code. Eight codes make a 32-bit
word, element e at bit 16 (e % 2) + 4 (e // 2).

Head counts follow the projections of this repository (4096 columns: 32 query heads of 128, shared by
fours) and the usual other ones.
"""
import random

import torch

own = False

_ARTIFACTS = {}
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_GROUP = 32
_MOST = 61440.0  # of a stored value


def _tokens(new, past):
    """New and cached tokens of a sequence: between two ends."""
    return {"new_low": new[0], "new_high": new[1], "past_low": past[0], "past_high": past[1]}


def _form(cap=0.0, distance=False, prefix=0, window=0, causal=True):
    """What the scores are besides products: capped at `cap`, less with the distance, the first (up to) `prefix` seen."""
    return {"cap": cap, "distance": distance, "prefix": prefix, "window": window, "causal": causal}


def listed():
    heads = {"HQ": 32, "HK": 8, "D": 128}
    qkv = {**heads, "R": 128, "interleaved": False}
    return [
        # the smallest call: a decoding sequence adds a token
        {"name": "append4_t1", "op": "paged_kv_append", "dtype": "f16", "cache": "int4", "norm": True, "T": 1, **qkv,
         "PAGE": 16, "PAGES": 256, "prepared": True},
        # a long prompt's keys and values, no norms
        {"name": "append4_t8192", "op": "paged_kv_append", "dtype": "bf16", "cache": "int4", "norm": False, "T": 8192,
         **qkv, "PAGE": 64, "PAGES": 192, "prepared": False},
        # an odd number of tokens, small heads rotated in part
        {"name": "append4_t777", "op": "paged_kv_append", "dtype": "f16", "cache": "int4", "norm": True, "T": 777,
         "HQ": 14, "HK": 2, "D": 64, "R": 32, "interleaved": True, "PAGE": 32, "PAGES": 64, "prepared": False},
        # a prompt's shared beginning, taken out of the cache for a plain product
        {"name": "read4_t4096", "op": "paged_kv_read", "dtype": "bf16", "cache": "int4", "T": 4096, **heads, "PAGE": 16,
         "PAGES": 400, "prepared": False},
        # a long session in 8 bits that moves to another place, page by page
        {"name": "read8_t50001", "op": "paged_kv_read", "dtype": "f16", "cache": "fp8", "T": 50001, **heads, "PAGE": 64,
         "PAGES": 1000, "prepared": False},
        # one sequence decoding over 4096 tokens
        {"name": "attn4_decode_s1", "op": "paged_attention", "dtype": "f16", "cache": "int4", "S": 1,
         **_tokens((1, 1), (4095, 4095)), **heads, "PAGE": 16, **_form(), "lens": 1, "prepared": True},
        # 64 sequences of ragged lengths decoding
        {"name": "attn4_decode_s64", "op": "paged_attention", "dtype": "bf16", "cache": "int4", "S": 64,
         **_tokens((1, 1), (300, 8191)), **heads, "PAGE": 64, **_form(), "lens": 2, "prepared": True},
        # four long sequences decoding
        {"name": "attn4_decode_s4_long", "op": "paged_attention", "dtype": "f16", "cache": "int4", "S": 4,
         **_tokens((1, 1), (60000, 131000)), **heads, "PAGE": 256, **_form(), "lens": 3, "prepared": True},
        # prompt chunks of ragged lengths over a cache of earlier chunks
        {"name": "attn4_chunk", "op": "paged_attention", "dtype": "bf16", "cache": "int4", "S": 2,
         **_tokens((1200, 2048), (9000, 16000)), **heads, "PAGE": 64, **_form(), "lens": 6, "prepared": False},
        # capped scores in a sliding window, wide heads shared by twos, 32 sequences decoding
        {"name": "capped_decode_s32", "op": "biased_paged_attention", "dtype": "bf16", "cache": "same", "S": 32,
         **_tokens((1, 1), (2000, 8000)), "HQ": 16, "HK": 8, "D": 256, "PAGE": 16, **_form(cap=50.0, window=4096),
         "lens": 8, "prepared": True},
        # a whole prompt whose first tokens (an image's, a document's) see one another, scores capped
        {"name": "prefix_prefill_4096", "op": "biased_paged_attention", "dtype": "bf16", "cache": "same", "S": 1,
         **_tokens((4096, 4096), (0, 0)), **heads, "PAGE": 64, **_form(cap=30.0, prefix=1000), "lens": 9,
         "prepared": False},
        # scores that fall with the distance, decoding sequences and chunks in one batch, a 4-bit cache
        {"name": "distance_mixed", "op": "biased_paged_attention", "dtype": "f16", "cache": "int4", "S": 24,
         **_tokens((1, 700), (0, 3000)), "HQ": 12, "HK": 12, "D": 64, "PAGE": 32, **_form(distance=True), "lens": 7,
         "prepared": False},
    ]


# ---- drawn cases -----------------------------------------------------------------------

def _log_int(rng, low, high):
    return min(high, max(low, int(low * (high / low) ** rng.random() + 0.5)))


def _heads(rng, sizes):
    HK = rng.choice((1, 2, 4, 8))
    return {"HQ": HK * rng.choice((1, 2, 4, 4, 5, 7, 8, 8)), "HK": HK, "D": rng.choice(sizes)}


def _draw_tokens(rng, op):
    most = 8192 if op == "paged_kv_append" else 50000
    c = {"op": op, "dtype": rng.choice(("f16", "bf16")), "T": _log_int(rng, 1, most),
         **_heads(rng, (64, 80, 128, 128, 128, 256))}
    page = rng.choice((16, 32, 64, 128))
    c |= {"PAGE": page, "PAGES": -(-c["T"] // page) + rng.randrange(1, 40), "prepared": c["T"] <= 256}
    if op == "paged_kv_read":
        return {**c, "cache": rng.choice(("same", "fp8", "int4", "int4"))}
    turned = c["D"] // 2 if c["D"] != 80 and rng.random() < 0.3 else c["D"]
    return {**c, "cache": "int4", "R": turned, "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.5}


def _draw_form(rng, most):
    return _form(cap=rng.choice((0.0, 20.0, 30.0, 50.0)), distance=rng.random() < 0.4,
                 prefix=_log_int(rng, 1, most) if rng.random() < 0.4 else 0,
                 window=_log_int(rng, 50, 5000) if rng.random() < 0.25 else 0, causal=rng.random() < 0.85)


def _draw_attention(rng, op):
    cache = "int4" if op == "paged_attention" else rng.choice(("same", "fp8", "int4"))
    c = {"op": op, "dtype": rng.choice(("f16", "bf16")), "cache": cache,
         **_heads(rng, (64, 96, 128, 128, 128, 256)), "PAGE": rng.choice((16, 32, 64, 256))}
    kind = rng.choice(("decode", "decode", "verify", "chunk", "chunk", "mixed"))
    row = c["HQ"] * 4.0  # bytes of one query token's scores against one cached token, in 32 bits
    if kind in ("decode", "verify"):
        S, new = _log_int(rng, 1, 128), 1 if kind == "decode" else rng.randrange(2, 9)
        most = int(min(131000, 2.0e9 / (S * c["HK"] * c["D"] * 4), 4e9 / (row * S * new)))
        high = _log_int(rng, min(64, most), most)
        new = (new, new)
    else:
        S = 1 if kind == "chunk" and rng.random() < 0.5 else rng.randrange(2, 20)
        new = _log_int(rng, 17, 4096 if S == 1 else 1024)
        most = int(min(30000, 5e9 / (row * S * new)))
        high = _log_int(rng, 16, max(16, most - new))
        new = (1 if kind == "mixed" else -(-new // 2), new)
    low = high if S == 1 else rng.randrange(0, high + 1)
    form = _draw_form(rng, high) if op == "biased_paged_attention" else _form()
    return {**c, "S": S, **_tokens(new, (low, high)), **form, "lens": rng.randrange(1 << 20),
            "prepared": kind in ("decode", "verify")}


def draw(rng):
    op = rng.choice(("paged_kv_append", "paged_kv_read", "paged_attention", "paged_attention",
                     "biased_paged_attention", "biased_paged_attention"))
    return (_draw_attention if op.endswith("attention") else _draw_tokens)(rng, op)


# ---- inputs ----------------------------------------------------------------------------

def _lengths(case):
    """New tokens, cached tokens (the new ones among them) and the prefix of each sequence."""
    rng = random.Random(case["lens"])
    new = [_log_int(rng, case["new_low"], case["new_high"]) for _ in range(case["S"])]
    kv = [n + rng.randint(case["past_low"], case["past_high"]) for n in new]
    return new, kv, [min(k, rng.randint((case["prefix"] + 1) // 2, case["prefix"])) for k in kv]


def _normal(g, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0, std, generator=g).to(dtype)


def _uniform(g, shape, low, high):
    return torch.empty(shape, dtype=torch.float32, device="cuda").uniform_(low, high, generator=g)


def _cache(g, case, pages):
    """Keys or values in pages, filled, and what the codes of 8 or 4 bits are read by."""
    HK, PAGE, D = case["HK"], case["PAGE"], case["D"]
    if case["cache"] == "same":
        return _normal(g, (pages, HK, PAGE, D), _TYPES[case["dtype"]]), None
    if case["cache"] == "fp8":
        codes = torch.empty((pages, HK, PAGE, D), dtype=torch.float16, device="cuda").normal_(0, 150, generator=g)
        return codes.clamp_(-448, 448).to(torch.float8_e4m3fn), _uniform(g, (pages, HK, PAGE), 0.004, 0.01)
    codes = torch.randint(0, 256, (pages, HK, PAGE, D // 2), dtype=torch.uint8, device="cuda", generator=g)
    scale = _uniform(g, (pages, HK, PAGE, -(-D // _GROUP)), 0.1, 0.3)
    low = torch.empty_like(scale).normal_(0, 0.3, generator=g).sub_(scale * 7.5)
    return codes, torch.stack((scale, low), -1).half()


def _rotation(R, length):
    """cos and sin of every position: [length, R], cosines in the first half."""
    inverse = 500000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    angle = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * inverse
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _add_caches(s, g, case, pages):
    for name in ("k", "v"):
        s[name + "_cache"], s[name + "_params"] = _cache(g, case, pages)


def _prepare_append(case, g):
    T, HQ, HK, D = (case[k] for k in ("T", "HQ", "HK", "D"))
    dt = _TYPES[case["dtype"]]
    # what the projection of queries, keys and values wrote: one row for each token; keys stand off zero by column
    qkv = _normal(g, (T, (HQ + 2 * HK) * D), torch.float32)
    qkv[:, HQ * D:(HQ + HK) * D] += _normal(g, (HK * D,), torch.float32, 2.0)
    q, k, v = (part.unflatten(1, (-1, D)) for part in qkv.to(dt).split((HQ * D, HK * D, HK * D), 1))
    weights = [(1 + _normal(g, (D if case["norm"] else 0,), torch.float32, 0.1)).to(dt) for _ in range(2)]
    length = 16384
    slots = torch.randperm(case["PAGES"] * case["PAGE"], device="cuda", generator=g)[:T]
    s = {"case": case, "q": q, "k": k, "v": v, "q_weight": weights[0], "k_weight": weights[1],
         "cos_sin": _rotation(case["R"], length),
         "positions": torch.randint(0, length, (T,), dtype=torch.int32, device="cuda", generator=g),
         "slots": slots.to(torch.int32), "q_out": torch.empty((T, HQ, D), dtype=dt, device="cuda")}
    s |= {name: torch.empty((T, HK, D), dtype=dt, device="cuda") for name in ("k_out", "v_out")}
    _add_caches(s, g, case, case["PAGES"])
    return s


def _prepare_read(case, g):
    T, PAGE = case["T"], case["PAGE"]
    # a sequence's pages lie anywhere, its tokens one behind the other in them; a few rows are padding
    pages = torch.randperm(case["PAGES"], device="cuda", generator=g)
    token = torch.arange(T, device="cuda")
    slots = pages[token // PAGE] * PAGE + token % PAGE
    slots = torch.where(_uniform(g, (T,), 0, 1) < 0.01, -1, slots)
    s = {"case": case, "slots": slots.to(torch.int32)}
    s |= {name: torch.empty((T, case["HK"], case["D"]), dtype=_TYPES[case["dtype"]], device="cuda")
          for name in ("k_out", "v_out")}
    _add_caches(s, g, case, case["PAGES"])
    return s


def _prepare_attention(case, g):
    new, kv, prefix = _lengths(case)
    T, S, PAGE, HQ = sum(new), case["S"], case["PAGE"], case["HQ"]
    dt = _TYPES[case["dtype"]]
    need = [-(-n // PAGE) for n in kv]
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    column = torch.arange(max(need) + 2, device="cuda")
    count = torch.tensor(need, device="cuda")[:, None]
    first = count.cumsum(0) - count
    table = torch.where(column < count, order[(first + column).clamp(max=pages - 1)], -1)
    offsets = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    s = {"case": case, "most_new": max(new), "most_kv": max(kv),
         "q": _normal(g, (T, HQ, case["D"]), dt, 6.0 if case["cap"] else 1.5),
         "page_table": table.to(torch.int32).contiguous(), "q_offsets": offsets,
         "kv_lens": torch.tensor(kv, dtype=torch.int32, device="cuda"), "scale": case["D"] ** -0.5,
         "out": torch.empty((T, HQ, case["D"]), dtype=dt, device="cuda")}
    if case["op"] == "biased_paged_attention":
        slopes = 2.0 ** (-8.0 * torch.arange(1, HQ + 1, dtype=torch.float64, device="cuda") / HQ)
        s["slopes"] = slopes.float() if case["distance"] else torch.empty(0, device="cuda")
        s["prefix_lens"] = torch.tensor(prefix if case["prefix"] else [], dtype=torch.int32, device="cuda")
    _add_caches(s, g, case, pages)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    make = {"paged_kv_append": _prepare_append, "paged_kv_read": _prepare_read}.get(case["op"], _prepare_attention)
    return make(case, g)


# ---- the framework's calls -------------------------------------------------------------

def _artifact(op, case, **constexprs):
    """The compiled operator a program keeps for its lifetime."""
    import intent_amd as intent

    name = (op if case["dtype"] == "f16" else case["dtype"] + "_" + op) + {"same": ""}.get(case["cache"],
                                                                                         "_" + case["cache"])
    key = (name, tuple(constexprs.items()))
    if key not in _ARTIFACTS:
        _ARTIFACTS[key] = intent.compile(getattr(intent, name), target=intent.MI355XTarget(0), constexprs=constexprs)
    return _ARTIFACTS[key]


_CACHE = ("k_cache", "v_cache", "k_params", "v_params")
_INPUTS = {"paged_kv_append": ("q", "k", "v", "q_weight", "k_weight", "cos_sin", "positions", "slots", *_CACHE),
           "paged_kv_read": (*_CACHE, "slots"),
           "paged_attention": ("q", *_CACHE, "page_table", "q_offsets", "kv_lens", "scale"),
           "biased_paged_attention": ("q", *_CACHE, "page_table", "q_offsets", "kv_lens", "slopes", "prefix_lens",
                                      "scale")}
_OUTPUTS = {"paged_kv_append": ("q_out",), "paged_kv_read": ("k_out", "v_out"), "paged_attention": ("out",),
            "biased_paged_attention": ("out",)}


def _call(s, op, artifact):
    inputs = tuple(s[name] for name in _INPUTS[op] if s[name] is not None)
    if s["case"]["prepared"]:  # a decoding loop binds its buffers once and launches for every token
        if op not in s:
            s[op] = artifact.prepare(*inputs, outputs=tuple(s[name] for name in _OUTPUTS[op]))
        s[op].launch()
        return tuple(s[name] for name in _OUTPUTS[op])
    made = artifact.run(*inputs)
    return made if isinstance(made, tuple) else (made,)


def _run_own(s):
    case = s["case"]
    if case["op"] == "paged_kv_read":
        return _call(s, "paged_kv_read", _artifact("paged_kv_read", case))
    if case["op"] == "paged_kv_append":  # and the values that the cache now holds for these tokens
        q = _call(s, "paged_kv_append", _artifact("paged_kv_append", case, INTERLEAVED=case["interleaved"]))
        return (*q, *_call(s, "paged_kv_read", _artifact("paged_kv_read", case)))
    constexprs = {"CAUSAL": case["causal"], "WINDOW": case["window"]}
    if case["op"] == "biased_paged_attention":
        constexprs["SOFTCAP"] = case["cap"]
    return _call(s, case["op"], _artifact(case["op"], case, **constexprs))


# ---- the plain forms: elementary operations in 32 bits ---------------------------------

def _norm_rope(case, x, weight, cos_sin, positions):
    x = x.float()
    if weight.numel():
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    R = case["R"]
    cos, sin = cos_sin[positions.long()][:, None].chunk(2, -1)
    if case["interleaved"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _store4(case, slots, rows, cache, params):
    """Rows [T, HK, D] to codes and (scale, lowest) of groups, at their slots."""
    D = case["D"]
    rows = rows.clamp(-_MOST, _MOST)
    more = -D % _GROUP
    high = torch.nn.functional.pad(rows, (0, more), value=float("-inf")).unflatten(-1, (-1, _GROUP)).amax(-1)
    low = torch.nn.functional.pad(rows, (0, more), value=float("inf")).unflatten(-1, (-1, _GROUP)).amin(-1)
    scale, low = ((high - low) / 15.0).half(), low.half()
    s, m = (t.float().repeat_interleave(_GROUP, -1)[..., :D] for t in (scale, low))
    code = torch.where(s > 0, ((rows - m) / s).round().clamp(0, 15), 0.0).to(torch.int32)
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=rows.device)
    words = (code.unflatten(-1, (-1, 8)) << shift).sum(-1).to(torch.int32)  # no two codes share a bit
    page, place = slots.long() // case["PAGE"], slots.long() % case["PAGE"]
    cache[page, :, place] = words.contiguous().view(torch.uint8)
    params[page, :, place] = torch.stack((scale, low), -1)


def _values(case, codes, params):
    """Cached rows in 32 bits, from what the cache holds of them."""
    if case["cache"] == "same":
        return codes.float()
    if case["cache"] == "fp8":
        return codes.float() * params[..., None]
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=codes.device)
    code = (codes.contiguous().view(torch.int32)[..., None] >> shift & 15).flatten(-2).float()
    s, m = params.float().repeat_interleave(_GROUP, -2)[..., :case["D"], :].unbind(-1)
    return code * s + m


def _rows_at(case, cache, params, page, place):
    return _values(case, cache[page, :, place], None if params is None else params[page, :, place])


def _run_read(s):
    case = s["case"]
    slots = s["slots"].long()
    inside = ((slots >= 0) & (slots < case["PAGES"] * case["PAGE"]))[:, None, None]
    slots = slots.clamp(0, case["PAGES"] * case["PAGE"] - 1)
    page, place = slots // case["PAGE"], slots % case["PAGE"]
    k = _rows_at(case, s["k_cache"], s["k_params"], page, place)
    v = _rows_at(case, s["v_cache"], s["v_params"], page, place)
    dt = _TYPES[case["dtype"]]
    return torch.where(inside, k, 0.0).to(dt), torch.where(inside, v, 0.0).to(dt)


def _run_append(s):
    case = s["case"]
    q = _norm_rope(case, s["q"], s["q_weight"], s["cos_sin"], s["positions"]).to(s["q"].dtype)
    k = _norm_rope(case, s["k"], s["k_weight"], s["cos_sin"], s["positions"])
    _store4(case, s["slots"], k, s["k_cache"], s["k_params"])
    _store4(case, s["slots"], s["v"].float(), s["v_cache"], s["v_params"])
    return (q, *_run_read(s))


def _run_attention(s):
    case = s["case"]
    S, HQ, HK, D, PAGE, window = (case[k] for k in ("S", "HQ", "HK", "D", "PAGE", "window"))
    Q, L, group = s["most_new"], s["most_kv"], case["HQ"] // case["HK"]
    offsets, kv = s["q_offsets"].long(), s["kv_lens"].long()
    T = s["q"].shape[0]
    token = torch.arange(L, device=kv.device)
    page, place = s["page_table"][:, token // PAGE].long().clamp(min=0), (token % PAGE).expand(S, L)
    k = _rows_at(case, s["k_cache"], s["k_params"], page, place).transpose(1, 2).contiguous()  # [S, HK, L, D]
    v = _rows_at(case, s["v_cache"], s["v_params"], page, place).transpose(1, 2).contiguous()
    v.masked_fill_((token >= kv[:, None])[:, None, :, None], 0.0)
    # queries padded to the longest chunk: [S, HK, group * Q, D]
    step = torch.arange(Q, device=kv.device)
    q = s["q"].float()[(offsets[:-1, None] + step).clamp(max=T - 1)]
    q = q.view(S, Q, HK, group, D).permute(0, 2, 3, 1, 4).reshape(S, HK, group * Q, D)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"]).view(S, HK, group, Q, L)
    at = (kv - (offsets[1:] - offsets[:-1]))[:, None] + step  # [S, Q] the queries' positions
    if case["cap"]:
        scores.div_(case["cap"]).tanh_().mul_(case["cap"])
    if case["distance"]:
        distance = (token - at[..., None]).abs_().float()
        scores.addcmul_(s["slopes"].view(1, HK, group, 1, 1), distance[:, None, None], value=-1.0)
    seen = (token < kv[:, None, None]).expand(S, Q, L)
    if case["causal"]:
        first = token <= at[..., None]
        if case["prefix"]:
            first |= token < s["prefix_lens"][:, None, None]
        seen = seen & first
    if window:
        seen = seen & (token > at[..., None] - window)
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weight = scores.sub_(top.masked_fill(top == float("-inf"), 0.0)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(S, HK, group * Q, L), v).view(S, HK, group, Q, D)
    out = (out / total.masked_fill(total == 0, 1.0)).permute(0, 3, 1, 2, 4).reshape(S * Q, HQ, D)
    row = torch.arange(T, device=kv.device)
    sequence = torch.searchsorted(offsets, row, right=True) - 1
    return (out[sequence * Q + row - offsets[sequence]].to(s["q"].dtype),)


def run(state):
    op = state["case"]["op"]
    if own:
        outputs = _run_own(state)
    else:
        outputs = {"paged_kv_append": _run_append, "paged_kv_read": _run_read}.get(op, _run_attention)(state)
    if op != "paged_kv_append":
        return dict(zip(_OUTPUTS[op], outputs))
    kept = {name: state[name] for name in ("k_params", "v_params")}
    return {**dict(zip(("q_out", "k_out", "v_out"), outputs)), **kept}


# ---- what a pass cannot do without -----------------------------------------------------

def _row_bytes(case):
    """Of a cached token's head, keys or values."""
    D = case["D"]
    return {"same": 2 * D, "fp8": D + 4, "int4": D // 2 + 4 * -(-D // _GROUP)}[case["cache"]]


def _attention_work(case):
    new, kv, prefix = _lengths(case)
    window = case["window"] or 1 << 40
    read = pairs = 0
    for n, total, front in zip(new, kv, prefix):
        first = total - n
        read += min(total, window + n - 1)
        pairs += sum((max(p + 1, front) if case["causal"] else total) - max(0, p + 1 - window)
                     for p in range(first, total))
    rows = 2 * sum(new) * case["HQ"] * case["D"] * 2
    return {"bytes": read * 2 * case["HK"] * _row_bytes(case) + rows, "flops": 4 * case["D"] * case["HQ"] * pairs}


def work(case):
    if case["op"].endswith("attention"):
        return _attention_work(case)
    T, HK, D = (case[k] for k in ("T", "HK", "D"))
    read = T * 2 * HK * (_row_bytes(case) + 2 * D)
    if case["op"] == "paged_kv_read":
        return {"bytes": read + 4 * T, "flops": T * 2 * HK * D * 2}
    heads = case["HQ"] + 2 * HK
    append = T * (heads * 2 * D + case["HQ"] * 2 * D + 2 * HK * _row_bytes(case) + 8) + min(T, 16384) * case["R"] * 4
    return {"bytes": append + read, "flops": T * heads * D * 12}


# ---- the definition in 64 bits ---------------------------------------------------------

def _exact_turn(case, heads, weight, angles):
    """Root-mean-square norm and rotation of heads [T, H, D], as complex numbers."""
    y = heads.double()
    if len(weight):
        y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * weight.double()
    half = case["R"] // 2
    turn = torch.complex(angles[:, :half], angles[:, half:])[:, None]
    head, rest = y[..., :2 * half], y[..., 2 * half:]
    if case["interleaved"]:
        z = torch.view_as_complex(head.unflatten(-1, (half, 2)).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) * turn
        head = torch.cat((z.real, z.imag), -1)
    return torch.cat((head, rest), -1)


def _exact_append(case, s):
    angles = s["cos_sin"].double()[s["positions"].long()]
    result = {"q_out": _exact_turn(case, s["q"], s["q_weight"], angles)}
    slot = s["slots"].long()
    for name, rows in (("k", _exact_turn(case, s["k"], s["k_weight"], angles)), ("v", s["v"].double())):
        # (scale, lowest) of tokens in one line: [HK, PAGES * PAGE, groups, 2]
        line = s[name + "_params"].double().transpose(0, 1).flatten(1, 2)
        values = torch.empty_like(rows)
        for n, part in enumerate(rows.split(_GROUP, -1)):
            part = part.clamp(-_MOST, _MOST)
            low = part.min(-1).values.half().double()
            scale = ((part.max(-1).values - part.min(-1).values) / 15).half().double()
            code = torch.round((part - low[..., None]) / scale[..., None]).clamp(0, 15)
            values[..., n * _GROUP:n * _GROUP + part.shape[-1]] = low[..., None] + scale[..., None] * code
            line[:, slot, n] = torch.stack((scale, low), -1).transpose(0, 1)
        result[name + "_out"] = values
        result[name + "_params"] = line.unflatten(1, (case["PAGES"], case["PAGE"])).transpose(0, 1)
    return result


def _exact_values(case, codes, params):
    if case["cache"] == "same":
        return codes.double()
    if case["cache"] == "fp8":
        return codes.double() * params.double()[..., None]
    word = codes.unflatten(-1, (-1, 4)).long() << torch.tensor([0, 8, 16, 24], device="cuda")
    word = word.sum(-1)
    values = torch.empty((*word.shape, 8), dtype=torch.float64, device="cuda")
    for e in range(8):
        values[..., e] = (word // (1 << (16 * (e % 2) + 4 * (e // 2))) % 16).double()
    values = values.flatten(-2)
    for n, part in enumerate(values.split(_GROUP, -1)):  # views
        part.mul_(params[..., n, 0:1].double()).add_(params[..., n, 1:2].double())
    return values


def _exact_read(case, s):
    result = {}
    slot = s["slots"].long()
    for name in ("k", "v"):
        lines = _exact_values(case, s[name + "_cache"], s[name + "_params"]).transpose(0, 1).flatten(1, 2)
        result[name + "_out"] = lines[:, slot.clamp(min=0)].transpose(0, 1) * (slot >= 0)[:, None, None]
    return result


def _exact_attention(case, s):
    group = case["HQ"] // case["HK"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for sequence, (n, total, front) in enumerate(zip(*_lengths(case))):
        pages = s["page_table"][sequence, :-(-total // case["PAGE"])].long()
        position = torch.arange(total - n, total, device="cuda")[:, None]
        token = torch.arange(total, device="cuda")
        hidden = (token > position) & (token >= front) if case["causal"] else torch.zeros_like(token > position)
        if case["window"]:
            hidden |= token + case["window"] <= position
        for head in range(case["HK"]):
            rows = []
            for name in ("k", "v"):
                params = s[name + "_params"]
                x = _exact_values(case, s[name + "_cache"][pages, head], None if params is None else params[pages, head])
                rows.append(x.flatten(0, 1)[:total])
            for one in range(head * group, head * group + group):
                logit = s["q"][start:start + n, one].double() @ rows[0].t() * s["scale"]
                if case["cap"]:
                    logit = case["cap"] * torch.tanh(logit / case["cap"])
                if case["distance"]:
                    logit = logit - s["slopes"][one].double() * (position - token).abs()
                share = torch.softmax(logit.masked_fill(hidden, float("-inf")), -1)
                out[start:start + n, one] = share @ rows[1]
        start += n
    return {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    return {"paged_kv_append": _exact_append, "paged_kv_read": _exact_read}.get(case["op"], _exact_attention)(case, s)
