"""Performance cases of the attention operators over a paged cache, through ``intent_amd.compile``.

Between the quantized projections of a layer a serving program runs three operators: the
norms of queries and keys with the position rotation (``qk_norm_rope``), the same pass
with the keys and values appended to a paged cache (``paged_kv_append``), and the attention
of the new tokens over that cache (``paged_attention``). Each case is one call of one of
them. ``own`` selects the framework's call; otherwise ``run`` computes the same operator
from elementary torch operations in 32 bits.

Head counts follow the projections of this repository (4096 columns: 32 query heads of
128, shared by fours) and the usual other ones: groups of seven, heads of 64 and 256.
"""
import random

import torch

own = False

_ARTIFACTS = {}
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _tokens(new, past):
    """New and cached tokens of a sequence: between two ends."""
    return {"new_low": new[0], "new_high": new[1], "past_low": past[0], "past_high": past[1]}


def listed():
    qkv = {"HQ": 32, "HK": 8, "D": 128, "R": 128, "interleaved": False}
    small = {"HQ": 14, "HK": 2, "D": 64, "R": 32, "interleaved": True}
    return [
        # the smallest call: one decoding sequence
        {"name": "norm_rope_t1", "op": "qk_norm_rope", "dtype": "f16", "T": 1, **qkv, "prepared": True},
        # a long prompt
        {"name": "norm_rope_t8192", "op": "qk_norm_rope", "dtype": "bf16", "T": 8192, **qkv, "prepared": False},
        # 64 decoding sequences, each adding a token to an 8-bit cache
        {"name": "append_t64_fp8", "op": "paged_kv_append", "dtype": "bf16", "cache": "fp8", "norm": True, "T": 64,
         **qkv, "PAGE": 16, "PAGES": 2048, "prepared": True},
        # a prompt of 8192 tokens into a cache of the activations' type, no norms
        {"name": "append_t8192", "op": "paged_kv_append", "dtype": "f16", "cache": "same", "norm": False, "T": 8192,
         **qkv, "PAGE": 64, "PAGES": 192, "prepared": False},
        # an odd number of tokens, small heads rotated in part
        {"name": "append_t1001_fp8", "op": "paged_kv_append", "dtype": "f16", "cache": "fp8", "norm": True, "T": 1001,
         **small, "PAGE": 32, "PAGES": 64, "prepared": False},
        # one sequence decoding over 4096 tokens
        {"name": "attn_decode_s1", "op": "paged_attention", "dtype": "f16", "cache": "same", "S": 1,
         **_tokens((1, 1), (4095, 4095)), "HQ": 32, "HK": 8, "D": 128, "PAGE": 16, "window": 0, "lens": 1,
         "prepared": True},
        # 64 sequences of ragged lengths decoding over an 8-bit cache
        {"name": "attn_decode_s64_fp8", "op": "paged_attention", "dtype": "bf16", "cache": "fp8", "S": 64,
         **_tokens((1, 1), (300, 8191)), "HQ": 32, "HK": 8, "D": 128, "PAGE": 64, "window": 0, "lens": 2,
         "prepared": True},
        # four long sequences decoding
        {"name": "attn_decode_s4_long", "op": "paged_attention", "dtype": "f16", "cache": "same", "S": 4,
         **_tokens((1, 1), (60000, 131000)), "HQ": 32, "HK": 8, "D": 128, "PAGE": 256, "window": 0, "lens": 3,
         "prepared": True},
        # five drafted tokens for each of 16 sequences, groups of seven heads
        {"name": "attn_verify_s16", "op": "paged_attention", "dtype": "bf16", "cache": "same", "S": 16,
         **_tokens((5, 5), (1000, 6000)), "HQ": 28, "HK": 4, "D": 128, "PAGE": 16, "window": 0, "lens": 4,
         "prepared": True},
        # a whole prompt, no past
        {"name": "attn_prefill_4096", "op": "paged_attention", "dtype": "bf16", "cache": "same", "S": 1,
         **_tokens((4096, 4096), (0, 0)), "HQ": 32, "HK": 8, "D": 128, "PAGE": 64, "window": 0, "lens": 5,
         "prepared": False},
        # prompt chunks of ragged lengths over an 8-bit cache of earlier chunks
        {"name": "attn_chunk_fp8", "op": "paged_attention", "dtype": "f16", "cache": "fp8", "S": 2,
         **_tokens((1200, 2048), (9000, 16000)), "HQ": 32, "HK": 8, "D": 128, "PAGE": 64, "window": 0, "lens": 6,
         "prepared": False},
        # decoding sequences and prompt chunks in one batch, small heads, a sliding window
        {"name": "attn_mixed_window", "op": "paged_attention", "dtype": "f16", "cache": "same", "S": 24,
         **_tokens((1, 700), (0, 3000)), "HQ": 14, "HK": 2, "D": 64, "PAGE": 32, "window": 1000,
         "lens": 7, "prepared": False},
    ]


# ---- drawn cases -----------------------------------------------------------------------

def _log_int(rng, low, high):
    return min(high, max(low, int(low * (high / low) ** rng.random() + 0.5)))


def _heads(rng):
    D = rng.choice((64, 128, 128, 128, 256))
    HK = rng.choice((1, 2, 4, 8))
    group = rng.choice((1, 2, 4, 4, 5, 7, 8, 8))
    return {"HQ": HK * group, "HK": HK, "D": D}


def _draw_tokens(rng, op):
    c = {"op": op, "dtype": rng.choice(("f16", "bf16")), "T": _log_int(rng, 1, 8192), **_heads(rng)}
    c |= {"R": rng.choice((c["D"], c["D"], c["D"] // 2)), "interleaved": rng.random() < 0.3}
    if op == "paged_kv_append":
        page = rng.choice((16, 32, 64, 128))
        c |= {"cache": rng.choice(("same", "fp8")), "norm": rng.random() < 0.5, "PAGE": page,
              "PAGES": -(-c["T"] // page) + rng.randrange(1, 40)}
    return {**c, "prepared": c["T"] <= 256}


def _draw_attention(rng):
    c = {"op": "paged_attention", "dtype": rng.choice(("f16", "bf16")), "cache": rng.choice(("same", "fp8")),
         **_heads(rng), "PAGE": rng.choice((16, 32, 64, 256))}
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
    window = _log_int(rng, 50, 5000) if rng.random() < 0.25 else 0
    return {**c, "S": S, **_tokens(new, (low, high)), "window": window, "lens": rng.randrange(1 << 20),
            "prepared": kind in ("decode", "verify")}


def draw(rng):
    op = rng.choice(("qk_norm_rope", "paged_kv_append", "paged_kv_append", "paged_attention", "paged_attention",
                     "paged_attention"))
    return _draw_attention(rng) if op == "paged_attention" else _draw_tokens(rng, op)


# ---- inputs ----------------------------------------------------------------------------

def _lengths(case):
    """New tokens and cached tokens (the new ones among them) of each sequence."""
    rng = random.Random(case["lens"])
    new = [_log_int(rng, case["new_low"], case["new_high"]) for _ in range(case["S"])]
    kv = [n + rng.randint(case["past_low"], case["past_high"]) for n in new]
    return new, kv


def _normal(g, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0, std, generator=g).to(dtype)


def _uniform(g, shape, low, high):
    return torch.empty(shape, dtype=torch.float32, device="cuda").uniform_(low, high, generator=g)


def _cache(g, case, pages):
    """Keys or values in pages [pages, HK, PAGE, D], filled, and the scales of an 8-bit cache."""
    shape = (pages, case["HK"], case["PAGE"], case["D"])
    if case["cache"] == "same":
        return torch.empty(shape, dtype=_TYPES[case["dtype"]], device="cuda").normal_(0, 1, generator=g), None
    codes = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0, 150, generator=g)
    return codes.clamp_(-448, 448).to(torch.float8_e4m3fn), _uniform(g, shape[:3], 0.004, 0.01)


def _rotation(R, length):
    """cos and sin of every position: [length, R], cosines in the first half."""
    inverse = 500000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    angle = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * inverse
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _prepare_tokens(case, g):
    T, HQ, HK, D = (case[k] for k in ("T", "HQ", "HK", "D"))
    dt = _TYPES[case["dtype"]]
    # what the projection of queries, keys and values wrote: one row for each token
    qkv = _normal(g, (T, (HQ + 2 * HK) * D), dt)
    q, k, v = (part.unflatten(1, (-1, D)) for part in qkv.split((HQ * D, HK * D, HK * D), 1))
    norm = case.get("norm", True)
    weights = [(1 + _normal(g, (D if norm else 0,), torch.float32, 0.1)).to(dt) for _ in range(2)]
    length = 16384
    s = {"case": case, "q": q, "k": k, "v": v, "q_weight": weights[0], "k_weight": weights[1],
         "cos_sin": _rotation(case["R"], length),
         "positions": torch.randint(0, length, (T,), dtype=torch.int32, device="cuda", generator=g),
         "q_out": torch.empty((T, HQ, D), dtype=dt, device="cuda")}
    if case["op"] == "qk_norm_rope":
        s["k_out"] = torch.empty((T, HK, D), dtype=dt, device="cuda")
        return s
    slots = torch.randperm(case["PAGES"] * case["PAGE"], device="cuda", generator=g)[:T]
    s["slots"] = slots.to(torch.int32)
    for name in ("k", "v"):
        s[name + "_cache"], s[name + "_scales"] = _cache(g, case, case["PAGES"])
    return s


def _prepare_attention(case, g):
    new, kv = _lengths(case)
    T, S, PAGE = sum(new), case["S"], case["PAGE"]
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
         "q": _normal(g, (T, case["HQ"], case["D"]), dt, 1.5), "page_table": table.to(torch.int32).contiguous(),
         "q_offsets": offsets, "kv_lens": torch.tensor(kv, dtype=torch.int32, device="cuda"),
         "scale": case["D"] ** -0.5, "out": torch.empty((T, case["HQ"], case["D"]), dtype=dt, device="cuda")}
    for name in ("k", "v"):
        s[name + "_cache"], s[name + "_scales"] = _cache(g, case, pages)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (_prepare_attention if case["op"] == "paged_attention" else _prepare_tokens)(case, g)


# ---- the framework's calls -------------------------------------------------------------

def _definition(case):
    name = case["op"] if case["dtype"] == "f16" else case["dtype"] + "_" + case["op"]
    return name + "_fp8" if case.get("cache") == "fp8" else name


def _artifact(case):
    """The compiled operator a program keeps for its lifetime."""
    import intent_amd as intent

    constexprs = {"WINDOW": case["window"]} if "window" in case else {"INTERLEAVED": case["interleaved"]}
    key = (_definition(case), tuple(constexprs.items()))
    if key not in _ARTIFACTS:
        _ARTIFACTS[key] = intent.compile(getattr(intent, key[0]), target=intent.MI355XTarget(0), constexprs=constexprs)
    return _ARTIFACTS[key]


_INPUTS = {"qk_norm_rope": ("q", "k", "q_weight", "k_weight", "cos_sin", "positions"),
           "paged_kv_append": ("q", "k", "v", "q_weight", "k_weight", "cos_sin", "positions", "slots", "k_cache",
                               "v_cache", "k_scales", "v_scales"),
           "paged_attention": ("q", "k_cache", "v_cache", "k_scales", "v_scales", "page_table", "q_offsets", "kv_lens",
                               "scale")}
_OUTPUTS = {"qk_norm_rope": ("q_out", "k_out"), "paged_kv_append": ("q_out",), "paged_attention": ("out",)}


def _run_own(s):
    case = s["case"]
    op, artifact = case["op"], _artifact(case)
    inputs = tuple(s[name] for name in _INPUTS[op] if s[name] is not None)
    outputs = tuple(s[name] for name in _OUTPUTS[op])
    if case["prepared"]:  # a decoding loop binds its buffers once and launches for every token
        if "call" not in s:
            s["call"] = artifact.prepare(*inputs, outputs=outputs)
        s["call"].launch()
    else:
        made = artifact.run(*inputs)
        outputs = made if isinstance(made, tuple) else (made,)
    return outputs


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


def _store(case, slots, rows, cache, scales):
    page, place = slots.long() // case["PAGE"], slots.long() % case["PAGE"]
    if scales is None:
        cache[page, :, place] = rows.to(cache.dtype)
        return
    scale = rows.abs().amax(-1).clamp(min=1e-12) / 448.0
    codes = (rows / scale[..., None]).clamp(-448.0, 448.0).to(cache.dtype)
    cache.view(torch.uint8)[page, :, place] = codes.view(torch.uint8)
    scales[page, :, place] = scale


def _run_tokens(s):
    case = s["case"]
    dt = s["q"].dtype
    q = _norm_rope(case, s["q"], s["q_weight"], s["cos_sin"], s["positions"]).to(dt)
    k = _norm_rope(case, s["k"], s["k_weight"], s["cos_sin"], s["positions"])
    if case["op"] == "qk_norm_rope":
        return q, k.to(dt)
    _store(case, s["slots"], k, s["k_cache"], s["k_scales"])
    _store(case, s["slots"], s["v"].float(), s["v_cache"], s["v_scales"])
    return (q,)


def _rows_of(cache, scales, page, place):
    """Cached rows [S, HK, L, D] in 32 bits."""
    rows = cache[page, :, place].float()
    if scales is not None:
        rows = rows * scales[page, :, place][..., None]
    return rows.transpose(1, 2).contiguous()


def _run_attention(s):
    case = s["case"]
    S, HQ, HK, D, PAGE, window = (case[k] for k in ("S", "HQ", "HK", "D", "PAGE", "window"))
    Q, L, group = s["most_new"], s["most_kv"], case["HQ"] // case["HK"]
    offsets, kv = s["q_offsets"].long(), s["kv_lens"].long()
    T = s["q"].shape[0]
    token = torch.arange(L, device=kv.device)
    page, place = s["page_table"][:, token // PAGE].long().clamp(min=0), (token % PAGE).expand(S, L)
    k = _rows_of(s["k_cache"], s["k_scales"], page, place)
    v = _rows_of(s["v_cache"], s["v_scales"], page, place)
    v.masked_fill_((token >= kv[:, None])[:, None, :, None], 0.0)
    # queries padded to the longest chunk: [S, HK, group * Q, D]
    step = torch.arange(Q, device=kv.device)
    q = s["q"].float()[(offsets[:-1, None] + step).clamp(max=T - 1)]
    q = q.view(S, Q, HK, group, D).permute(0, 2, 3, 1, 4).reshape(S, HK, group * Q, D)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"]).view(S, HK, group, Q, L)
    at = (kv - (offsets[1:] - offsets[:-1]))[:, None] + step  # [S, Q] the queries' positions
    seen = (token <= at[..., None]) & (token < kv[:, None, None])
    if window:
        seen &= token > at[..., None] - window
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
    if own:
        outputs = _run_own(state)
    elif state["case"]["op"] == "paged_attention":
        outputs = _run_attention(state)
    else:
        outputs = _run_tokens(state)
    result = dict(zip(_OUTPUTS[state["case"]["op"]], outputs))
    if state["case"]["op"] == "paged_kv_append":
        kept = ("k_cache", "v_cache", "k_scales", "v_scales")
        result |= {name: state[name] for name in kept if state[name] is not None}
    return result


# ---- what a pass cannot do without -----------------------------------------------------

def _attention_work(case):
    new, kv = _lengths(case)
    size = 2 if case["cache"] == "same" else 1
    window = case["window"] or 1 << 40
    read = pairs = 0
    for n, total in zip(new, kv):
        first = total - n
        read += min(total, window + n - 1)
        pairs += sum(min(p + 1, window) for p in range(first, total))
    token = 2 * case["HK"] * (case["D"] * size + (4 if size == 1 else 0))
    rows = 2 * sum(new) * case["HQ"] * case["D"] * 2
    return {"bytes": read * token + rows, "flops": 4 * case["D"] * case["HQ"] * pairs}


def work(case):
    if case["op"] == "paged_attention":
        return _attention_work(case)
    T, HQ, HK, D, R = (case[k] for k in ("T", "HQ", "HK", "D", "R"))
    heads, kept = HQ + HK, (HQ + HK) * 2 * D
    if case["op"] == "paged_kv_append":
        heads += HK
        kept = HQ * 2 * D + 2 * HK * (2 * D if case["cache"] == "same" else D + 4)
    # every distinct position's row of the table is read once, however many tokens share it
    return {"bytes": T * (heads * 2 * D + kept + 4) + min(T, 16384) * R * 4, "flops": T * heads * D * 8}


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


def _exact_tokens(case, s):
    angles = s["cos_sin"].double()[s["positions"].long()]
    keys = _exact_turn(case, s["k"], s["k_weight"], angles)
    result = {"q_out": _exact_turn(case, s["q"], s["q_weight"], angles)}
    if case["op"] == "qk_norm_rope":
        return {**result, "k_out": keys}
    slot = s["slots"].long()
    for name, rows in (("k", keys), ("v", s["v"].double())):
        # tokens of a head in one line: [HK, PAGES * PAGE, ...]
        lines = s[name + "_cache"].double().transpose(0, 1).flatten(1, 2)
        if case["cache"] == "fp8":
            scale = rows.abs().max(-1).values.clamp(min=1e-12) / 448
            every = s[name + "_scales"].double().transpose(0, 1).flatten(1, 2)
            every[:, slot] = scale.t()
            result[name + "_scales"] = every.unflatten(1, (case["PAGES"], case["PAGE"])).transpose(0, 1)
            rows = rows / scale[..., None]
        lines[:, slot] = rows.transpose(0, 1)
        result[name + "_cache"] = lines.unflatten(1, (case["PAGES"], case["PAGE"])).transpose(0, 1)
    return result


def _exact_attention(case, s):
    group = case["HQ"] // case["HK"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for sequence, (n, total) in enumerate(zip(*_lengths(case))):
        pages = s["page_table"][sequence, :-(-total // case["PAGE"])].long()
        position = torch.arange(total - n, total, device="cuda")[:, None]
        token = torch.arange(total, device="cuda")
        hidden = token > position
        if case["window"]:
            hidden |= token + case["window"] <= position
        for head in range(case["HK"]):
            rows = []
            for name in ("k", "v"):
                x = s[name + "_cache"][pages, head].double()
                if case["cache"] == "fp8":
                    x = x * s[name + "_scales"][pages, head].double()[..., None]
                rows.append(x.flatten(0, 1)[:total])
            for one in range(head * group, head * group + group):
                logit = s["q"][start:start + n, one].double() @ rows[0].t() * s["scale"]
                share = torch.softmax(logit.masked_fill(hidden, float("-inf")), -1)
                out[start:start + n, one] = share @ rows[1]
        start += n
    return {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attention(case, s) if case["op"] == "paged_attention" else _exact_tokens(case, s)
