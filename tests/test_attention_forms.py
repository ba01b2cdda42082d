"""The 4-bit paged cache (append, read back, attention) and attention with capped, distance-biased and
prefix-masked scores: against their formulas in 64 bits, a decoding loop over them, and their refusals (CPU).

Tolerances are those of the attention over 16 and 8 bits (test_attention.py), with these besides:
* values in 4 bits go into the products as f16: 2^-11 of each key (scores by 2^-11 sum |q k|, weights by
  twice that) and of each value; nothing where lowest + scale * code is an f16. Their weights are f16 (2^-11,
  or 2^-25 absolute), in bf16 too;
* a capped score is 2^-21 of the cap off: 1 - 2 / (exp2(x) + 1) from a reciprocal and an exponential good to
  2^-23 each, two products and a sum; it passes on no more than its argument's error (its slope is at most 1);
* a distance's product: 2^-24 each for the slope in base 2, the product and its sum with the score.
"""
import math

import pytest
import torch

import intent_amd as intent
from intent_amd import _native, errors
from test_attention import (ATTENTION_CASES, F8, FAKE, HALF_STEP, TYPES, _append_args, _close, _cuda, _gen, _heads, _randn,
                            _slot_rows, ref_norm_rope, rounded_bound, runtime_for, status)

BITS = [16 * (e % 2) + 4 * (e // 2) for e in range(8)]
MOST = 61440.0
SUFFIX = {"same": "", "fp8": "_fp8", "int4": "_int4"}


def _compile(op, dt, cache="same", **constexprs):
    name = ("" if dt == "f16" else dt + "_") + op + SUFFIX[cache]
    return intent.compile(getattr(intent, name), target=intent.MI355XTarget(0), constexprs=constexprs or None)


# ---- the cache's formats ---------------------------------------------------------------

def pack4(code):
    """Codes 0..15 [..., D] -> bytes [..., D / 2]."""
    word = sum(code[..., e::8].long() << bit for e, bit in enumerate(BITS))
    return torch.stack([(word >> 8 * b & 255).to(torch.uint8) for b in range(4)], -1).flatten(-2)


def codes4(packed):
    word = sum(packed[..., b::4].long() << 8 * b for b in range(4))
    return torch.stack([word >> bit & 15 for bit in BITS], -1).flatten(-2)


def spread4(pairs, D):
    """Scale and lowest value of every element, in f64."""
    every = pairs.double().repeat_interleave(32, -2)[..., :D, :]
    return every[..., 0], every[..., 1]


def values4(packed, pairs):
    scale, low = spread4(pairs, 2 * packed.shape[-1])
    return low + scale * codes4(packed).double()


def quantize4(x):
    """(codes, pairs) of rows [..., D] by the formula, in f32."""
    D = x.shape[-1]
    x = x.float().clamp(-MOST, MOST)
    parts = x.split(32, -1)
    high, low = (torch.stack([getattr(p, f)(-1) for p in parts], -1) for f in ("amax", "amin"))
    pairs = torch.stack((((high - low) * torch.tensor(1 / 15, dtype=torch.float32)).half(), low.half()), -1)
    scale, lowest = (t.float() for t in spread4(pairs, D))
    code = torch.where(scale > 0, ((x - lowest) / scale).round().clamp(0, 15), 0.0)
    return code, pairs


def _caches(gen, dt, cache, pages, HK, PAGE, D, extra=16, fine=False):
    """[k, v, then scales or groups of both], filled; pages lie `extra` elements apart. `fine`: every value is an f16."""
    made, beside = [], []
    for _ in range(2):
        if cache == "int4":
            x = torch.randint(0, 256, (pages, HK * PAGE * (D // 2) + extra), generator=gen, dtype=torch.uint8)
            made.append(x[:, :HK * PAGE * (D // 2)].unflatten(1, (HK, PAGE, D // 2)))
            G = (D + 31) // 32
            shape = (pages, HK * PAGE * G)
            if fine:  # multiples of 2^-6 below 2^5
                scale = torch.randint(4, 24, shape, generator=gen) / 64.0
                low = torch.randint(-200, 20, shape, generator=gen) / 64.0
            else:
                scale = torch.rand(shape, generator=gen) * 0.2 + 0.1
                low = torch.randn(shape, generator=gen) * 0.3 - 7.5 * scale
            pairs = torch.zeros(pages, HK * PAGE * G * 2 + extra, dtype=torch.float16)
            pairs[:, :HK * PAGE * G * 2] = torch.stack((scale, low), -1).flatten(1).half()
            beside.append(pairs[:, :HK * PAGE * G * 2].unflatten(1, (HK, PAGE, G, 2)))
            continue
        x = _randn(gen, pages, HK * PAGE * D + extra)
        x = (x * 100).clamp(-448, 448).to(F8) if cache == "fp8" else x.to(TYPES[dt])
        made.append(x[:, :HK * PAGE * D].unflatten(1, (HK, PAGE, D)))
        if cache == "fp8":
            x = torch.rand(pages, HK * PAGE + extra, generator=gen) * 0.01 + 0.002
            beside.append(x[:, :HK * PAGE].unflatten(1, (HK, PAGE)))
    return made + beside


def _values(cache, codes, params):
    if cache == "int4":
        return values4(codes, params)
    return codes.double() if cache == "same" else codes.double() * params.double()[..., None]


# ---- append ----------------------------------------------------------------------------

APPEND_CASES = [
    # dtype, T, HQ, HK, D, R, interleaved, norms, page size, pages
    ("f16", 1, 32, 8, 128, 128, False, "qk", 16, 4), ("bf16", 7, 4, 2, 64, 32, True, "qk", 32, 3),
    ("f16", 33, 3, 1, 80, 48, False, "k", 16, 5), ("bf16", 65, 8, 2, 256, 64, False, "", 64, 2),
    ("f16", 9, 2, 2, 96, 96, False, "qk", 8, 4), ("bf16", 5, 1, 4, 8, 0, False, "q", 4, 9),
    ("f16", 130, 14, 2, 64, 64, False, "qk", 128, 2), ("bf16", 6, 2, 1, 512, 512, True, "qk", 2, 9),
    ("f16", 12, 0, 3, 192, 0, False, "", 16, 1), ("bf16", 4, 2, 1, 40, 16, False, "qk", 64, 1),
    ("f16", 20, 4, 0, 64, 64, False, "q", 16, 2), ("bf16", 3, 1, 2, 264, 256, True, "k", 1, 40),
    # two heads to a lane group
    ("bf16", 6561, 4, 3, 96, 96, False, "k", 32, 206), ("f16", 3641, 5, 2, 192, 64, True, "qk", 256, 15),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPEND_CASES, ids=lambda c: "-".join(map(str, c)))
def test_paged_kv_append_int4(gpu, case):
    dt, T, HQ, HK, D, R, interleaved, norms, PAGE, pages = case
    gen = _gen(11)
    heads = _heads(7, dt, T, HQ, HK, D, R, norms)
    q, k, v, qw, kw, table, positions = heads
    count = pages * PAGE
    order = torch.randperm(max(count, T), generator=gen)[:T].to(torch.int32)
    order[order >= count] = -1
    if T > 3:  # padded rows and slots past the cache: skipped
        order[1], order[2], order[3] = -1, count, 2 ** 31 - 1
    kept = (order >= 0) & (order < count)
    # pages of whole 16 bytes
    size = HK * PAGE * (D // 2)
    caches = _caches(gen, dt, "int4", pages, HK, PAGE, D, extra=16 + -size % 16)
    before = [c.clone() for c in caches]
    device = _cuda(*caches)
    q_out = _compile("paged_kv_append", dt, "int4", INTERLEAVED=interleaved).run(*_cuda(*heads, order), *device)
    want, bound = ref_norm_rope(q, qw, table, positions, 1e-6, interleaved)
    _close(q_out, want, rounded_bound(want, bound, TYPES[dt]), case)
    after = [c.cpu() for c in device]
    touched = torch.zeros(pages, PAGE, dtype=torch.bool)
    touched.view(-1)[order[kept].long()] = True
    for new, old in zip(after, before):  # every other row is left as it was
        same = (new == old).flatten(3).all(-1)
        assert bool(same[~touched[:, None, :].expand(same.shape)].all())
    if not int(kept.sum()) or not HK:
        return
    slots = order[kept]
    # values pass no arithmetic before the quantizer: bit-exact with the formula in f32
    code, pairs = quantize4(v[kept])
    assert torch.equal(_slot_rows(after[3], slots), pairs)
    assert torch.equal(_slot_rows(after[1], slots), pack4(code))
    # keys are known to their bound
    key, limit = ref_norm_rope(k[kept], kw, table, positions[kept], 1e-6, interleaved)
    got = _slot_rows(after[2], slots)
    for n, (part, off) in enumerate(zip(key.split(32, -1), limit.split(32, -1))):
        top, low, off = part.amax(-1), part.amin(-1), off.amax(-1)
        scale, lowest = got[:, :, n, 0].double(), got[:, :, n, 1].double()
        assert bool(((scale - (top - low) / 15).abs() <= (2 * off + (top - low) * 2.0 ** -22) / 15 + scale * 2.0 ** -11 + 2.0 ** -25).all())
        assert bool(((lowest - low).abs() <= off + low.abs() * 2.0 ** -11 + 2.0 ** -25).all())
    # the code: half a scale; at a group's ends what rounding its scale and lowest value moved them by
    scale, lowest = spread4(got, D)
    value = values4(_slot_rows(after[0], slots), got)
    slack = scale * (0.5 + 16 * 2.0 ** -11) + lowest.abs() * 2.0 ** -11 + 20 * 2.0 ** -25 + 3 * limit.amax(-1, keepdim=True)
    assert bool(((value - key).abs() <= slack + key.abs() * 2.0 ** -20).all())


@pytest.mark.gpu
def test_paged_kv_append_int4_extremes(gpu):
    """Equal elements, zeros, values past f16, infinities and NaN: each group by itself."""
    D, T = 96, 6
    v = torch.ones(T, 1, D, dtype=torch.bfloat16)
    v[1] = 0
    v[2, 0, :32], v[2, 0, 3] = 2.0, float("nan")
    v[3, 0, 40], v[3, 0, 41] = float("inf"), -3.0
    v[4, 0, 0], v[4, 0, 33], v[4, 0, 64:] = 1e30, -1e30, 1e-30
    v[5] = (_randn(_gen(1), 1, D) * 1e5).bfloat16()
    none = torch.zeros(0, dtype=torch.bfloat16)
    caches = _cuda(*_caches(_gen(2), "bf16", "int4", 2, 1, 4, D))
    slots = torch.arange(T, dtype=torch.int32) + 1
    empty = torch.zeros(T, 0, D, dtype=torch.bfloat16)
    _compile("paged_kv_append", "bf16", "int4").run(*_cuda(empty, v, v, none, none, torch.zeros(1, 0), slots, slots), *caches)
    got = [c.cpu() for c in caches]
    for i in (0, 1):
        codes, pairs = _slot_rows(got[i], slots), _slot_rows(got[2 + i], slots)
        values = values4(codes, pairs)[:, 0]
        assert bool((values[0] == 1).all() and (values[1] == 0).all())
        assert bool(values[2, :32].isnan().all() and (values[2, 32:] == 1).all())
        assert bool(values[3, 32:64].isnan().all() and (values[3, :32] == 1).all() and (values[3, 64:] == 1).all())
        # ends clamped to +-61440, the others within half a step
        assert abs(float(values[4, 0]) - MOST) <= MOST * 2.0 ** -9 and abs(float(values[4, 33]) + MOST) <= MOST * 2.0 ** -9
        assert bool((values[4, 64:].abs() <= 2.0 ** -25).all())
        code, want = quantize4(v[5])
        assert torch.equal(pairs[5], want) and torch.equal(codes[5], pack4(code))
        assert bool(values[5].half().isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_int4_values_are_as_near_as_stated(gpu, dt):
    """Groups far off zero and of small ranges: half a scale, or what rounding the pair to f16 moves the ends by."""
    T, HK, D, PAGE, pages = 256, 2, 128, 16, 17
    gen = _gen(6)
    offset = 10.0 ** torch.linspace(-8, 4.2, T)[:, None, None] * (1 - 2 * torch.randint(0, 2, (T, HK, 1), generator=gen))
    reach = 10.0 ** -torch.linspace(0, 4, D // 32).repeat_interleave(32)
    v = (offset * (1 + torch.rand(T, HK, D, generator=gen) * reach)).to(TYPES[dt])
    caches, slots = _cuda(*_caches(gen, dt, "int4", pages, HK, PAGE, D)), torch.randperm(pages * PAGE, generator=gen)[:T].to(torch.int32)
    none = torch.zeros(0, dtype=TYPES[dt])
    _compile("paged_kv_append", dt, "int4").run(*_cuda(torch.zeros(T, 0, D, dtype=TYPES[dt]), v, v, none, none,
                                                       torch.zeros(1, 0), slots, slots), *caches)
    exact = v.double()
    lowest = torch.stack([p.amin(-1) for p in exact.split(32, -1)], -1).repeat_interleave(32, -1)
    for i in (0, 1):
        pairs = _slot_rows(caches[2 + i].cpu(), slots)
        scale, _ = spread4(pairs, D)
        bound = torch.maximum(scale / 2, 2.0 ** -11 * (lowest.abs() + 15 * scale) + 2.0 ** -21)
        # the code is found in f32: 2^-22 of what it is found from
        off = (values4(_slot_rows(caches[i].cpu(), slots), pairs) - exact).abs()
        assert bool((off <= bound + exact.abs() * 2.0 ** -22).all())
        assert bool((scale == 0).any() and (off > scale / 2 * 1.001).any())  # both ends of the bound are met


# ---- reading back ----------------------------------------------------------------------

READ_CASES = [
    # dtype, cache, T, HK, D, page size, pages
    ("f16", "int4", 1, 8, 128, 16, 3), ("bf16", "int4", 77, 2, 64, 32, 4), ("f16", "int4", 30, 1, 80, 8, 5),
    ("bf16", "int4", 9, 3, 512, 4, 7), ("f16", "int4", 5, 2, 8, 16, 2), ("bf16", "fp8", 33, 2, 128, 16, 4),
    ("f16", "fp8", 7, 1, 264, 2, 9), ("f16", "same", 50, 4, 96, 64, 2), ("bf16", "same", 3, 1, 256, 1, 40),
    ("bf16", "int4", 4001, 8, 128, 16, 300), ("f16", "fp8", 3000, 4, 64, 64, 64), ("f16", "int4", 0, 2, 64, 16, 2),
    ("bf16", "same", 2049, 7, 80, 128, 17), ("f16", "fp8", 4, 0, 64, 16, 2), ("bf16", "int4", 6, 2, 64, 16, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", READ_CASES, ids=lambda c: "-".join(map(str, c)))
def test_paged_kv_read(gpu, case):
    dt, cache, T, HK, D, PAGE, pages = case
    gen = _gen(5)
    row = D // 2 if cache == "int4" else D
    caches = _caches(gen, dt, cache, pages, HK, PAGE, D, extra=16 + -(HK * PAGE * row) % 16)
    count = pages * PAGE
    slots = torch.randint(0, max(count, 1), (T,), generator=gen, dtype=torch.int32)  # some twice
    if T > 3:
        slots[0], slots[2], slots[3] = -1, count, -2 ** 31
    inside = (slots >= 0) & (slots < count)
    art = _compile("paged_kv_read", dt, cache)
    got = art.run(*_cuda(*caches, slots))
    # into rows of wider ones
    wide = torch.full((T, 2, HK, D), 7.0, dtype=TYPES[dt], device="cuda")
    art(*_cuda(*caches, slots), wide[:, 0], wide[:, 1])
    for i, out in enumerate(got):
        want = torch.zeros(T, HK, D, dtype=TYPES[dt])
        if int(inside.sum()):
            params = _slot_rows(caches[2 + i], slots[inside]) if len(caches) > 2 else None
            rows = _values(cache, _slot_rows(caches[i], slots[inside]), params)
            want[inside] = rows.float().to(TYPES[dt])  # an f32 product or fused sum, rounded once more
        assert torch.equal(out.cpu(), want)
        assert torch.equal(wide[:, i].cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_from_8_bits_to_4_and_back(gpu, dt):
    """Tokens of an 8-bit cache read out, appended to a 4-bit one as they are, and read out of that."""
    T, HK, D, PAGE, pages = 100, 2, 128, 16, 9
    gen = _gen(8)
    eight, four = _cuda(*_caches(gen, dt, "fp8", pages, HK, PAGE, D)), _cuda(*_caches(gen, dt, "int4", pages, HK, PAGE, D))
    first, second = _cuda(*(torch.randperm(pages * PAGE, generator=gen)[:T].to(torch.int32) for _ in range(2)))
    k, v = _compile("paged_kv_read", dt, "fp8").run(*eight, first)
    none, q = torch.zeros(0, dtype=TYPES[dt], device="cuda"), torch.zeros(T, 0, D, dtype=TYPES[dt], device="cuda")
    _compile("paged_kv_append", dt, "int4").run(q, k, v, none, none, torch.zeros(1, 0, device="cuda"), second, second, *four)
    for out, x in zip(_compile("paged_kv_read", dt, "int4").run(*four, second), (k.cpu(), v.cpu())):
        code, pairs = quantize4(x)
        assert torch.equal(out.cpu(), values4(pack4(code), pairs).float().to(TYPES[dt]))


# ---- attention -------------------------------------------------------------------------

def ref_attention(q, caches, cache, table, q_offsets, kv_lens, scale, causal, window, cap=0.0, slopes=None, prefix=None,
                  fine=False):
    """(out [T, HQ, D], tolerance) in f64; rows of no sequence are NaN in out."""
    T, HQ, D = q.shape
    pages, HK, PAGE = caches[0].shape[:3]
    u = HALF_STEP[q.dtype]
    weight = 2.0 ** -11 if cache == "int4" else u        # of the weights' type
    narrow = 2.0 ** -11 if cache == "int4" and not fine else 0.0  # of a value in 4 bits
    out = torch.full((T, HQ, D), float("nan"), dtype=torch.float64)
    tol = torch.zeros((T, HQ, D), dtype=torch.float64)
    for s in range(kv_lens.numel()):
        start = min(max(int(q_offsets[s]), 0), T)
        n = max(min(int(q_offsets[s + 1]), T) - start, 0)
        kv = min(max(int(kv_lens[s]), 0), table.shape[1] * PAGE if pages else 0)
        if not n:
            continue
        if not kv:
            out[start:start + n] = 0
            continue
        ids = (table[s, :-(-kv // PAGE)].to(torch.int64) & 0xffffffff).clamp(max=pages - 1)
        rows = [_values(cache, caches[i][ids], caches[2 + i][ids] if len(caches) > 2 else None)
                .transpose(1, 2).reshape(-1, HK, D)[:kv] for i in (0, 1)]
        p, t = torch.arange(kv - n, kv)[:, None], torch.arange(kv)[None]
        seen = torch.ones(n, kv, dtype=torch.bool)
        if causal:
            seen &= (t <= p) | (t < (int(prefix[s]) if prefix is not None else 0))
        if window:
            seen &= t > p - window
        for h in range(HQ):
            qh, k, v = q[start:start + n, h].double(), rows[0][:, h // (HQ // HK)], rows[1][:, h // (HQ // HK)]
            logit = qh @ k.T * scale
            more = torch.zeros(n, 1, dtype=torch.float64)  # of a score, absolute
            if cap:
                logit = cap * torch.tanh(logit / cap)
                more += cap * 2.0 ** -21
            if slopes is not None:
                far = float(slopes[h].abs()) * (t - p).abs().double()
                logit = logit - float(slopes[h]) * (t - p).abs().double()
                more += 3 * 2.0 ** -24 * far.masked_fill(~seen, 0).amax(-1, keepdim=True)
            w = torch.softmax(logit.masked_fill(~seen, -math.inf), -1).masked_fill(~seen, 0.0)
            if v.isfinite().all():
                o, size, big = w @ v, w @ v.abs(), v.abs().amax(0)
            else:  # what a row does not see does not reach it, whatever it holds
                o = torch.stack([w[i, seen[i]] @ v[seen[i]] for i in range(n)])
                size = torch.stack([w[i, seen[i]] @ v[seen[i]].abs() for i in range(n)])
                big = torch.stack([v[seen[i]].abs().amax(0) if seen[i].any() else v.new_zeros(D) for i in range(n)])
            off = (qh.abs() @ k.abs().nan_to_num(0, 0, 0).T * abs(scale)).masked_fill(~seen, 0).amax(-1, keepdim=True)
            many = seen.sum(-1, keepdim=True).double()
            out[start:start + n, h] = o
            slack = weight + 2 * (D + 4) * 2.0 ** -24 * off + 2.0 ** -21 + 2 * many * 2.0 ** -24 + 2 * more
            slack = slack + torch.expm1(2 * narrow * off) + narrow
            tol[start:start + n, h] = size * slack + o.abs() * u + (many * 2.0 ** -25 * big if weight == 2.0 ** -11 else 0)
            tol[start:start + n, h] += 2.0 ** -25 if u == 2.0 ** -11 else 0
    return out, tol


def _inputs(seed, dt, cache, lens, HQ, HK, D, PAGE, poison=True, q_std=1.5, spare=0, fine=True):
    """Ragged sequences over shuffled pages: (q, caches, table, offsets, lengths). What no sequence reaches is NaN,
    unused table entries -1."""
    gen = _gen(seed)
    T = sum(n for n, _ in lens)
    need = [-(-kv // PAGE) for _, kv in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=gen)
    q = _randn(gen, T + spare, HQ, D, dtype=TYPES[dt], std=q_std)
    row = D // 2 if cache == "int4" else D
    caches = _caches(gen, dt, cache, pages, HK, PAGE, D, extra=16 + -(HK * PAGE * row) % 16, fine=fine)
    table = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
    live = torch.zeros(pages, PAGE, dtype=torch.bool)
    at = 0
    for s, ((_, kv), n) in enumerate(zip(lens, need)):
        table[s, :n] = order[at:at + n].to(torch.int32)
        live[order[at:at + n]] = (torch.arange(n * PAGE) < kv).view(n, PAGE)
        at += n
    if poison:
        for c in caches:
            dead = ~live[:, None].expand(c.shape[:3])
            if c.dtype is F8:
                c.view(torch.uint8)[dead] = 0x7f
            elif c.dtype is torch.uint8:
                c[dead] = 0xff
            else:
                c[dead] = float("nan")
    offsets = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32)
    return q, caches, table, offsets, torch.tensor([kv for _, kv in lens], dtype=torch.int32)


def _attend(inputs, dt, cache, scale, causal=True, window=0, out=None, cap=0.0, slopes=None, prefix=None, biased=None):
    q, caches, *rest = inputs
    biased = (cap or slopes is not None or prefix is not None) if biased is None else biased
    forms = {"CAUSAL": causal, "WINDOW": window, **({"SOFTCAP": cap} if biased else {})}
    art = _compile(("biased_" if biased else "") + "paged_attention", dt, cache, **forms)
    more = ()
    if biased:
        more = (torch.zeros(0) if slopes is None else slopes, torch.zeros(0, dtype=torch.int32) if prefix is None else prefix)
    device = _cuda(q, *caches, *rest, *more)
    if out is None:
        return art.run(*device, scale)
    art(*device, out, scale)
    return out


def _prefixes(lens, at):
    """None, whole and partial prefixes, some past the sequence's end."""
    return torch.tensor([(0, kv // 3, kv, kv + 5, -4, max(kv - n, 0) + n // 2, 1)[(s + at) % 7]
                         for s, (n, kv) in enumerate(lens)], dtype=torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("at", range(len(ATTENTION_CASES)))
def test_paged_attention_int4(gpu, at):
    dt, _, lens, HQ, HK, D, PAGE, causal, window = ATTENTION_CASES[at]
    fine = at % 4 != 3
    inputs = _inputs(21, dt, "int4", lens, HQ, HK, D, PAGE, fine=fine)
    want, tol = ref_attention(inputs[0], inputs[1], "int4", *inputs[2:], D ** -0.5, causal, window, fine=fine)
    _close(_attend(inputs, dt, "int4", D ** -0.5, causal, window), want, tol, at)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "fp8", "int4"])
@pytest.mark.parametrize("at", range(len(ATTENTION_CASES)))
def test_biased_paged_attention(gpu, at, cache):
    """Every form alone and with the others."""
    dt, _, lens, HQ, HK, D, PAGE, causal, window = ATTENTION_CASES[at]
    forms = (at + {"same": 0, "fp8": 3, "int4": 5}[cache]) % 7 + 1
    cap = (5.0, 20.0)[at % 2] if forms & 1 else 0.0
    slopes = (2.0 ** (-8.0 * torch.arange(1, HQ + 1) / HQ)).float() if forms & 2 else None
    prefix = _prefixes(lens, at) if forms & 4 else None
    inputs = _inputs(23, dt, cache, lens, HQ, HK, D, PAGE, q_std=4.0 if cap else 1.5)
    want, tol = ref_attention(inputs[0], inputs[1], cache, *inputs[2:], D ** -0.5, causal, window, cap, slopes, prefix,
                              fine=True)
    _close(_attend(inputs, dt, cache, D ** -0.5, causal, window, cap=cap, slopes=slopes, prefix=prefix), want, tol, at)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("cache", ["same", "fp8", "int4"])
@pytest.mark.parametrize("forms", range(5))
def test_chunks_beside_short_sequences(gpu, forms, cache, dt):
    """Heads of 64, chunks and sequences on both sides of 16 rows of a head, rows of no sequence before and behind:
    scores without a form, capped, biased by distance, both, and a prefix alone."""
    lens = [(1, 3000), (300, 700), (1, 33), (17, 400), (16, 90), (200, 200), (0, 40), (9, 0), (129, 131), (1, 1), (2, 500)]
    HQ, HK, window = ((12, 12, 0), (14, 2, 150))[(forms + (dt == "f16")) % 2]
    inputs = list(_inputs(41, dt, cache, lens, HQ, HK, 64, 16, q_std=4.0 if forms in (1, 3) else 1.5, spare=38))
    inputs[3] = inputs[3] + 20
    more = {"cap": 20.0 if forms in (1, 3) else 0.0,
            "slopes": (2.0 ** (-8.0 * torch.arange(1, HQ + 1) / HQ)).float() if forms in (2, 3) else None,
            "prefix": _prefixes(lens, forms) if forms >= 3 else None}
    want, tol = ref_attention(inputs[0], inputs[1], cache, *inputs[2:], 0.125, True, window, fine=True, **more)
    out = torch.full_like(inputs[0], 7.0, device="cuda")
    got = _attend(inputs, dt, cache, 0.125, True, window, out=out, **more).cpu()
    inside = ~want.isnan().flatten(1).any(1)
    assert int(inside.sum()) == sum(n for n, _ in lens) and bool((got[~inside] == 7).all())
    _close(got[inside], want[inside], tol[inside])


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("lens", [[(1, 900), (1, 33)], [(70, 200)]], ids=str)
def test_biased_without_forms_is_the_plain_attention(gpu, cache, lens):
    inputs = _inputs(24, "bf16", cache, lens, 8, 2, 128, 16)
    assert torch.equal(_attend(inputs, "bf16", cache, 0.1, biased=True), _attend(inputs, "bf16", cache, 0.1))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("std", [1e-6, 3e3])
@pytest.mark.parametrize("lens,D", [([(1, 200)], 64), ([(4, 90)], 128), ([(80, 200)], 96), ([(3, 70)], 80)], ids=str)
def test_paged_attention_int4_queries_of_many_sizes(gpu, dt, std, lens, D):
    """Rows far below and above one, and a row that holds both ends."""
    inputs = _inputs(25, dt, "int4", lens, 4, 2, D, 16, q_std=std)
    inputs[0][-1, :, ::3] *= 2.0 ** -9
    if dt == "bf16" and std < 1:
        inputs[0][-1] *= 2.0 ** -60
        inputs[0][0, 0] = 0
    scale = 0.3 / max(std, 1.0)
    want, tol = ref_attention(inputs[0], inputs[1], "int4", *inputs[2:], scale, True, 0, fine=True)
    _close(_attend(inputs, dt, "int4", scale), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("new,HQ,D", [(1, 4, 128), (5, 4, 64), (64, 4, 128), (200, 2, 64), (40, 2, 256), (3, 2, 80)])
def test_int4_masked_values_do_not_reach_a_row(gpu, new, HQ, D, dt, biased):
    """Groups whose values are not finite (a NaN, and finite pairs whose sum is no f16): rows that do not see them
    are finite, those that do are not, in those columns alone."""
    kv, PAGE, HK = new + 70, 16, 2
    inputs = _inputs(26, dt, "int4", [(new, kv)], HQ, HK, D, PAGE, poison=False)
    q, caches, table, offsets, lens = inputs
    last = kv - 1
    page, place = int(table[0, last // PAGE]), last % PAGE
    caches[3][page, :, place, 0] = torch.tensor([0.0, float("nan")], dtype=torch.float16)
    if new > 1:  # the second group of the token before: infinite for some codes
        page, place = int(table[0, (last - 1) // PAGE]), (last - 1) % PAGE
        caches[3][page, :, place, 1] = torch.tensor([0.0, float("inf")], dtype=torch.float16)
    slopes = torch.full((HQ,), 0.01) if biased else None
    out = _attend(inputs, dt, "int4", D ** -0.5, slopes=slopes).cpu()
    assert bool(out[-1, :, :32].isnan().all()) and bool(out[-1, :, 64 if new > 1 else 32:].isfinite().all())
    if new > 1:
        assert bool(out[:-1, :, :32].isfinite().all()) and bool((out[-2:, :, 32:64] == float("inf")).all())
    if new > 2:
        want, tol = ref_attention(q, caches, "int4", *inputs[2:], D ** -0.5, True, 0, slopes=slopes, fine=True)
        _close(out[:-2], want[:-2], tol[:-2])


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "fp8", "int4"])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_bad_pages_and_lengths(gpu, cache, new):
    """Page ids, lengths and prefixes outside the cache are clamped: the formula over the clamped ones."""
    inputs = list(_inputs(27, "f16", cache, [(new, 90), (new, 60)], 4, 2, 64, 16, poison=False))
    inputs[2][0, 1], inputs[2][1, 0] = 10 ** 6, -7
    inputs[4][1] = 10 ** 6
    prefix = torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    for forms in ({}, {"prefix": prefix, "cap": 9.0}):
        want, tol = ref_attention(inputs[0], inputs[1], cache, *inputs[2:], 0.125, True, 0, fine=True, **forms)
        _close(_attend(inputs, "f16", cache, 0.125, **forms), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "int4"])
@pytest.mark.parametrize("lens", [[(1, 130), (1, 70)], [(6, 130), (5, 70)], [(70, 200), (90, 120)]], ids=str)
def test_rows_that_belong_to_no_sequence(gpu, lens, cache):
    inputs = list(_inputs(28, "bf16", cache, lens, 8, 2, 64, 16, spare=9))
    inputs[3] = inputs[3] + 4
    prefix = torch.tensor([50, 0], dtype=torch.int32)
    T = inputs[0].shape[0]
    out = torch.full((T, 2, 8, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    for forms in ({}, {"prefix": prefix}):
        want, tol = ref_attention(inputs[0], inputs[1], cache, *inputs[2:], 0.125, True, 0, fine=True, **forms)
        _attend(inputs, "bf16", cache, 0.125, out=out[:, 0], **forms)
        got = out[:, 0].cpu()
        inside = ~want.isnan().flatten(1).any(1)
        assert bool((got[~inside] == 7).all()) and bool((out[:, 1] == 7).all())
        _close(got[inside], want[inside], tol[inside])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 80, 128])
def test_scores_past_the_cap(gpu, D):
    """Scores far past the cap, infinite ones among them, are the cap: weights of tokens at it are alike."""
    inputs = list(_inputs(29, "bf16", "same", [(2, 100), (100, 300)], 4, 2, D, 16, q_std=1e4))
    inputs[1][0] *= 100
    inputs[0][0, 0, 0] = 1e38
    want, tol = ref_attention(inputs[0], inputs[1], "same", *inputs[2:], 1.0, True, 0, cap=3.0)
    # a score of no size beside the cap would pass its own error on; none is as small here
    tol = (want.abs() + inputs[1][1].float().nan_to_num(0).abs().max().double()) * (2.0 ** -8 + 2.0 ** -16) + 2.0 ** -20 * 300
    _close(_attend(inputs, "bf16", "same", 1.0, cap=3.0), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [2.0 ** -100, 0.01, 100.0, 4096.0])
@pytest.mark.parametrize("new,D", [(1, 64), (40, 128), (300, 128), (5, 256), (9, 80)])
@pytest.mark.parametrize("cache", ["same", "fp8", "int4"])
def test_caps_of_many_sizes(gpu, cap, new, D, cache):
    """From caps that leave all scores alike to caps that leave them as they are, with slopes and without."""
    inputs = _inputs(35, "f16", cache, [(new, new + 150)], 4, 2, D, 16, q_std=4.0)
    for slopes in (None, torch.tensor([0.5, 0.0, 0.01, 1.0])):
        want, tol = ref_attention(inputs[0], inputs[1], cache, *inputs[2:], D ** -0.5, True, 0, cap, slopes, fine=True)
        _close(_attend(inputs, "f16", cache, D ** -0.5, cap=cap, slopes=slopes), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.2, 3e-36, 3.0])
@pytest.mark.parametrize("lens", [[(1, 200)], [(4, 90)], [(80, 200)]], ids=str)
@pytest.mark.parametrize("cache", ["same", "fp8", "int4"])
def test_scales(gpu, lens, scale, cache):
    inputs = _inputs(36, "bf16", cache, lens, 4, 2, 128, 16, q_std=0.5)
    for forms in ({}, {"cap": 7.0}, {"slopes": torch.tensor([0.5, 0.0, 0.01, -0.02])},
                  {"cap": 2.0, "slopes": torch.tensor([0.5, 0.0, 0.01, 1.0]), "prefix": torch.tensor([70], dtype=torch.int32)}):
        want, tol = ref_attention(inputs[0], inputs[1], cache, *inputs[2:], scale, True, 0, fine=True, **forms)
        _close(_attend(inputs, "bf16", cache, scale, **forms), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 6, 90])
def test_int4_queries_that_are_not_finite(gpu, dt, new):
    """A query that holds an infinity or NaN leaves the other rows alone."""
    inputs = _inputs(37, dt, "int4", [(new, 120), (new, 40)], 4, 2, 64, 16)
    want, tol = ref_attention(inputs[0], inputs[1], "int4", *inputs[2:], 0.125, True, 0, fine=True)
    inputs[0][0, 1, 5], inputs[0][-1, 2, 9] = float("inf"), float("nan")
    out = _attend(inputs, dt, "int4", 0.125).cpu()
    bad = torch.zeros(2 * new, 4, dtype=torch.bool)
    bad[0, 1], bad[-1, 2] = True, True
    assert bool(out[bad].isnan().any(-1).all())
    _close(out[~bad], want[~bad], tol[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[(1, 300)], [(5, 90)], [(80, 200)]], ids=str)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_int4_pairs_of_many_sizes(gpu, dt, lens):
    """Scales below zero, zero, of f16's subnormals and large ones; lowest values far off."""
    inputs = _inputs(38, dt, "int4", lens, 4, 2, 128, 16)
    for i in (2, 3):
        pairs = inputs[1][i]
        pairs[..., 0, 0] = -pairs[..., 0, 0].abs()
        pairs[..., 1, 0] = 0
        pairs[..., 2, :] = torch.tensor([3 * 2.0 ** -24, -5 * 2.0 ** -24])
        pairs[..., 3, :] = torch.tensor([4096.0, -30720.0]) if i == 3 else torch.tensor([1.0, 32.0])
    want, tol = ref_attention(inputs[0], inputs[1], "int4", *inputs[2:], 0.02, True, 0, fine=True)
    _close(_attend(inputs, dt, "int4", 0.02), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40, 300])
def test_long_distances(gpu, new):
    """Slopes so steep that only the nearest tokens count, and none at all for some heads, over a long cache."""
    inputs = _inputs(30, "f16", "int4", [(new, 30011)], 4, 2, 64, 64)
    slopes = torch.tensor([20.0, 0.0, 1e-4, -0.001])
    want, tol = ref_attention(inputs[0], inputs[1], "int4", *inputs[2:], 0.125, True, 0, slopes=slopes, fine=True)
    _close(_attend(inputs, "f16", "int4", 0.125, slopes=slopes), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "int4"])
@pytest.mark.parametrize("new", [1, 40, 300])
def test_distances_past_24_bits(gpu, new, cache):
    """Positions that no f32 tells apart: with steep slopes the tokens behind 2^24 others give what they give alone
    (weights of tokens 1024 and more away are below 2^-1000)."""
    HQ, HK, D, PAGE, near = 4, 2, 64, 256, 2048
    q, caches, table, offsets, _ = _inputs(39, "f16", cache, [(new, near)], HQ, HK, D, PAGE, poison=False)
    slopes = torch.tensor([1.0, 2.0, 1.5, 30.0])
    far = (1 << 24) + 3 * PAGE
    long = torch.cat((torch.zeros(1, far // PAGE, dtype=torch.int32), table), 1)
    # rows whose last tokens are as near as 1024: the others see what lies before
    want, tol = ref_attention(q, caches, cache, table, offsets, torch.tensor([near], dtype=torch.int32), 0.125, True, 0,
                              slopes=slopes, fine=True)
    got = _attend((q, caches, long, offsets, torch.tensor([far + near], dtype=torch.int32)), "f16", cache, 0.125, slopes=slopes)
    # sums of as many terms of f32, none of which counts but the nearest
    _close(got, want, tol + 2.0 ** -20)


@pytest.mark.gpu
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("new,HQ,kv,D", [(1, 4, 20000, 64), (7, 8, 9000, 96), (1, 2, 9000, 256), (352, 8, 5000, 128)])
def test_split_and_unsplit(gpu, new, HQ, kv, D, biased):
    """With a workspace and without: both by the formula; twice the same, bit for bit."""
    inputs = _inputs(31, "bf16", "int4", [(new, kv)], HQ, 1, D, 64)
    forms = {"cap": 30.0, "prefix": torch.tensor([kv], dtype=torch.int32)} if biased else {}
    want, tol = ref_attention(inputs[0], inputs[1], "int4", *inputs[2:], D ** -0.5, True, 0, fine=True, **forms)
    got = _attend(inputs, "bf16", "int4", D ** -0.5, **forms)
    _close(got, want, tol)
    assert torch.equal(got, _attend(inputs, "bf16", "int4", D ** -0.5, **forms))
    q, caches, table, offsets, lens = _cuda(inputs[0]) + [_cuda(*inputs[1])] + _cuda(*inputs[2:])
    alone = torch.empty_like(q)
    k, v, kg, vg = caches
    prefix = forms.get("prefix")
    prefix = None if prefix is None else prefix.cuda()
    _native.call("intent_biased_paged_attention", q.data_ptr(), new, HQ, q.stride(0), 1, 2, k.data_ptr(), k.stride(0),
                 v.data_ptr(), v.stride(0), kg.data_ptr(), kg.stride(0), vg.data_ptr(), vg.stride(0), k.shape[0], 1, 64, D,
                 table.data_ptr(), 1, table.shape[1], table.stride(0), offsets.data_ptr(), lens.data_ptr(), D ** -0.5, 1, 0,
                 forms.get("cap", 0.0), None, None if prefix is None else prefix.data_ptr(), alone.data_ptr(),
                 alone.stride(0), None, 0, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    _close(alone, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 80, 256])
def test_without_a_cache(gpu, D):
    """A table of no pages, and a cache of none: nothing is seen, every row is zero."""
    for new in (1, 5, 90):
        inputs = list(_inputs(33, "f16", "int4", [(new, 40)], 4, 2, D, 16, poison=False))
        forms = {"prefix": torch.tensor([30], dtype=torch.int32), "slopes": torch.ones(4)}
        inputs[2] = inputs[2][:, :0]
        assert bool((_attend(inputs, "f16", "int4", 0.1) == 0).all() and (_attend(inputs, "f16", "int4", 0.1, **forms) == 0).all())
        inputs[2] = torch.zeros(1, 3, dtype=torch.int32)
        inputs[1] = [c[:0] for c in inputs[1]]
        assert bool((_attend(inputs, "f16", "int4", 0.1) == 0).all() and (_attend(inputs, "f16", "int4", 0.1, **forms) == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "int4"])
@pytest.mark.parametrize("new", [1, 40])
def test_far_pages(gpu, new, cache):
    """Pages past 2^31 bytes from the cache's start."""
    HK, D, PAGE = 2, 64, 16
    inputs = list(_inputs(34, "f16", cache, [(new, 100)], 4, HK, D, PAGE, poison=False))
    caches, far = inputs[1], []
    pages = caches[0].shape[0]
    step = (1 << 31) // (pages - 1) // 16 * 16 + 4096
    for c in caches:  # the same rows, each page `step` elements behind the last
        flat = torch.zeros((pages - 1) * step + c[0].numel(), dtype=c.dtype, device="cuda")
        view = flat.as_strided(c.shape, (step, *c.contiguous().stride()[1:]))
        view.copy_(c)
        far.append(view)
    prefix = torch.tensor([60], dtype=torch.int32)
    for forms in ({}, {"prefix": prefix}):
        near = _attend(inputs, "f16", cache, 0.125, **forms)
        assert torch.equal(_attend([inputs[0], far, *inputs[2:]], "f16", cache, 0.125, **forms), near)
    slots = torch.arange(pages * PAGE, dtype=torch.int32)
    read = _compile("paged_kv_read", "f16", cache)
    assert all(torch.equal(a, b) for a, b in zip(read.run(*far, slots.cuda()), read.run(*_cuda(*caches), slots.cuda())))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [7, 900])
def test_keys_and_values_of_one_allocation(gpu, T):
    """Append, attention and reading over kv[:, 0] and kv[:, 1]: both halves get their own rows, all others stay."""
    HQ, HK, D, PAGE, pages = 8, 2, 64, 16, 70
    gen = _gen(45)
    heads = _heads(46, "bf16", T, HQ, HK, D, 0, "")
    slots = torch.randperm(pages * PAGE, generator=gen)[:T].to(torch.int32)
    k, v, kg, vg = _caches(gen, "bf16", "int4", pages, HK, PAGE, D)
    alone = _cuda(*[c.contiguous() for c in (k, v, kg, vg)])
    views = [t[:, i] for t in _cuda(torch.stack((k, v), 1), torch.stack((kg, vg), 1)) for i in (0, 1)]
    append, args = _compile("paged_kv_append", "bf16", "int4"), _cuda(*heads, slots)
    for _ in range(2):  # bound, and known
        q_out = append.run(*args, *views)
    assert torch.equal(q_out, append.run(*args, *alone))
    assert all(torch.equal(got, want) for got, want in zip(views, alone))
    rest = _cuda(torch.randperm(pages, generator=gen).to(torch.int32)[None], torch.tensor([0, T], dtype=torch.int32),
                 torch.tensor([pages * PAGE - 3], dtype=torch.int32))
    attend, read = _compile("paged_attention", "bf16", "int4"), _compile("paged_kv_read", "bf16", "int4")
    assert torch.equal(attend.run(q_out, *views, *rest, 0.125), attend.run(q_out, *alone, *rest, 0.125))
    assert all(torch.equal(a, b) for a, b in zip(read.run(*views, args[-1]), read.run(*alone, args[-1])))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,cache", [("f16", "int4"), ("bf16", "int4"), ("bf16", "fp8"), ("f16", "same")])
def test_decoding_loop(gpu, dt, cache):
    """A prompt in two chunks and three decoding steps of two sequences, as a program runs them: projection, append,
    attention with capped and distance-biased scores, output projection, each step over the cache that the steps
    before left; the whole cache read back at the end."""
    gen = _gen(40)
    HQ, HK, D, PAGE, H = 8, 2, 64, 16, 256
    gemm = intent.compile(intent.gemm if dt == "f16" else intent.bf16_gemm, target=intent.MI355XTarget(0))
    append, read = _compile("paged_kv_append", dt, cache), _compile("paged_kv_read", dt, cache)
    attend = _compile("biased_paged_attention", dt, cache, SOFTCAP=20.0)
    w_qkv, w_out = (_randn(gen, *s, dtype=TYPES[dt], std=H ** -0.5).cuda() for s in ((H, (HQ + 2 * HK) * D), (HQ * D, H)))
    weights = [(1 + _randn(gen, D, std=0.1)).to(TYPES[dt]) for _ in range(2)]
    slopes = (2.0 ** -torch.arange(1, HQ + 1).float())
    angle = torch.outer(torch.arange(200, dtype=torch.float64), 10000.0 ** (-torch.arange(0, D, 2).double() / D))
    table_cs = torch.cat((angle.cos(), angle.sin()), 1).float()
    caches = _cuda(*_caches(gen, dt, cache, 20, HK, PAGE, D))
    pages = torch.randperm(20, generator=gen).to(torch.int32).view(2, 10)
    prefix = torch.tensor([25, 0], dtype=torch.int32)
    device = _cuda(*weights, table_cs)
    lengths = [0, 0]
    keys, values, places = [], [], []
    for news in ((37, 20), (30, 1), (1, 1), (1, 1), (1, 1)):
        T = sum(news)
        qkv = gemm.run(_randn(gen, T, H, dtype=TYPES[dt]).cuda(), w_qkv)
        q, k, v = (p.unflatten(1, (-1, D)) for p in qkv.split((HQ * D, HK * D, HK * D), 1))
        at = [torch.arange(n, n + m) for n, m in zip(lengths, news)]
        slots = torch.cat([pages[s][t // PAGE].long() * PAGE + t % PAGE for s, t in enumerate(at)]).to(torch.int32)
        positions = torch.cat(at).to(torch.int32)
        lengths = [n + m for n, m in zip(lengths, news)]
        q_out = append.run(q, k, v, *device, *_cuda(positions, slots), *caches)
        offsets, kv = torch.tensor([0, news[0], T], dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32)
        out = attend.run(q_out, *caches, *_cuda(pages, offsets, kv, slopes, prefix), D ** -0.5)
        want, tol = ref_attention(q_out.cpu(), [c.cpu() for c in caches], cache, pages, offsets, kv, D ** -0.5, True, 0, 20.0,
                                  slopes, prefix)
        _close(out, want, tol, news)
        assert bool(torch.isfinite(gemm.run(out.view(T, HQ * D), w_out)).all())
        key, _ = ref_norm_rope(k.cpu(), weights[1], table_cs, positions, 1e-6, False)
        keys.append(key), values.append(v.cpu().double()), places.append(slots)
    got = read.run(*caches, torch.cat(places).cuda())
    for out, x in zip(got, (torch.cat(keys), torch.cat(values))):
        # the format's step (4 bits: of a group's range; 8: of the value, or of the subnormals'; 16: none), the
        # output's, and f32 arithmetic before
        span = torch.stack([p.amax(-1) - p.amin(-1) for p in x.split(32, -1)], -1).repeat_interleave(32, -1)
        step = {"int4": span / 30 + span * 2.0 ** -10 + x.abs().amax(-1, keepdim=True) * 2.0 ** -10,
                "fp8": torch.maximum(x.abs() * 2.0 ** -4, x.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -10), "same": 0}[cache]
        _close(out, x, step + (x.abs() + step) * HALF_STEP[TYPES[dt]] + x.abs().amax(-1, keepdim=True) * 2.0 ** -17)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 5, 70])
def test_captured_and_replayed(gpu, new):
    """Append, attention and reading back of a step in a graph, replayed over lengths, slots, slopes and prefixes that
    change in place, with eager calls of the same operators in between: every replay equals the eager step."""
    HQ, HK, D, PAGE = 8, 2, 128, 16
    heads = list(_cuda(*_heads(41, "bf16", 2 * new, HQ, HK, D, D, "qk", length=600)))
    inputs = _inputs(42, "bf16", "int4", [(new, 500), (new, 400)], HQ, HK, D, PAGE, poison=False)
    caches, (table, offsets, kv) = _cuda(*inputs[1]), _cuda(*inputs[2:])
    slots = torch.zeros(2 * new, dtype=torch.int32, device="cuda")
    slopes, prefix = torch.ones(HQ, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    q_out, out = (torch.empty(2 * new, HQ, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    rows = [torch.empty(2 * new, HK, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    calls = [_compile("paged_kv_append", "bf16", "int4").prepare(*heads, slots, *caches, outputs=(q_out,)),
             _compile("biased_paged_attention", "bf16", "int4", SOFTCAP=10.0).prepare(
                 q_out, *caches, table, offsets, kv, slopes, prefix, 0.0884, outputs=(out,)),
             _compile("paged_kv_read", "bf16", "int4").prepare(*caches, slots, outputs=tuple(rows))]

    def place(first, second):
        at = torch.cat([torch.arange(n - new, n) for n in (first, second)])
        row = torch.arange(2).repeat_interleave(new)
        slots.copy_((inputs[2][row, at // PAGE].long() * PAGE + at % PAGE).to(torch.int32))
        kv.copy_(torch.tensor([first, second], dtype=torch.int32))
        prefix.copy_(torch.tensor([first // 2, second], dtype=torch.int32))
        slopes.copy_(torch.rand(HQ) * 0.1)
        heads[6].copy_(at.to(torch.int32))

    place(500, 400)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        [c.launch() for c in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        [c.launch() for c in calls]
    for first, second in ((500, 400), (new, 399), (256, 17 + new), (511, 410)):
        place(first, second)
        [c.launch() for c in calls]
        kept = [t.clone() for t in (out, *rows, *caches)]
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, *rows, *caches), kept)), (first, second)


@pytest.mark.gpu
def test_two_graphs_of_unprepared_calls(gpu):
    """run() captured twice (decoding and a chunk, both split), the graphs replayed in turn and at once on two
    streams, with eager calls between."""
    forms = (torch.rand(8, generator=_gen(1)) * 0.01, torch.zeros(0, dtype=torch.int32))
    art = _compile("biased_paged_attention", "bf16", "int4", SOFTCAP=30.0)
    sets = [_inputs(70 + i, "bf16", "int4", lens, 8, 2, 128, 16, poison=False)
            for i, lens in enumerate(([(1, 3000), (1, 900)], [(60, 2500)]))]
    device = [[*_cuda(s[0], *s[1], *s[2:], *forms), 0.0884] for s in sets]
    for d in device:
        art.run(*d)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for d in device:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(art.run(*d))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for cut in (0, 700, 1300, 0):
        eager = []
        for d, s in zip(device, sets):
            d[7].copy_((s[4] - cut).clamp(min=0).to(torch.int32))
            eager.append(art.run(*d))
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for i, graph in enumerate(graphs):
            assert torch.equal(outs[i], eager[i]), (cut, i)
            outs[i].fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], eager[i]), (cut, i)


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    """Calls of one artifact on two streams, in flight together, share nothing."""
    art = _compile("paged_attention", "f16", "int4")
    sets = [_inputs(50 + i, "f16", "int4", [(1, 2000 - 300 * i)] * 3, 8, 2, 128, 16) for i in range(2)]
    device = [[*_cuda(s[0], *s[1], *s[2:]), 0.0884] for s in sets]
    alone = [art.run(*d) for d in device]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = [[], []]
    for _ in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(art.run(*device[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(r, alone[i]) for r in results[i])


@pytest.mark.gpu
def test_as_torch_ops(gpu):
    """Append, read and biased attention as torch operators, the cache as an argument that they change."""
    T, HQ, HK, D, PAGE = 5, 4, 2, 64, 16
    heads = _cuda(*_heads(9, "f16", T, HQ, HK, D, D, "qk"))
    caches = _cuda(*[c.contiguous() for c in _caches(_gen(3), "f16", "int4", 3, HK, PAGE, D)])
    other = [c.clone() for c in caches]
    slots = torch.arange(T, dtype=torch.int32, device="cuda") * 3
    append, read = _compile("paged_kv_append", "f16", "int4"), _compile("paged_kv_read", "f16", "int4")
    attend = _compile("biased_paged_attention", "f16", "int4", SOFTCAP=30.0)
    want = append.run(*heads, slots, *caches)
    assert torch.equal(append.as_torch_op("intent_test_forms::append")(*heads, slots, *other), want)
    assert all(torch.equal(a, b) for a, b in zip(caches, other))
    for a, b in zip(read.as_torch_op("intent_test_forms::read")(*caches, slots), read.run(*caches, slots)):
        assert torch.equal(a, b)
    rest = _cuda(torch.tensor([[0, 1, 2]], dtype=torch.int32), torch.tensor([0, T], dtype=torch.int32),
                 torch.tensor([40], dtype=torch.int32), torch.ones(HQ), torch.tensor([9], dtype=torch.int32))
    op = attend.as_torch_op("intent_test_forms::attend")
    assert torch.equal(op(want, *caches, *rest, 0.125), attend.run(want, *caches, *rest, 0.125))


# ---- refusals (CPU) --------------------------------------------------------------------

def test_packing():
    code = torch.randint(0, 16, (3, 24), generator=_gen(1))
    assert torch.equal(codes4(pack4(code)), code)
    assert pack4(torch.tensor([1, 2, 3, 4, 5, 6, 7, 8])).tolist() == [0x31, 0x75, 0x42, 0x86]


def test_outputs_are_inferred():
    inputs = _inputs(1, "f16", "int4", [(2, 9), (1, 3)], 4, 2, 80, 4)
    flat = (inputs[0], *inputs[1], *inputs[2:])
    assert runtime_for("paged_attention_int4").infer_outputs((*flat, 0.1)).shape == (3, 4, 80)
    none = torch.zeros(0), torch.zeros(0, dtype=torch.int32)
    assert runtime_for("biased_paged_attention_int4").infer_outputs((*flat, *none, 0.1)).shape == (3, 4, 80)
    k, v = runtime_for("bf16_paged_kv_read_int4").infer_outputs((*inputs[1], torch.zeros(7, dtype=torch.int32)))
    assert k.shape == v.shape == (7, 2, 80) and k.dtype is torch.bfloat16
    q, k, v, *more = _heads(1, "bf16", 5, 6, 2, 80, 32, "qk")
    caches = _caches(_gen(1), "bf16", "int4", 3, 2, 4, 80)
    got = runtime_for("bf16_paged_kv_append_int4").infer_outputs((q, k, v, *more, torch.zeros(5, dtype=torch.int32), *caches))
    assert got.shape == (5, 6, 80)


def test_arguments_are_checked():
    inputs = _inputs(1, "f16", "int4", [(2, 9), (1, 3)], 4, 2, 80, 4)
    flat = [inputs[0], *inputs[1], *inputs[2:], torch.ones(4), torch.zeros(2, dtype=torch.int32)]
    rt = runtime_for("biased_paged_attention_int4", SOFTCAP=9.0)
    rt.infer_outputs((*flat, 0.1))
    for i, bad, error, match in ((1, flat[1][..., :32], ValueError, "must be 40"), (3, flat[3][..., :2, :], ValueError, "must be 3"),
                                 (4, flat[4][..., :1], ValueError, "must be 2"), (8, torch.ones(3), ValueError, "slopes"),
                                 (9, torch.zeros(3, dtype=torch.int32), ValueError, "prefix_lens"),
                                 (8, torch.ones(4).double(), TypeError, "dtype"), (9, torch.zeros(2), TypeError, "dtype"),
                                 (3, flat[3].float(), TypeError, "dtype"), (1, flat[1].to(torch.int8), TypeError, "dtype"),
                                 (6, flat[6][:2], ValueError, "q_offsets")):
        change = list(flat)
        change[i] = bad
        with pytest.raises(error, match=match):
            rt.infer_outputs((*change, 0.1))
    for cap in (-1.0, float("nan"), float("inf"), 1e-40, 5000.0, 1e39):
        with pytest.raises(ValueError, match="SOFTCAP"):
            runtime_for("biased_paged_attention_int4", SOFTCAP=cap).infer_outputs((*flat, 0.1))
    with pytest.raises(ValueError, match="SOFTCAP"):
        runtime_for("paged_attention_int4", SOFTCAP=1.0)
    slots = torch.zeros(3, dtype=torch.int32)
    read = runtime_for("paged_kv_read_int4")
    with pytest.raises(NotImplementedError, match="multiple of 8"):
        read.infer_outputs((*(torch.zeros(2, 1, 4, 30, dtype=torch.uint8),) * 2, *(torch.zeros(2, 1, 4, 2, 2).half(),) * 2, slots))
    with pytest.raises(NotImplementedError, match="power of two"):
        read.infer_outputs((*(torch.zeros(2, 1, 6, 32, dtype=torch.uint8),) * 2, *(torch.zeros(2, 1, 6, 2, 2).half(),) * 2, slots))
    with pytest.raises(ValueError, match="relation"):
        runtime_for("paged_kv_read").infer_outputs((torch.zeros(2, 1, 4, 32).half(), torch.zeros(2, 1, 4, 64).half(), slots))


def test_writes_may_not_overlap(monkeypatch):
    rt = runtime_for("paged_kv_append_int4")
    rt._home = torch.device("cpu")
    monkeypatch.setattr(rt, "_launch", lambda binding: None)
    heads = _heads(1, "f16", 5, 6, 2, 64, 32, "qk")
    k, v, kg, vg = [c.contiguous() for c in _caches(_gen(1), "f16", "int4", 4, 2, 8, 64)]
    slots = torch.zeros(5, dtype=torch.int32)
    rt.run(*heads, slots, k, v, kg, vg)
    for bad, match in (((k, k, kg, vg), "k_cache and v_cache"), ((k, v, kg, kg), "k_groups and v_groups")):
        with pytest.raises(ValueError, match=match):
            rt.run(*heads, slots, *bad)
    read = runtime_for("paged_kv_read")
    read._home = torch.device("cpu")
    monkeypatch.setattr(read, "_launch", lambda binding: None)
    cache = torch.zeros(4, 2, 8, 64).half()
    out = torch.zeros(5, 2, 64).half()
    with pytest.raises(ValueError, match="k_out and v_out"):
        read.launch(cache, cache.clone(), slots, out, out)
    with pytest.raises(ValueError, match="overlap"):
        read.launch(cache, cache.clone(), slots, out, cache.view(-1)[:640].view(5, 2, 64))


def _append4_args(**change):
    a = dict(q=FAKE, T=4, HQ=4, q_ld=256, k=FAKE, HK=2, k_ld=128, v=FAKE, v_ld=128, D=64, qw=FAKE, kw=None, eps=1e-6,
             cs=FAKE, P=8, R=64, cs_ld=64, inter=0, pos=FAKE, slots=FAKE, bf16=0, kc=FAKE, kc_ld=1024, vc=FAKE,
             vc_ld=1024, kg=FAKE, kg_ld=128, vg=FAKE, vg_ld=128, pages=4, page=16, q_out=FAKE, q_out_ld=256, stream=None)
    assert set(change) <= set(a)
    return list({**a, **change}.values())


def _read_args(**change):
    a = dict(format=2, kc=FAKE, kc_ld=1024, vc=FAKE, vc_ld=1024, kg=FAKE, kg_ld=128, vg=FAKE, vg_ld=128, pages=4, HK=2,
             page=16, D=64, slots=FAKE, T=4, bf16=0, k_out=FAKE, k_ld=128, v_out=FAKE, v_ld=128, stream=None)
    assert set(change) <= set(a)
    return list({**a, **change}.values())


def _biased_args(**change):
    a = dict(q=FAKE, T=4, HQ=4, q_ld=256, bf16=0, format=2, kc=FAKE, kc_ld=1024, vc=FAKE, vc_ld=1024, kg=FAKE, kg_ld=128,
             vg=FAKE, vg_ld=128, pages=4, HK=2, page=16, D=64, table=FAKE, S=2, width=3, table_ld=3, offsets=FAKE,
             kv=FAKE, scale=0.1, causal=1, window=0, cap=0.0, slopes=None, prefix=None, out=FAKE, out_ld=256, ws=None,
             ws_bytes=0, stream=None)
    assert set(change) <= set(a)
    return list({**a, **change}.values())


INVALID, ALIGN, UNSUPPORTED = errors.INTENT_ERR_INVALID_ARGUMENT, errors.INTENT_ERR_ALIGNMENT, errors.INTENT_ERR_UNSUPPORTED
A4, RD, BA = ("intent_paged_kv_append_int4", _append4_args), ("intent_paged_kv_read", _read_args), \
    ("intent_biased_paged_attention", _biased_args)


@pytest.mark.parametrize("entry,code,change", [
    (A4, INVALID, dict(kg=None)), (A4, INVALID, dict(vc=None)), (A4, INVALID, dict(kc_ld=1008)), (A4, INVALID, dict(vg_ld=126)),
    (A4, INVALID, dict(pages=1 << 30)), (A4, UNSUPPORTED, dict(page=12)), (A4, UNSUPPORTED, dict(D=68)),
    (A4, ALIGN, dict(kc=FAKE + 8)), (A4, ALIGN, dict(vc_ld=1032)), (A4, ALIGN, dict(kg=FAKE + 2)), (A4, ALIGN, dict(kg_ld=129)),
    (RD, INVALID, dict(format=3)), (RD, INVALID, dict(format=-1)), (RD, INVALID, dict(T=-1)), (RD, INVALID, dict(slots=None)),
    (RD, INVALID, dict(v_out=None)), (RD, INVALID, dict(k_ld=120)), (RD, INVALID, dict(vg=None)), (RD, INVALID, dict(kc_ld=512)),
    (RD, INVALID, dict(format=1, kc_ld=1024)), (RD, INVALID, dict(pages=1 << 30)), (RD, UNSUPPORTED, dict(D=36)),
    (RD, UNSUPPORTED, dict(D=520)), (RD, UNSUPPORTED, dict(page=3)), (RD, UNSUPPORTED, dict(T=1 << 24)),
    (RD, ALIGN, dict(v_ld=132)), (RD, ALIGN, dict(k_out=FAKE + 8)), (RD, ALIGN, dict(vc=FAKE + 4)), (RD, ALIGN, dict(vg_ld=131)),
    (BA, INVALID, dict(format=4)), (BA, INVALID, dict(cap=-1.0)), (BA, INVALID, dict(cap=float("nan"))),
    (BA, INVALID, dict(cap=float("inf"))), (BA, INVALID, dict(cap=1e-38)), (BA, INVALID, dict(cap=4097.0)), (BA, INVALID, dict(scale=float("nan"))),
    (BA, INVALID, dict(kg=None)), (BA, INVALID, dict(vg_ld=64)), (BA, INVALID, dict(HQ=5, q_ld=400, out_ld=400)),
    (BA, INVALID, dict(window=-1)), (BA, INVALID, dict(format=0)), (BA, UNSUPPORTED, dict(page=10)), (BA, UNSUPPORTED, dict(D=36)),
    (BA, ALIGN, dict(kc_ld=1028)), (BA, ALIGN, dict(kg=FAKE + 2)), (BA, ALIGN, dict(vg_ld=129)), (BA, ALIGN, dict(out_ld=260)),
    (BA, ALIGN, dict(slopes=FAKE + 2)), (BA, ALIGN, dict(prefix=FAKE + 1)),
])
def test_entries_refuse(entry, code, change):
    """Every call here fails before any HIP call."""
    assert status(entry[0], *entry[1](**change)) == code, _native.last_error()
    assert _native.last_error()


def test_empty_calls_are_no_ops():
    assert status(A4[0], *_append4_args(T=0)) == 0
    assert status(RD[0], *_read_args(T=0)) == 0 and status(RD[0], *_read_args(HK=0)) == 0
    assert status(BA[0], *_biased_args(T=0)) == 0 and status(BA[0], *_biased_args(S=0)) == 0


def test_replayed_calls_are_checked():
    """A call kept as slots goes through its entry's own checks."""
    for entry, args in (A4, RD, BA):
        with pytest.raises(NotImplementedError, match="power of two"):
            _native.Record(entry, tuple(args(page=12)[:-1]))(0)
        _native.Record(entry, tuple(args(T=0)[:-1]))(0)
    with pytest.raises(ValueError, match="intent_biased_paged_attention"):  # a cap that no f32 holds
        _native.Record(BA[0], tuple(_biased_args(cap=1e39)[:-1]))(0)
    assert len(_append_args()) == len(_append4_args()) + 1  # without the cache's format


CALLS = ["qk_norm_rope", "paged_kv_append", "paged_kv_append_fp8", "paged_kv_append_int4", "paged_kv_read",
         "paged_kv_read_fp8", "paged_kv_read_int4", "paged_attention", "paged_attention_fp8", "paged_attention_int4",
         "biased_paged_attention", "biased_paged_attention_fp8", "biased_paged_attention_int4"]


@pytest.mark.parametrize("name", CALLS)
def test_known_layouts_make_the_same_call(monkeypatch, name):
    """The second call of a layout hands over what the first does: addresses, scratch and scalars of its own, in every
    place that takes them, with no norm, one view given twice, and memory too short for scratch."""
    cache = "fp8" if name.endswith("_fp8") else "int4" if name.endswith("_int4") else "same"
    rt = runtime_for(name)
    rt._home = torch.device("cpu")
    made = []
    monkeypatch.setattr(_native, "call_packed", lambda entry, arguments, stream: made.append((entry, list(arguments))))
    monkeypatch.setattr("intent_amd.runtime._current_stream", lambda device: 0)
    buffer = torch.zeros(1 << 22, dtype=torch.uint8)
    monkeypatch.setattr(rt, "_scratch_of", lambda need: None if need > buffer.numel() else buffer[:need])

    def arguments(seed, n):
        if "attention" in name:
            q, caches, *rest = _inputs(seed, "f16", cache, [(1, 900), (1, 300 + seed)], 8, 2, 64, 16)
            forms = (torch.ones(8), torch.zeros(0, dtype=torch.int32)) if "biased" in name else ()
            return [q, *caches, *rest, *forms], [torch.empty_like(q)], [0.1 * (seed + 1)]
        heads = _heads(seed, "f16", n, 6, 2, 64, 32, "k")
        caches = [c.contiguous() for c in _caches(_gen(seed), "f16", cache, 3, 2, 8, 64)]
        slots = torch.zeros(n, dtype=torch.int32)
        if "read" in name:
            return [*caches, slots], [torch.empty(n, 2, 64).half() for _ in range(2)], []
        out = [torch.empty(n, 6, 64).half()]
        if "norm" in name:
            return [heads[0], heads[1], *heads[3:]], out + [torch.empty(n, 2, 64).half()], []
        return [*heads[:6], slots, slots, *caches], out, []  # positions are the slots

    for seed in (1, 1, 2):
        ins, outs, scalars = arguments(seed, 5)
        assert (rt.rebind((*ins, *outs, *scalars), True) is not None) == (len(made) > 0)
        rt.launch(*ins, *outs, *scalars)
        bound = rt.rebind((*ins, *outs, *scalars), True)
        assert bound.call is not None and bound.outputs == tuple(outs)
        rt.launch_bound(bound)
        assert made[-1] == made[-2] and (made[-1][1].count(buffer.data_ptr()) == 1) == ("attention" in name)
        rt.run(*ins, *scalars)
        again = rt.rebind((*ins, *scalars), False)
        rt.launch_bound(again)
        want = rt.definition.call({**{p.name: t for p, t in zip(rt._supplied, ins)},
                                   **{p.name: t for p, t in zip([p for p in rt.definition.params if p.name in rt._outputs],
                                                                again.outputs)}},
                                  again.env, again.workspace)
        assert made[-1] == (want[0], list(want[1]))
    if "attention" in name:
        monkeypatch.setattr(rt, "_scratch_of", lambda need: None)
        bound = rt.rebind((*ins, *outs, *scalars), True)
        assert bound.call is None
        rt.launch_bound(bound)
        assert made[-1][1][-2:] == [0, 0]
