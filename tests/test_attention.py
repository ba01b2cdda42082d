"""Norms with rotation, paged cache append and paged attention: against their formulas in 64 bits,
the chain of them as a decoding loop runs it, and their refusals (CPU).

Tolerances are derived from the arithmetic, per element (u = half a step of the output's type):
* norm and rotation: f32 sums over D terms and a handful of roundings of 2^-24, then one rounding of u;
* E4M3 codes: one rounding of 2^-4 of the value (2^-10 of the scale below the normal range), scales f32;
* attention: weights rounded once to q's type (u each, or 2^-25 absolute below f16's normal range, and a
  weight of 1 exists), scores in f32 (D + 4 roundings of sum |q k|), sums over n tokens in f32, and the
  output's own rounding.
"""
import ctypes
import math

import pytest
import torch

import intent_amd as intent
from intent_amd import _native, errors
from intent_amd import runtime as runtime_module
from intent_amd.runtime import HIPRuntime

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F8 = torch.float8_e4m3fn


def _name(op, dt, fp8=False):
    return ("" if dt == "f16" else dt + "_") + op + ("_fp8" if fp8 else "")


def _compile(op, dt, fp8=False, **constexprs):
    return intent.compile(getattr(intent, _name(op, dt, fp8)), target=intent.MI355XTarget(0), constexprs=constexprs or None)


def _randn(gen, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=gen, dtype=torch.float64) * std).to(dtype)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- formulas in 64 bits ---------------------------------------------------------------

def ref_norm_rope(x, weight, cos_sin, positions, eps, interleaved):
    """x [T, H, D] -> (y, bound on |f32 evaluation - y| before the last rounding), both f64."""
    x = x.double()
    D, R = x.shape[-1], cos_sin.shape[1]
    y = x
    if weight.numel():
        y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.double()
    # sum of D squares (relative D * 2^-24, halved by the root), root, two products
    bound = y.abs() * ((D / 2 + 8) * 2.0 ** -24 if weight.numel() else 0.0)
    if R:
        turn = cos_sin.double()[positions.long().clamp(0, cos_sin.shape[0] - 1)][:, None]
        cos, sin = turn[..., :R // 2], turn[..., R // 2:]
        pick = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
        a, b = y[..., pick[0]].clone(), y[..., pick[1]].clone()
        ea, eb = bound[..., pick[0]].clone(), bound[..., pick[1]].clone()
        y, bound = y.clone(), bound.clone()
        size = (a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()
        y[..., pick[0]], y[..., pick[1]] = a * cos - b * sin, b * cos + a * sin
        bound[..., pick[0]] = ea * cos.abs() + eb * sin.abs() + size[0] * 2.0 ** -22
        bound[..., pick[1]] = eb * cos.abs() + ea * sin.abs() + size[1] * 2.0 ** -22
    return y, bound


def rounded_bound(y, bound, dtype):
    u, tiny = HALF_STEP[dtype], 2.0 ** -25 if dtype is torch.float16 else 2.0 ** -134
    return bound * (1 + u) + y.abs() * u * (1 + 2.0 ** -20) + tiny


def ref_attention(q, k_cache, v_cache, k_scales, v_scales, table, q_offsets, kv_lens, scale, causal, window):
    """(out [T, HQ, D], tolerance) in f64; rows of no sequence are NaN in out."""
    T, HQ, D = q.shape
    pages, HK, PAGE, _ = k_cache.shape
    u = HALF_STEP[q.dtype]
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
        ids = table[s, :-(-kv // PAGE)].to(torch.int64) & 0xffffffff
        ids = ids.clamp(max=pages - 1)
        rows = []
        for cache, scales in ((k_cache, k_scales), (v_cache, v_scales)):
            x = cache[ids].double()
            if scales is not None:
                x = x * scales[ids].double()[..., None]
            rows.append(x.transpose(1, 2).reshape(-1, HK, D)[:kv])
        p = torch.arange(kv - n, kv)[:, None]
        t = torch.arange(kv)[None]
        seen = torch.ones(n, kv, dtype=torch.bool)
        if causal:
            seen &= t <= p
        if window:
            seen &= t > p - window
        for h in range(HQ):
            qh, k, v = q[start:start + n, h].double(), rows[0][:, h // (HQ // HK)], rows[1][:, h // (HQ // HK)]
            logit = (qh @ k.T * scale).masked_fill(~seen, -math.inf)
            w = torch.softmax(logit, -1).masked_fill(~seen, 0.0)  # no seen token: a row of NaN, masked to zeros
            if v.isfinite().all():
                o, size, big = w @ v, w @ v.abs(), v.abs().amax(0)
            else:  # what a row does not see does not reach it, whatever it holds
                o = torch.stack([w[i, seen[i]] @ v[seen[i]] for i in range(n)])
                size = torch.stack([w[i, seen[i]] @ v[seen[i]].abs() for i in range(n)])
                big = torch.stack([v[seen[i]].abs().amax(0) if seen[i].any() else v.new_zeros(D) for i in range(n)])
            off = (qh.abs() @ k.abs().nan_to_num(0, 0, 0).T * abs(scale)).masked_fill(~seen, 0).amax(-1, keepdim=True)
            many = seen.sum(-1, keepdim=True).double()
            out[start:start + n, h] = o
            # weights: u; scores: (D + 4) 2^-24 of their size, twice (numerator and denominator), and the
            # exponentials' own 2^-22; sums of `many` terms twice
            slack = u + 2 * (D + 4) * 2.0 ** -24 * off + 2.0 ** -21 + 2 * many * 2.0 ** -24
            tol[start:start + n, h] = size * slack + o.abs() * u + (many * 2.0 ** -25 * big if u == 2.0 ** -11 else 0)
            tol[start:start + n, h] += 2.0 ** -25 if u == 2.0 ** -11 else 0
    return out, tol


def _close(got, want, tol, what=""):
    got = got.double().cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    ok = same | ((got - want).abs() <= tol)
    assert bool(ok.all()), (what, int((~ok).sum()), float(((got - want).abs() / tol)[~ok].max()))


# ---- norms and rotation ----------------------------------------------------------------

NORM_CASES = [
    # dtype, T, HQ, HK, D, R, interleaved, norms
    ("f16", 1, 32, 8, 128, 128, False, "qk"), ("bf16", 1, 1, 1, 8, 0, False, "qk"), ("f16", 3, 5, 1, 16, 16, False, "q"),
    ("bf16", 7, 14, 2, 64, 32, True, "qk"), ("f16", 9, 2, 2, 96, 96, False, "k"), ("bf16", 33, 4, 4, 80, 48, False, "qk"),
    ("f16", 5, 3, 1, 256, 64, True, ""), ("bf16", 65, 8, 2, 128, 128, False, "qk"), ("f16", 4, 7, 1, 512, 512, False, "qk"),
    ("bf16", 6, 1, 2, 264, 256, True, "qk"), ("f16", 130, 32, 8, 128, 64, False, "qk"), ("bf16", 2, 0, 3, 64, 64, False, "k"),
    ("f16", 2, 3, 0, 64, 64, False, "q"), ("bf16", 257, 16, 2, 192, 192, False, "qk"), ("f16", 0, 4, 2, 64, 64, False, "qk"),
]


def _heads(seed, dt, T, HQ, HK, D, R, norms, std=1.0, length=300, strided=True):
    """Queries, keys and values as slices of one projection's rows, weights, table and positions."""
    gen, dtype = _gen(seed), TYPES[dt]
    row = (HQ + 2 * HK) * D
    rows = _randn(gen, max(T, 1), row + (24 if strided else 0), dtype=dtype, std=std)[:T, :row]
    q, k, v = (part.unflatten(1, (n, D)) for part, n in zip(rows.split((HQ * D, HK * D, HK * D), 1), (HQ, HK, HK)))
    weights = [(1 + _randn(gen, D if c in norms else 0, std=0.2)).to(dtype) for c in "qk"]
    angle = torch.outer(torch.arange(length, dtype=torch.float64), 10000.0 ** (-torch.arange(0, R, 2).double() / max(R, 1)))
    table = torch.cat((angle.cos(), angle.sin()), 1).float()
    positions = torch.randint(0, length, (T,), generator=gen, dtype=torch.int32)
    return q, k, v, weights[0], weights[1], table, positions


def _cuda(*tensors):
    """Copies on the GPU that keep their strides."""
    made = []
    for t in tensors:
        if t is None:
            made.append(None)
            continue
        d = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
        made.append(d.view(torch.uint8).copy_(t.view(torch.uint8)).view(t.dtype) if t.dtype is F8 else d.copy_(t))
    return made


@pytest.mark.gpu
@pytest.mark.parametrize("case", NORM_CASES, ids=lambda c: "-".join(map(str, c)))
def test_qk_norm_rope(gpu, case):
    dt, T, HQ, HK, D, R, interleaved, norms = case
    q, k, _, qw, kw, table, positions = _heads(3, dt, T, HQ, HK, D, R, norms)
    if T > 2:
        positions[0], positions[1] = -5, 10 ** 6  # clamped to the table
    art = _compile("qk_norm_rope", dt, INTERLEAVED=interleaved, EPS=1e-5)
    got = art.run(*_cuda(q, k, qw, kw, table, positions))
    for out, x, w in zip(got, (q, k), (qw, kw)):
        want, bound = ref_norm_rope(x, w, table, positions, 1e-5, interleaved)
        assert out.dtype is TYPES[dt] and out.shape == x.shape
        _close(out, want, rounded_bound(want, bound, TYPES[dt]), case)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_qk_norm_rope_extremes(gpu, dt):
    """Rows of zeros (eps alone under the root), of the largest values and of subnormals; infinities
    and NaN stay in their own head."""
    q, k, _, qw, kw, table, positions = _heads(5, dt, 6, 4, 2, 64, 64, "qk")
    q, k = q.clone(), k.clone()
    q[0] = 0
    q[1] = torch.finfo(TYPES[dt]).max / 64 if dt == "f16" else 1e15
    q[2] = torch.finfo(TYPES[dt]).smallest_normal / 8 if dt == "f16" else 1e-15
    q[3, 1] = float("nan")
    k[4, 0, 3] = float("inf")
    got = _compile("qk_norm_rope", dt).run(*_cuda(q, k, qw, kw, table, positions))
    for out, x, w, bad in zip(got, (q, k), (qw, kw), ((3, 1), (4, 0))):
        want, bound = ref_norm_rope(x, w, table, positions, 1e-6, False)
        keep = torch.ones(x.shape[:2], dtype=torch.bool)
        keep[bad] = False
        assert not torch.isfinite(out.cpu()[bad]).any() or x is k
        _close(out[keep.to(out.device)], want[keep], rounded_bound(want, bound, TYPES[dt])[keep], dt)


# ---- append ----------------------------------------------------------------------------

APPEND_CASES = [
    # dtype, fp8, T, HQ, HK, D, R, interleaved, norms, page size, pages
    ("f16", False, 1, 32, 8, 128, 128, False, "qk", 16, 3), ("bf16", True, 1, 4, 1, 64, 64, False, "", 1, 2),
    ("f16", True, 37, 14, 2, 64, 32, True, "qk", 32, 5), ("bf16", False, 130, 6, 3, 96, 96, False, "k", 64, 4),
    ("bf16", True, 67, 8, 8, 256, 128, False, "qk", 16, 9), ("f16", True, 20, 2, 1, 8, 0, False, "", 4, 8),
    ("f16", False, 15, 3, 1, 512, 512, False, "q", 8, 3), ("bf16", True, 9, 5, 5, 200, 16, True, "qk", 2, 20),
    ("f16", False, 6, 0, 2, 128, 128, False, "k", 256, 1), ("f16", True, 0, 4, 2, 64, 64, False, "qk", 16, 2),
    ("bf16", False, 5, 4, 2, 128, 0, False, "", 16, 0),
]


def _caches(gen, dt, fp8, pages, HK, PAGE, D, extra=0, std=1.0):
    """Filled caches (and scales) whose pages lie `extra` elements apart."""
    made = []
    for _ in range(2):
        x = _randn(gen, pages, HK * PAGE * D + extra, std=std)
        x = (x * 100).clamp(-448, 448).to(F8) if fp8 else x.to(TYPES[dt])
        made.append(x[:, :HK * PAGE * D].unflatten(1, (HK, PAGE, D)))
    if fp8:
        for _ in range(2):
            x = torch.rand(pages, HK * PAGE + extra, generator=gen) * 0.01 + 0.002
            made.append(x[:, :HK * PAGE].unflatten(1, (HK, PAGE)))
    return made


def _slot_rows(cache, slots):
    """Rows [T, HK, ...] of slots in a cache [pages, HK, PAGE, ...]."""
    PAGE = cache.shape[2]
    return cache[slots.long() // PAGE, :, slots.long() % PAGE]


def _check_fp8(codes, scales, want, bound):
    """Codes and scales of rows whose f64 values are known to `bound`."""
    amax = want.abs().amax(-1)
    top = bound.amax(-1)
    s = amax.clamp(min=1e-12) / 448
    assert bool(((scales.double() - s).abs() <= (top / 448 + s * 2.0 ** -23)).all())
    value = codes.double() * scales.double()[..., None]
    # the code: half a step of the value, or of the subnormal range; the value itself: bound
    step = torch.maximum(want.abs() * 2.0 ** -4, scales.double()[..., None] * 2.0 ** -10)
    assert bool(((value - want).abs() <= step * (1 + 2.0 ** -10) + 2 * bound + want.abs() * 2.0 ** -20).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPEND_CASES, ids=lambda c: "-".join(map(str, c)))
def test_paged_kv_append(gpu, case):
    dt, fp8, T, HQ, HK, D, R, interleaved, norms, PAGE, pages = case
    gen = _gen(11)
    heads = _heads(7, dt, T, HQ, HK, D, R, norms)
    q, k, v, qw, kw, table, positions = heads
    count = pages * PAGE
    order = torch.randperm(max(count, T), generator=gen)[:T].to(torch.int32)
    order[order >= count] = -1
    if T > 3:  # padded rows and slots past the cache: skipped
        order[1], order[2] = -1, count
        order[3] = 2 ** 31 - 1
    kept = (order >= 0) & (order < count)
    caches = _caches(gen, dt, fp8, pages, HK, PAGE, D, extra=32)
    before = [c.clone() for c in caches]
    device = _cuda(*caches)
    q_out = _compile("paged_kv_append", dt, fp8, INTERLEAVED=interleaved).run(*_cuda(*heads, order), *device)
    want, bound = ref_norm_rope(q, qw, table, positions, 1e-6, interleaved)
    _close(q_out, want, rounded_bound(want, bound, TYPES[dt]), case)
    key, key_bound = ref_norm_rope(k, kw, table, positions, 1e-6, interleaved)
    after = [c.cpu() for c in device]
    touched = torch.zeros(pages, PAGE, dtype=torch.bool)
    touched.view(-1)[order[kept].long()] = True
    for new, old in zip(after, before):  # every other row is left as it was
        axis = touched[:, None, :].expand(new.shape[:3])
        same = new.view(torch.uint8) == old.view(torch.uint8) if new.dtype is F8 else new == old
        assert bool((same.flatten(3).all(-1) if same.dim() == 4 else same)[~axis].all())
    if not int(kept.sum()):
        return
    slots = order[kept]
    for i, (rows, limit) in enumerate(((key[kept], key_bound[kept]), (v[kept].double(), torch.zeros_like(key_bound[kept])))):
        got = _slot_rows(after[i], slots)
        if fp8:
            _check_fp8(got, _slot_rows(after[2 + i], slots), rows, limit)
        else:
            _close(got, rows, rounded_bound(rows, limit, TYPES[dt]), case)
    if fp8:  # values pass no arithmetic before the quantizer: bit-exact with the formula in f32
        x = v[kept].float()
        scale = x.abs().amax(-1).clamp(min=1e-12) / 448.0
        codes = (x / scale[..., None]).clamp(-448.0, 448.0).to(F8)
        assert torch.equal(_slot_rows(after[3], slots), scale)
        assert torch.equal(_slot_rows(after[1], slots).view(torch.uint8), codes.view(torch.uint8))


# Prompts: two heads to a lane group (2^20 lanes and more), of one kind or at the seams between queries, keys and
# values, and an odd one left over.
PROMPT_CASES = [
    # dtype, fp8, T, HQ, HK, D, R, interleaved, norms, page size, pages
    ("f16", False, 18733, 3, 2, 64, 64, False, "qk", 16, 1175), ("bf16", True, 18733, 3, 2, 64, 32, True, "q", 64, 300),
    ("bf16", False, 6561, 4, 3, 96, 96, False, "k", 32, 206), ("f16", True, 13109, 3, 1, 128, 128, False, "qk", 128, 104),
    ("bf16", False, 3641, 5, 2, 192, 64, True, "qk", 256, 15), ("bf16", True, 6560, 1, 2, 256, 128, False, "", 16, 411),
    ("f16", True, 1827, 7, 1, 512, 512, False, "qk", 8, 240), ("f16", False, 65537, 0, 1, 64, 0, False, "", 2, 32800),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", PROMPT_CASES, ids=lambda c: "-".join(map(str, c)))
def test_prompts(gpu, case):
    dt, fp8, T, HQ, HK, D, R, interleaved, norms, _, _ = case
    test_paged_kv_append(gpu, case)
    assert "2 heads" in _native.last_kernel()
    lanes = 8 if D <= 64 else 16 if D <= 128 else 32 if D <= 256 else 64
    more = -(-2 ** 20 // (lanes * (HQ + HK)))  # without the values
    test_qk_norm_rope(gpu, (dt, more + 5, HQ, HK, D, R, interleaved, norms))
    assert "2 heads" in _native.last_kernel()


@pytest.mark.gpu
def test_paged_kv_append_zero_rows_and_large_values(gpu):
    """fp8: a zero head gets the smallest scale and zero codes; the largest values stay finite."""
    heads = list(_heads(7, "bf16", 4, 2, 2, 64, 0, "", strided=False))
    heads[1], heads[2] = heads[1].clone(), heads[2].clone()
    heads[1][0], heads[2][1] = 0, 3e38
    caches = _cuda(*_caches(_gen(1), "bf16", True, 1, 2, 4, 64))
    _compile("paged_kv_append", "bf16", True).run(*_cuda(*heads, torch.arange(4, dtype=torch.int32)), *caches)
    k, v, ks, vs = (c.cpu() for c in caches)
    assert bool((k[0, :, 0].float() == 0).all()) and torch.equal(ks[0, :, 0], torch.full((2,), 1e-12) / 448.0)
    assert bool((v[0, :, 1].float().abs() == 448).all()) and bool(torch.isfinite(vs).all())


@pytest.mark.gpu
def test_paged_kv_append_values_that_are_not_finite(gpu):
    """fp8: a head that holds an infinity or NaN reads as NaN, its neighbours as without it."""
    heads = list(_heads(7, "bf16", 6, 2, 2, 64, 0, "k", strided=False))
    clean = [h.clone() for h in heads]
    heads[1], heads[2] = heads[1].clone(), heads[2].clone()
    heads[1][3, 0, 1] = float("nan")
    heads[2][1, 0, 3], heads[2][2, 1, 63], heads[2][4, 1, 0] = float("nan"), float("inf"), float("-inf")
    results = []
    for h in (heads, clean):
        caches = _cuda(*_caches(_gen(1), "bf16", True, 1, 2, 8, 64))
        _compile("paged_kv_append", "bf16", True).run(*_cuda(*h, torch.arange(6, dtype=torch.int32)), *caches)
        k, v, ks, vs = (c.cpu() for c in caches)
        results.append((k[0, :, :6].float() * ks[0, :, :6, None], v[0, :, :6].float() * vs[0, :, :6, None]))
    for got, want, bad in zip(*results, ([(0, 3)], [(0, 1), (1, 2), (1, 4)])):
        held = torch.zeros(2, 6, dtype=torch.bool)
        for head, token in bad:
            held[head, token] = True
        assert bool(got[held].isnan().all()) and torch.equal(got[~held], want[~held])


# ---- attention -------------------------------------------------------------------------

ATTENTION_CASES = [
    # dtype, fp8, [(new, cached)], HQ, HK, D, page size, causal, window
    ("f16", False, [(1, 1)], 1, 1, 64, 16, True, 0),
    ("bf16", True, [(1, 1)], 8, 2, 128, 1, True, 0),
    ("f16", False, [(1, 65), (1, 64), (1, 63), (1, 1), (1, 33)], 8, 2, 128, 16, True, 0),
    ("bf16", False, [(1, 700), (1, 31), (0, 90), (1, 0), (1, 257)], 28, 4, 128, 32, True, 0),
    ("f16", True, [(1, 1000), (1, 129), (1, 16)], 32, 8, 128, 64, True, 0),
    ("bf16", True, [(1, 515)], 7, 1, 64, 256, True, 0),
    ("f16", False, [(1, 300), (1, 77)], 4, 4, 256, 16, True, 0),
    ("bf16", True, [(1, 200), (2, 90)], 12, 2, 256, 8, True, 0),
    ("f16", False, [(5, 205), (5, 5), (5, 3), (4, 64)], 14, 2, 64, 16, True, 0),
    ("bf16", False, [(3, 100), (8, 200), (1, 40)], 28, 4, 128, 2, True, 0),
    ("f16", True, [(7, 450), (2, 66)], 16, 2, 128, 32, True, 0),
    ("bf16", False, [(64, 64)], 4, 1, 128, 16, True, 0),
    ("f16", False, [(100, 333), (129, 129)], 8, 2, 128, 64, True, 0),
    ("bf16", True, [(200, 500)], 6, 2, 64, 128, True, 0),
    ("f16", True, [(70, 70), (33, 161)], 4, 1, 256, 16, True, 0),
    ("bf16", False, [(90, 150), (1, 400), (0, 30), (17, 0), (30, 12)], 8, 8, 128, 32, True, 0),
    ("f16", False, [(40, 300), (1, 200), (129, 400)], 8, 2, 64, 16, True, 70),
    ("bf16", True, [(1, 900), (1, 20), (3, 200)], 8, 2, 128, 16, True, 100),
    ("f16", False, [(1, 300), (60, 200)], 4, 2, 128, 16, True, 1),
    ("bf16", False, [(50, 120), (1, 65)], 4, 2, 128, 16, False, 0),
    ("f16", True, [(50, 120), (20, 300), (9, 4)], 4, 2, 64, 16, False, 33),
    ("bf16", False, [(20, 90), (1, 50)], 6, 2, 96, 16, True, 0),
    ("f16", True, [(1, 90), (11, 50)], 6, 2, 80, 16, True, 0),
    ("f16", False, [(3, 90), (1, 150)], 2, 1, 512, 4, True, 0),
    ("bf16", False, [(1, 3000), (1, 2500)], 8, 1, 128, 16, True, 0),
    ("f16", False, [(300, 1200)], 8, 1, 128, 16, True, 0),
    # equal chunks of 48 and 64 rows, pages smaller than a load, and chunks of eight waves
    ("bf16", False, [(6, 300), (6, 70)], 28, 4, 128, 16, True, 0),
    ("f16", True, [(8, 100), (8, 900)], 16, 2, 64, 2, True, 0),
    ("f16", True, [(7, 450), (9, 66)], 14, 2, 96, 32, True, 0),
    ("bf16", False, [(70, 700)], 4, 2, 128, 2, True, 0),
    ("f16", True, [(100, 1000)], 4, 2, 128, 4, True, 60),
    ("f16", True, [(600, 700)], 8, 2, 64, 16, True, 0),
    ("bf16", True, [(260, 900)], 16, 2, 128, 64, True, 0),
    ("f16", False, [(800, 900)], 128, 1, 64, 16, True, 0),
    ("bf16", True, [(800, 860)], 128, 1, 96, 32, True, 300),
    ("f16", True, [(1100, 1130), (1, 400)], 96, 1, 128, 16, True, 0),
    ("bf16", False, [(300, 500), (400, 420)], 8, 1, 96, 16, True, 0),
    ("f16", False, [(40, 300), (1, 500), (2, 30), (90, 90)], 4, 2, 256, 32, True, 0),
    ("bf16", False, [(1, 40 + 13 * i) for i in range(70)] + [(0, 5)] * 60 + [(2, 30)], 4, 2, 64, 16, True, 0),
    # heads of 256: two tiles of 16 rows, fewer than 512 rows, and a round of uneven sequences
    ("f16", True, [(3, 300), (3, 90)], 16, 2, 256, 16, True, 0),
    ("bf16", False, [(60, 200), (60, 400)], 3, 1, 256, 32, True, 50),
    ("bf16", True, [(7, 60 + 900 * (i % 17 == 3)) for i in range(70)], 16, 2, 256, 16, True, 0),
    # more sequences than a wave takes at once, one of them split
    ("f16", False, [(1, 1 + 7 * i % 40) for i in range(555)] + [(1, 9000), (1, 0)] + [(1, 33)] * 60, 2, 1, 64, 16, True, 0),
    ("bf16", True, [(4, 4 + i % 30) for i in range(300)] + [(700, 900)] + [(1, 50)] * 5, 4, 1, 64, 16, True, 0),
]


def _attention_inputs(seed, dt, fp8, lens, HQ, HK, D, PAGE, poison=True, q_std=1.5, spare=0):
    """Ragged sequences over shuffled pages; what no sequence reaches is NaN, unused table entries -1."""
    gen = _gen(seed)
    T = sum(n for n, _ in lens)
    need = [-(-kv // PAGE) for _, kv in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=gen)
    q = _randn(gen, T + spare, HQ, D, dtype=TYPES[dt], std=q_std)
    caches = _caches(gen, dt, fp8, pages, HK, PAGE, D, extra=16)
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
            else:
                c[dead] = float("nan")
    offsets = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32)
    kv_lens = torch.tensor([kv for _, kv in lens], dtype=torch.int32)
    k_scales, v_scales = (caches[2], caches[3]) if fp8 else (None, None)
    return q, caches[0], caches[1], k_scales, v_scales, table, offsets, kv_lens


def _run_attention(inputs, dt, fp8, scale, causal, window, out=None):
    art = _compile("paged_attention", dt, fp8, CAUSAL=causal, WINDOW=window)
    device = [t for t in _cuda(*inputs) if t is not None]
    if out is None:
        return art.run(*device, scale)
    art(*device, out, scale)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTENTION_CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", "")[:90])
def test_paged_attention(gpu, case):
    dt, fp8, lens, HQ, HK, D, PAGE, causal, window = case
    inputs = _attention_inputs(21, dt, fp8, lens, HQ, HK, D, PAGE)
    scale = D ** -0.5
    want, tol = ref_attention(*inputs, scale, causal, window)
    _close(_run_attention(inputs, dt, fp8, scale, causal, window), want, tol, case)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens", [[(1, 130), (1, 70)], [(6, 130), (5, 70)], [(70, 200), (90, 120)]], ids=str)
def test_paged_attention_rows_that_belong_to_no_sequence(gpu, lens, fp8):
    """Padded rows before the first and behind the last sequence are left as they were; offsets past the
    tensor are clamped; strided rows."""
    inputs = list(_attention_inputs(22, "f16", fp8, lens, 8, 2, 64, 16, spare=9))
    inputs[6] = inputs[6] + 3
    T = inputs[0].shape[0]
    wide = torch.full((T, 8 * 64 + 40), 7.0, dtype=torch.float16, device="cuda")
    out = wide[:, :512].unflatten(1, (8, 64))
    want, tol = ref_attention(*inputs, 0.125, True, 0)
    _run_attention(inputs, "f16", fp8, 0.125, True, 0, out)
    rows = ~want[:, 0, 0].isnan()
    assert int(rows.sum()) == sum(n for n, _ in lens)
    _close(out[rows.to("cuda")], want[rows], tol[rows])
    assert bool((out[~rows.to("cuda")] == 7).all()) and bool((wide[:, 512:] == 7).all())
    inputs[6] = inputs[6] * 1
    inputs[6][-1] = 10 ** 6
    want, tol = ref_attention(*inputs, 0.125, True, 0)
    got = _run_attention(inputs, "f16", fp8, 0.125, True, 0)
    rows = ~want[:, 0, 0].isnan()
    _close(got[rows.to("cuda")], want[rows], tol[rows])


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("fp8", [False, True])
def test_paged_attention_bad_pages_and_lengths(gpu, fp8, new):
    """Page ids outside the cache and lengths past the table are clamped to them."""
    inputs = list(_attention_inputs(23, "bf16", fp8, [(new, 100), (new, 90)], 4, 2, 64, 16, poison=False))
    inputs[5][0, 2], inputs[5][1, 1], inputs[5][0, 4] = -7, 2 ** 31 - 1, inputs[1].shape[0]
    inputs[7] = torch.tensor([10 ** 6, -4], dtype=torch.int32)
    want, tol = ref_attention(*inputs, 0.125, True, 0)
    assert bool((want[new:] == 0).all())
    _close(_run_attention(inputs, "bf16", fp8, 0.125, True, 0), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("new,HQ", [(1, 4), (5, 4), (64, 4), (200, 2)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_paged_attention_masked_values_do_not_reach_a_row(gpu, new, HQ, bad):
    """NaN and infinities in keys, values and scales that a row does not see leave it as it is, also where
    other rows of the same tile see them."""
    lens = [(new, new + 150)]
    for dt, fp8 in (("f16", False), ("bf16", False), ("f16", True)):
        inputs = list(_attention_inputs(24, dt, fp8, lens, HQ, 2, 64, 16, poison=False))
        clean = [None if t is None else t.clone() for t in inputs]
        for at in (new + 149, 3) if new > 1 else (3,):  # the newest token, and one that a window hides
            page, place = int(inputs[5][0, at // 16]), at % 16
            for i in (1, 2):
                if not fp8:
                    inputs[i][page, 0, place, 5] = bad
                else:
                    inputs[i].view(torch.uint8)[page, 0, place, 5] = 0x7f  # NaN
                    inputs[i + 2][page, 1, place] = bad
        got = _run_attention(inputs, dt, fp8, 0.125, True, 140).cpu()
        want, tol = ref_attention(*[None if t is None else t for t in clean], 0.125, True, 140)
        hidden = slice(0, new - 1) if new > 1 else slice(0, 1)
        p = torch.arange(150, 150 + new)[hidden]
        sees_old = (3 > p - 140)
        assert not bool(sees_old.any())
        _close(got[hidden], want[hidden], tol[hidden], (dt, fp8))
        if new > 1:  # the row that sees the newest token has it in its result
            assert not bool(torch.isfinite(got[-1]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("lens", [[(1, 200)], [(4, 90)], [(80, 200)]], ids=str)
def test_paged_attention_scales(gpu, lens, scale):
    """A zero and a negative scale, and one that makes the softmax pick single tokens."""
    inputs = _attention_inputs(25, "f16", False, lens, 4, 2, 128, 16)
    want, tol = ref_attention(*inputs, scale, True, 0)
    _close(_run_attention(inputs, "f16", False, scale, True, 0), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[(1, 500)], [(90, 300)]], ids=str)
def test_paged_attention_fp8_scales_below_zero(gpu, lens):
    inputs = list(_attention_inputs(32, "f16", True, lens, 8, 2, 64, 16, poison=False))
    inputs[3], inputs[4] = -inputs[3], -300 * inputs[4]
    want, tol = ref_attention(*inputs, 0.1, True, 0)
    _close(_run_attention(inputs, "f16", True, 0.1, True, 0), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[(1, 500)], [(90, 300)]], ids=str)
def test_paged_attention_fp8_scales_of_many_sizes(gpu, lens):
    """Tokens whose values differ by orders of magnitude, and tokens of zeros."""
    for dt in ("f16", "bf16"):
        inputs = _attention_inputs(26, dt, True, lens, 4, 2, 128, 16, poison=False)
        gen = _gen(1)
        inputs[4].mul_(10.0 ** (torch.rand(inputs[4].shape, generator=gen) * 5 - 4))
        inputs[4][torch.rand(inputs[4].shape, generator=gen) < 0.1] = 0
        want, tol = ref_attention(*inputs, 0.0884, True, 0)
        _close(_run_attention(inputs, dt, True, 0.0884, True, 0), want, tol, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 6, 130])
@pytest.mark.parametrize("fp8", [False, True])
def test_paged_attention_rising_scores(gpu, new, fp8):
    """Scores that rise along the cache, so that the running maximum moves in every tile, and fall."""
    for order in (1, -1):
        inputs = _attention_inputs(27, "f16", fp8, [(new, 900)], 4, 1, 64, 16, poison=False)
        q, k, table = inputs[0], inputs[1], inputs[5]
        q[..., 0] = 4.0
        t = torch.arange(900)
        rise = (order * (t - 450) / 20.0)
        k[table[0, t // 16].long(), 0, t % 16, 0] = (rise * (5 if fp8 else 1)).to(k.dtype)
        if fp8:
            inputs[3].fill_(0.2)
        want, tol = ref_attention(*inputs, 0.5, True, 0)
        _close(_run_attention(inputs, "f16", fp8, 0.5, True, 0), want, tol, order)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_paged_attention_far_pages(gpu, new):
    """Pages that lie more than 2^31 elements (4 GiB) apart."""
    inputs = list(_attention_inputs(28, "f16", False, [(new, 60)], 4, 2, 64, 16, poison=False))
    step = (1 << 31) + 64
    pages = inputs[1].shape[0]
    far = []
    for c in inputs[1:3]:
        base = torch.empty((pages - 1) * step + c[0].numel(), dtype=c.dtype, device="cuda")
        view = base.as_strided(c.shape, (step, c.shape[2] * c.shape[3], c.shape[3], 1))
        view.copy_(c.cuda())
        far.append(view)
    want, tol = ref_attention(*inputs, 0.125, True, 0)
    rest = _cuda(inputs[0], *inputs[5:])
    art = _compile("paged_attention", "f16")
    _close(art.run(rest[0], far[0], far[1], *rest[1:], 0.125), want, tol)
    # and the append to the last of them
    q, k, v, qw, kw, table, positions = _heads(29, "f16", 2, 4, 2, 64, 0, "")
    slots = torch.tensor([pages * 16 - 1, 0], dtype=torch.int32)
    _compile("paged_kv_append", "f16").run(*_cuda(q, k, v, qw, kw, table, positions, slots), *far)
    assert torch.equal(far[0][pages - 1, :, 15].cpu(), k[0]) and torch.equal(far[1][0, :, 0].cpu(), v[1])


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[(1, 900), (1, 30)], [(60, 400)]], ids=str)
def test_paged_attention_repeats_bit_for_bit(gpu, lens):
    inputs = _attention_inputs(30, "bf16", False, lens, 8, 2, 128, 16)
    first = _run_attention(inputs, "bf16", False, 0.0884, True, 0)
    for _ in range(3):
        assert torch.equal(first, _run_attention(inputs, "bf16", False, 0.0884, True, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [[0, 40, 0, 40, 0, 40], [40, 0, 40, 0, 40, 0], [-9, 40, 7, 99, -1, 3], [50, 50, 50, 0, 0, 50]])
@pytest.mark.parametrize("D", [64, 80])
def test_paged_attention_offsets_that_overlap(gpu, offsets, D):
    """Sequences whose rows overlap (no valid batch) end with rows of either; no row outside the tensor and
    nothing behind the workspace is written."""
    lens = [(8, 700)] * 5
    q, k, v, _, _, table, _, kv = _cuda(*_attention_inputs(32, "f16", False, lens, 4, 2, D, 16, poison=False))
    T = q.shape[0]
    need = _native.library().intent_paged_attention_workspace_size(T, 4, 2, D, 5, table.shape[1], 16)
    guard = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
    wide = torch.full((T + 8, 4, D), 7.0, dtype=torch.float16, device="cuda")
    offs = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    _native.call("intent_paged_attention", q.data_ptr(), T, 4, q.stride(0), 0, 0, k.data_ptr(), k.stride(0), v.data_ptr(),
                 v.stride(0), None, 0, None, 0, k.shape[0], 2, 16, D, table.data_ptr(), 5, table.shape[1], table.stride(0),
                 offs.data_ptr(), kv.data_ptr(), 0.125, 1, 0, wide.data_ptr(), wide.stride(0), guard.data_ptr(), need,
                 torch.cuda.current_stream().cuda_stream)
    assert bool((guard[need:] == 0x5a).all()) and bool((wide[T:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new,HQ,kv,PAGE,D,fp8", [(1, 4, 20000, 16, 64, False), (1, 2, 17000, 64, 128, True),
                                                  (70, 2, 9500, 64, 64, False), (40, 4, 13000, 16, 128, True),
                                                  (130, 1, 5000, 16, 256, False)])
def test_paged_attention_without_a_workspace(gpu, new, HQ, kv, PAGE, D, fp8):
    """The entry with no workspace runs unsplit, over tables longer than what a wave keeps of one; and the
    split call agrees with it."""
    inputs = _attention_inputs(31, "f16", fp8, [(new, kv)], HQ, 1, D, PAGE, poison=False)
    q, k, v, ks, vs, table, offsets, lens = _cuda(*inputs)
    out = torch.full_like(q, float("nan"))
    scales = (ks.data_ptr(), ks.stride(0), vs.data_ptr(), vs.stride(0)) if fp8 else (None, 0, None, 0)
    _native.call("intent_paged_attention", q.data_ptr(), new, HQ, q.stride(0), 0, int(fp8), k.data_ptr(), k.stride(0),
                 v.data_ptr(), v.stride(0), *scales, k.shape[0], 1, PAGE, D, table.data_ptr(), 1, table.shape[1],
                 table.stride(0), offsets.data_ptr(), lens.data_ptr(), D ** -0.5, 1, 0, out.data_ptr(), out.stride(0),
                 None, 0, torch.cuda.current_stream().cuda_stream)
    want, tol = ref_attention(*inputs, D ** -0.5, True, 0)
    _close(out, want, tol)
    assert "splits" not in _native.last_kernel()
    _close(_run_attention(inputs, "f16", fp8, D ** -0.5, True, 0), want, tol)
    assert "splits" in _native.last_kernel()


@pytest.mark.gpu
@pytest.mark.parametrize("new,HQ,D,n", [(1, 4, 64, 30000), (7, 8, 96, 20000), (1, 1, 256, 20000), (352, 8, 64, 9000),
                                         (352, 8, 128, 9000), (64, 8, 256, 9000)])
@pytest.mark.parametrize("fp8", [False, True])
def test_paged_attention_one_token_over_a_flat_tail(gpu, new, HQ, D, n, fp8):
    """f16: the first token outweighs each of the others by about 2^26.5 and its value is zero, so the output is
    what the others' weights leave. A weight is off by half a step of the type, or by 2^-32 of the highest (2^-25
    where that is 2^7), not by 2^-25 of it."""
    inputs = list(_attention_inputs(34, "f16", fp8, [(new, n)], HQ, 1, D, 16, poison=False, q_std=0.3))
    q, k, v, ks, vs, table = inputs[:6]
    gen, scale = _gen(2), D ** -0.5
    q[..., 0] = 4.0
    high = 26.5 * math.log(2) / (4.0 * scale)
    tail = (64 + _randn(gen, *v.shape, std=16)).clamp(8, 128)
    page = int(table[0, 0])
    if fp8:
        ks.fill_(0.01), vs.copy_(0.9 + 0.2 * torch.rand(vs.shape, generator=gen))
        v.copy_(tail.to(F8))
        k[..., 0], k[page, 0, 0] = 0, 0
        k[page, 0, 0, 0] = 448
        ks[page, 0, 0] = high / 448
    else:
        v.copy_(tail.half())
        k[..., 0], k[page, 0, 0] = 0, 0
        k[page, 0, 0, 0] = high
    v[page, 0, 0] = 0
    want, _ = ref_attention(*inputs, scale, True, 0)
    big = 128 * (1.1 if fp8 else 1.0)
    keys = k.double() if ks is None else k.double() * ks.double()[..., None]
    off = scale * (keys.abs() @ q.double().abs().amax((0, 1))).amax()
    # the values are positive, so size = |out|: weights and output by 2^-11, scores (twice), exponentials, sums
    tol = want * (2 * 2.0 ** -11 + 2 * (D + 4) * 2.0 ** -24 * off + 2.0 ** -21 + 2 * n * 2.0 ** -24) + 2.0 ** -25
    tol += n * 2.0 ** -32 * big
    assert 0.002 < float(want.min()) and float((tol / want).max()) < 0.06
    _close(_run_attention(inputs, "f16", fp8, scale, True, 0), want, tol)
    dq, dk, dv, dks, dvs, dtable, offsets, lens = _cuda(*inputs)
    out = torch.full_like(dq, float("nan"))
    scales = (dks.data_ptr(), dks.stride(0), dvs.data_ptr(), dvs.stride(0)) if fp8 else (None, 0, None, 0)
    _native.call("intent_paged_attention", dq.data_ptr(), new, HQ, dq.stride(0), 0, int(fp8), dk.data_ptr(), dk.stride(0),
                 dv.data_ptr(), dv.stride(0), *scales, dk.shape[0], 1, 16, D, dtable.data_ptr(), 1, dtable.shape[1],
                 dtable.stride(0), offsets.data_ptr(), lens.data_ptr(), scale, 1, 0, out.data_ptr(), out.stride(0),
                 None, 0, torch.cuda.current_stream().cuda_stream)
    _close(out, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("new,n", [(1, 20000), (352, 5000)])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_paged_attention_fp8_values_of_zero(gpu, new, n, dt):
    """Value scales of zero throughout, and scores that rise: the sums of weights stay finite, every row is zero."""
    inputs = list(_attention_inputs(35, dt, True, [(new, n)], 8, 1, 64, 16, poison=False))
    q, k, ks, table = inputs[0], inputs[1], inputs[3], inputs[5]
    q[..., 0], k[..., 0] = 4.0, 64.0
    t = torch.arange(n)
    ks[table[0, t // 16].long(), 0, t % 16] = t / n
    inputs[4].zero_()
    assert bool((_run_attention(inputs, dt, True, 0.5, True, 0) == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 3e-36, -3e-36])
@pytest.mark.parametrize("new,D", [(1, 64), (100, 128), (3, 80)])
@pytest.mark.parametrize("fp8", [False, True])
def test_paged_attention_scales_beside_large_scores(gpu, new, D, fp8, scale):
    """A scale far below one is taken as it is where q.k is as large as bf16 heads make it, zero as zero."""
    inputs = list(_attention_inputs(36, "bf16", fp8, [(new, 300)], 8, 2, D, 16, poison=False, q_std=1e17))
    if fp8:
        inputs[3].mul_(1e17)
    else:
        inputs[1].mul_(1e17)
    want, tol = ref_attention(*inputs, scale, True, 0)
    _close(_run_attention(inputs, "bf16", fp8, scale, True, 0), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("n,D,fp8", [(50003, 64, False), (131000, 128, True)])
def test_paged_attention_most_parts(gpu, n, D, fp8):
    """One sequence over more units of tokens than a tile is cut into parts (256)."""
    inputs = _attention_inputs(37, "bf16", fp8, [(1, n)], 4, 1, D, 64, poison=False)
    want, tol = ref_attention(*inputs, D ** -0.5, True, 0)
    _close(_run_attention(inputs, "bf16", fp8, D ** -0.5, True, 0), want, tol)
    assert "splits" in _native.last_kernel()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("chunk,spare", [(138, 0), (137, 0), (130, 7), (129, 7)])
@pytest.mark.parametrize("fp8", [False, True])
def test_paged_attention_decoding_beside_a_chunk(gpu, chunk, spare, D, fp8):
    """Seven decoding sequences and a chunk, whose tokens (and padded rows) are a multiple of the sequences or not:
    one list of tiles or two."""
    lens = [(1, 60 + 97 * i) for i in range(4)] + [(chunk, chunk + 300)] + [(1, 1200), (1, 1), (1, 333)]
    for window in (0, 200):
        inputs = _attention_inputs(38, "f16", fp8, lens, 16, 1, D, 16, spare=spare)
        want, tol = ref_attention(*inputs, D ** -0.5, True, window)
        got = _run_attention(inputs, "f16", fp8, D ** -0.5, True, window)
        rows = sum(n for n, _ in lens)
        _close(got[:rows], want[:rows], tol[:rows])


# ---- together --------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dt,fp8", [("f16", False), ("bf16", False), ("f16", True), ("bf16", True)])
def test_decoding_loop(gpu, dt, fp8):
    """A prompt in two chunks and three decoding steps of two sequences: projection, append, attention and
    output projection, each step over the cache that the steps before left. The attention is compared
    with the formula over the tensors that it was given, and at the end with the whole sequence's keys
    and values, never paged."""
    gen = _gen(40)
    HQ, HK, D, PAGE, H = 8, 2, 64, 16, 256
    gemm = intent.compile(intent.gemm if dt == "f16" else intent.bf16_gemm, target=intent.MI355XTarget(0))
    append, attend = _compile("paged_kv_append", dt, fp8), _compile("paged_attention", dt, fp8)
    w_qkv, w_out = (_randn(gen, *s, dtype=TYPES[dt], std=H ** -0.5).cuda() for s in ((H, (HQ + 2 * HK) * D), (HQ * D, H)))
    weights = [(1 + _randn(gen, D, std=0.1)).to(TYPES[dt]) for _ in range(2)]
    angle = torch.outer(torch.arange(200, dtype=torch.float64), 10000.0 ** (-torch.arange(0, D, 2).double() / D))
    table_cs = torch.cat((angle.cos(), angle.sin()), 1).float()
    caches = _cuda(*_caches(gen, dt, fp8, 20, HK, PAGE, D))
    pages = torch.randperm(20, generator=gen).to(torch.int32).view(2, 10)
    device = _cuda(*weights, table_cs)
    lengths = [0, 0]
    keys, values = [[], []], [[], []]
    for news in ((37, 20), (30, 1), (1, 1), (1, 1), (1, 1)):
        T = sum(news)
        x = _randn(gen, T, H, dtype=TYPES[dt]).cuda()
        qkv = gemm.run(x, w_qkv)
        q, k, v = (p.unflatten(1, (-1, D)) for p in qkv.split((HQ * D, HK * D, HK * D), 1))
        at = [torch.arange(n, n + m) for n, m in zip(lengths, news)]
        slots = torch.cat([pages[s][t // PAGE].long() * PAGE + t % PAGE for s, t in enumerate(at)]).to(torch.int32)
        positions = torch.cat(at).to(torch.int32)
        lengths = [n + m for n, m in zip(lengths, news)]
        q_out = append.run(q, k, v, *device, *_cuda(positions, slots), *caches)
        offsets = torch.tensor([0, news[0], T], dtype=torch.int32)
        kv = torch.tensor(lengths, dtype=torch.int32)
        scales = tuple(caches[2:]) if fp8 else (None, None)
        out = attend.run(q_out, *caches, *_cuda(pages, offsets, kv), D ** -0.5)
        host = [None if c is None else c.cpu() for c in (caches[0], caches[1], *scales)]
        want, tol = ref_attention(q_out.cpu(), *host, pages, offsets, kv, D ** -0.5, True, 0)
        _close(out, want, tol, news)
        y = gemm.run(out.view(T, HQ * D), w_out)
        assert bool(torch.isfinite(y).all())
        key, _ = ref_norm_rope(k.cpu(), weights[1], table_cs, positions, 1e-6, False)
        for s, (rows, vals) in enumerate(zip(key.split(news), v.cpu().double().split(news))):
            keys[s].append(rows)
            values[s].append(vals)
    # last step: the whole sequence's own keys and values, in 64 bits; the cache adds its rounding
    u = 2.0 ** -4 if fp8 else HALF_STEP[TYPES[dt]]
    for s in range(2):
        k, v = torch.cat(keys[s]), torch.cat(values[s])
        for h in range(HQ):
            logit = k[:, h // 4] @ q_out[s, h].cpu().double() * D ** -0.5
            w = torch.softmax(logit, 0)
            want = w @ v[:, h // 4]
            # keys off by u of each element (scores by u sum |q k|, weights by twice that), values by u
            off = (k[:, h // 4].abs() @ q_out[s, h].cpu().double().abs() * D ** -0.5).amax() * u
            tol = (w @ v[:, h // 4].abs()) * (math.expm1(2 * off) + 2 * u) + 2.0 ** -20
            _close(out[s, h], want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 5, 70])
def test_captured_and_replayed(gpu, new):
    """Append and attention of a step in a graph, replayed over lengths and slots that change in place,
    with eager calls of the same operators in between: every replay equals the eager step."""
    HQ, HK, D, PAGE = 8, 2, 128, 16
    heads = list(_heads(41, "bf16", 2 * new, HQ, HK, D, D, "qk", length=600))
    inputs = _attention_inputs(42, "bf16", True, [(new, 500), (new, 400)], HQ, HK, D, PAGE, poison=False)
    _, kc, vc, ks, vs, table, offsets, kv = _cuda(*inputs)
    heads = _cuda(*heads)
    slots = torch.zeros(2 * new, dtype=torch.int32, device="cuda")
    q_out = torch.empty(2 * new, HQ, D, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q_out)
    append = _compile("paged_kv_append", "bf16", True).prepare(*heads, slots, kc, vc, ks, vs, outputs=(q_out,))
    attend = _compile("paged_attention", "bf16", True).prepare(q_out, kc, vc, ks, vs, table, offsets, kv, 0.0884,
                                                               outputs=(out,))

    def place(first, second):
        at = torch.cat([torch.arange(n - new, n) for n in (first, second)])
        row = torch.arange(2).repeat_interleave(new)
        slots.copy_((inputs[5][row, at // PAGE].long() * PAGE + at % PAGE).to(torch.int32))
        kv.copy_(torch.tensor([first, second], dtype=torch.int32))
        heads[6].copy_(at.to(torch.int32))

    place(500, 400)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        append.launch()
        attend.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        append.launch()
        attend.launch()
    for first, second in ((500, 400), (new, 399), (256, 17 + new), (511, 410)):
        place(first, second)
        append.launch()
        attend.launch()
        eager = out.clone(), kc.view(torch.uint8).clone(), ks.clone()
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]), (first, second)
        assert torch.equal(kc.view(torch.uint8), eager[1]) and torch.equal(ks, eager[2])


@pytest.mark.gpu
def test_two_graphs_of_unprepared_calls(gpu):
    """run() captured twice (decoding and a chunk, both split), the graphs replayed in turn and at once on two
    streams, over lengths that change in place, with eager calls between."""
    art = _compile("paged_attention", "bf16")
    sets = [_attention_inputs(70 + i, "bf16", False, lens, 8, 2, 128, 16, poison=False)
            for i, lens in enumerate(([(1, 3000), (1, 900)], [(60, 2500)]))]
    device = [[t for t in _cuda(*s) if t is not None] for s in sets]
    for d in device:
        art.run(*d, 0.0884)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for d in device:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(art.run(*d, 0.0884))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for cut in (0, 700, 1300, 0):
        eager = []
        for d, s in zip(device, sets):
            d[5].copy_((s[7] - cut).clamp(min=0).to(torch.int32))
            eager.append(art.run(*d, 0.0884))
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


def _combined(gen, dt, fp8, pages, HK, PAGE, D):
    """One allocation of keys and values side by side in each page [pages, 2, HK, PAGE, D] (and their scales)."""
    x = _randn(gen, pages, 2, HK, PAGE, D)
    kv = (x * 100).clamp(-448, 448).to(F8) if fp8 else x.to(TYPES[dt])
    return (kv, torch.rand(pages, 2, HK, PAGE, generator=gen) * 0.01 + 0.002) if fp8 else (kv,)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [7, 900])
@pytest.mark.parametrize("dt,fp8", [("f16", False), ("bf16", True)])
def test_keys_and_values_of_one_allocation(gpu, dt, fp8, T):
    """Append and attention over kv[:, 0] and kv[:, 1]: both halves get their own rows, all others stay."""
    HQ, HK, D, PAGE, pages = 8, 2, 64, 16, 70
    gen = _gen(45)
    heads = _heads(46, dt, T, HQ, HK, D, 0, "")
    slots = torch.randperm(pages * PAGE, generator=gen)[:T].to(torch.int32)
    tensors = _combined(gen, dt, fp8, pages, HK, PAGE, D)
    apart = [t[:, i].clone().contiguous() for t in tensors for i in (0, 1)]
    device, alone = _cuda(*tensors), _cuda(*apart)
    views = [t[:, i] for t in device for i in (0, 1)]
    append = _compile("paged_kv_append", dt, fp8)
    args = _cuda(*heads, slots)
    for _ in range(2):  # bound, and known
        q_out = append.run(*args, *views)
    assert torch.equal(q_out, append.run(*args, *alone))
    for got, want in zip(views, alone):
        assert torch.equal(got.contiguous().view(torch.uint8), want.view(torch.uint8))
    table = torch.randperm(pages, generator=gen).to(torch.int32)[None]
    rest = _cuda(table, torch.tensor([0, T], dtype=torch.int32), torch.tensor([pages * PAGE - 3], dtype=torch.int32))
    attend = _compile("paged_attention", dt, fp8)
    out = attend.run(q_out, *views, *rest, 0.125)
    assert torch.equal(out, attend.run(q_out, *alone, *rest, 0.125))
    # and an output between the queries of one buffer
    wide = torch.zeros(T, 2, HQ, D, dtype=TYPES[dt], device="cuda")
    wide[:, 0] = q_out
    for _ in range(2):
        attend(wide[:, 0], *views, *rest, wide[:, 1], 0.125)
    assert torch.equal(wide[:, 0], q_out) and torch.equal(wide[:, 1], out)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 80, 256])
@pytest.mark.parametrize("fp8", [False, True])
def test_paged_attention_without_a_cache(gpu, D, fp8):
    """A table of no pages, and a cache of none: nothing is seen, every row is zero."""
    for new in (1, 5, 90):
        inputs = list(_attention_inputs(33, "f16", fp8, [(new, 40)], 4, 2, D, 16, poison=False))
        inputs[5] = inputs[5][:, :0]
        assert bool((_run_attention(inputs, "f16", fp8, 0.1, True, 0) == 0).all())
        inputs[5] = torch.zeros(1, 3, dtype=torch.int32)
        inputs[1:5] = [None if c is None else c[:0] for c in inputs[1:5]]
        assert bool((_run_attention(inputs, "f16", fp8, 0.1, True, 0) == 0).all())


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    """Calls of one artifact on two streams, in flight together, share nothing."""
    art = _compile("paged_attention", "f16")
    sets = [_attention_inputs(50 + i, "f16", False, [(1, 2000 - 300 * i)] * 3, 8, 2, 128, 16) for i in range(2)]
    device = [[t for t in _cuda(*s) if t is not None] for s in sets]
    alone = [art.run(*d, 0.0884) for d in device]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = [[], []]
    for _ in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(art.run(*device[i], 0.0884))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(r, alone[i]) for r in results[i])


@pytest.mark.gpu
def test_as_torch_op(gpu):
    inputs = [t for t in _cuda(*_attention_inputs(60, "f16", False, [(1, 40), (3, 20)], 4, 2, 64, 16)) if t is not None]
    art = _compile("paged_attention", "f16")
    op = art.as_torch_op("intent_amd_attention_test::paged_attention")
    assert torch.equal(op(*inputs, 0.125), art.run(*inputs, 0.125))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,fp8", [("f16", False), ("bf16", True)])
def test_append_as_torch_op(gpu, dt, fp8):
    """Caches and scales written in place; views of one storage are the artifact's, not the operator's."""
    heads, slots = _cuda(*_heads(61, dt, 9, 4, 2, 64, 64, "qk")), torch.arange(3, 12, dtype=torch.int32, device="cuda")
    first, second = (_cuda(*_caches(_gen(3), dt, fp8, 3, 2, 8, 64)) for _ in range(2))
    art = _compile("paged_kv_append", dt, fp8)
    op = art.as_torch_op(f"intent_amd_attention_test::{dt}_append_{int(fp8)}")
    assert torch.equal(op(*heads, slots, *first), art.run(*heads, slots, *second))
    for got, want in zip(first, second):
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    kv = _cuda(*_combined(_gen(4), dt, fp8, 3, 2, 8, 64))
    with pytest.raises(NotImplementedError, match="shares storage"):
        op(*heads, slots, *(t[:, i] for t in kv for i in (0, 1)))


# ---- refusals (CPU) --------------------------------------------------------------------

def runtime_for(name, **constexprs):
    defn = getattr(intent, name)
    return HIPRuntime(defn, 0, defn.resolve_constexprs(constexprs or None), "gfx950")


def test_outputs_are_inferred():
    rt = runtime_for("bf16_qk_norm_rope")
    heads = _heads(1, "bf16", 5, 6, 2, 64, 32, "qk")
    q_out, k_out = rt.infer_outputs((heads[0], heads[1], *heads[3:]))
    assert q_out.shape == (5, 6, 64) and k_out.shape == (5, 2, 64) and q_out.dtype is torch.bfloat16
    inputs = [t for t in _attention_inputs(1, "f16", True, [(2, 9), (1, 3)], 4, 2, 64, 4)]
    assert runtime_for("paged_attention_fp8").infer_outputs((*inputs, 0.1)).shape == (3, 4, 64)


def test_heads_are_checked():
    q, k, v, qw, kw, table, positions = _heads(1, "f16", 5, 6, 2, 64, 32, "qk")
    rt = runtime_for("qk_norm_rope")
    good = [q, k, qw, kw, table, positions]

    def refused(error, match, **change):
        names = ("q", "k", "q_weight", "k_weight", "cos_sin", "positions")
        with pytest.raises(error, match=match):
            rt.infer_outputs(tuple(change.get(n, t) for n, t in zip(names, good)))

    refused(ValueError, "q_weight", q_weight=qw[:8])
    refused(ValueError, "k_weight", k_weight=torch.cat((kw, kw)))
    refused(ValueError, "even and at most", cos_sin=torch.zeros(9, 80))
    refused(NotImplementedError, "multiple of 16", cos_sin=torch.zeros(9, 8))
    refused(ValueError, "at least one position", cos_sin=torch.zeros(0, 32))
    refused(ValueError, "relation", positions=positions[:4])
    refused(TypeError, "dtype", positions=positions.long())
    refused(TypeError, "dtype", q=q.float())
    refused(ValueError, "relation", k=k[..., :56])
    with pytest.raises(NotImplementedError, match="multiple of 8"):
        runtime_for("qk_norm_rope").infer_outputs((torch.zeros(2, 3, 60, dtype=torch.float16),
                                                   torch.zeros(2, 3, 60, dtype=torch.float16), qw[:0], kw[:0],
                                                   torch.zeros(1, 0), positions[:2]))


def test_cache_and_sequences_are_checked():
    inputs = list(_attention_inputs(1, "f16", False, [(2, 9), (1, 3)], 4, 2, 64, 4))
    inputs = [t for t in inputs if t is not None]
    rt = runtime_for("paged_attention")
    rt.infer_outputs((*inputs, 0.1))
    for i, bad, error, match in ((6 - 2, inputs[4][:2], ValueError, "q_offsets"), (5, inputs[5][:1], ValueError, "relation"),
                                 (1, inputs[1][..., :32], ValueError, "relation"),
                                 (0, inputs[0][:, :3], ValueError, "multiple of HK"),
                                 (3, inputs[3].long(), TypeError, "dtype")):
        change = list(inputs)
        change[i] = bad
        with pytest.raises(error, match=match):
            rt.infer_outputs((*change, 0.1))
    odd = [torch.zeros(3, 2, 12, 64, dtype=torch.float16)] * 2
    with pytest.raises(NotImplementedError, match="power of two"):
        rt.infer_outputs((inputs[0], *odd, *inputs[3:], 0.1))
    with pytest.raises(ValueError, match="WINDOW"):
        runtime_for("paged_attention", WINDOW=-1).infer_outputs((*inputs, 0.1))


def test_layouts_are_checked(monkeypatch):
    """Slices of a projection's rows, and pages apart, are taken; heads apart and overlapping rows are not."""
    rt = runtime_for("paged_kv_append")
    rt._home = torch.device("cpu")
    param = {p.name: p for p in intent.paged_kv_append.params}
    q, k, v, *_ = _heads(1, "f16", 5, 6, 2, 64, 32, "qk")
    rt._check_layout(param["q"], q)
    rt._check_layout(param["k"], k)
    cache = torch.zeros(4, 2, 2, 8, 64, dtype=torch.float16)
    rt._check_layout(param["k_cache"], cache[:, 1])
    with pytest.raises(ValueError, match="contiguous behind"):
        rt._check_layout(param["q"], q.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="contiguous behind"):
        rt._check_layout(param["k_cache"], cache[:, :, 0, :])
    with pytest.raises(ValueError, match="smaller than the row"):
        rt._check_layout(param["q"], q[:1].expand(5, 6, 64))


def test_views_between_one_another_are_taken(monkeypatch):
    """Keys and values of one allocation, and outputs of one row, share no element; views that do are refused
    on the first call and on a known layout."""
    rt = runtime_for("paged_kv_append_fp8")
    rt._home = torch.device("cpu")
    monkeypatch.setattr(rt, "_launch", lambda binding: None)
    q, k, v, qw, kw, table, positions = _heads(1, "f16", 5, 6, 2, 64, 32, "qk")
    kv, scales = _combined(_gen(1), "f16", True, 4, 2, 8, 64)
    slots = torch.zeros(5, dtype=torch.int32)
    args = (q, k, v, qw, kw, table, positions, slots, kv[:, 0], kv[:, 1], scales[:, 0], scales[:, 1])
    assert rt.rebind(args, False) is None
    rt.run(*args)
    assert rt.rebind(args, False) is not None
    swapped = args[:8] + (kv[:, 1], kv[:, 0], scales[:, 1], scales[:, 0])
    assert rt.rebind(swapped, False) is not None
    row = kv.stride(0)

    def refused(a, b):
        for _ in range(2):
            change = args[:8] + (a, b) + args[10:]
            assert rt.rebind(change, False) is None
            with pytest.raises(ValueError, match="k_cache and v_cache overlap"):
                rt.run(*change)

    flat = torch.zeros(5 * row, dtype=torch.uint8).view(F8)
    part = [flat[at:at + 4 * row].view(4, 2, 2, 8, 64)[:, 0] for at in (0, row // 2, row // 2 - 16, row // 2 + 16, 16)]
    rt.run(*args[:8], part[0], part[1], *args[10:])  # the rows fill the step exactly
    for other in (part[0], part[2], part[3], part[4]):
        refused(part[0], other)
    attend = runtime_for("paged_attention")
    attend._home = torch.device("cpu")
    monkeypatch.setattr(attend, "_launch", lambda binding: None)
    inputs = [t for t in _attention_inputs(1, "f16", False, [(2, 9), (1, 3)], 4, 2, 64, 4) if t is not None]
    rows = torch.zeros(3, 2, 4, 64, dtype=torch.float16)
    attend.launch(rows[:, 0], *inputs[1:], rows[:, 1], 0.1)
    assert attend.rebind((rows[:, 0], *inputs[1:], rows[:, 1], 0.1), True) is not None
    with pytest.raises(ValueError, match="overlap"):
        attend.launch(rows[:, 0], *inputs[1:], rows[:, 0], 0.1)
    with pytest.raises(ValueError, match="overlap"):  # steps that differ: rows meet further on
        attend.launch(rows[:, 0], *inputs[1:], rows.view(-1)[256:256 + 768].view(3, 4, 64), 0.1)
    single = rows[1:2, 1]  # a view of one row, between or within the rows of the other
    assert runtime_module._rows_apart(runtime_module._row_pair(rows[:, 0], single), rows.data_ptr(), single.data_ptr())
    assert not runtime_module._rows_apart(runtime_module._row_pair(rows[:, 1], single), rows[:, 1].data_ptr(),
                                          single.data_ptr())


FAKE = 0x1000


def status(entry, *args):
    return getattr(_native.library(), entry)(*args)


def _norm_args(**change):
    a = dict(q=FAKE, T=4, HQ=4, q_ld=256, k=FAKE, HK=2, k_ld=128, D=64, qw=FAKE, kw=None, eps=1e-6, cs=FAKE, P=8, R=64,
             cs_ld=64, inter=0, pos=FAKE, bf16=0, q_out=FAKE, q_out_ld=256, k_out=FAKE, k_out_ld=128, stream=None)
    assert set(change) <= set(a)
    return list({**a, **change}.values())


def _append_args(**change):
    a = dict(q=FAKE, T=4, HQ=4, q_ld=256, k=FAKE, HK=2, k_ld=128, v=FAKE, v_ld=128, D=64, qw=FAKE, kw=None, eps=1e-6,
             cs=FAKE, P=8, R=64, cs_ld=64, inter=0, pos=FAKE, slots=FAKE, bf16=0, fp8=1, kc=FAKE, kc_ld=2048, vc=FAKE,
             vc_ld=2048, ks=FAKE, ks_ld=32, vs=FAKE, vs_ld=32, pages=4, page=16, q_out=FAKE, q_out_ld=256, stream=None)
    assert set(change) <= set(a)
    return list({**a, **change}.values())


def _attention_args(**change):
    a = dict(q=FAKE, T=4, HQ=4, q_ld=256, bf16=0, fp8=1, kc=FAKE, kc_ld=2048, vc=FAKE, vc_ld=2048, ks=FAKE, ks_ld=32,
             vs=FAKE, vs_ld=32, pages=4, HK=2, page=16, D=64, table=FAKE, S=2, width=3, table_ld=3, offsets=FAKE,
             kv=FAKE, scale=0.1, causal=1, window=0, out=FAKE, out_ld=256, ws=None, ws_bytes=0, stream=None)
    assert set(change) <= set(a)
    return list({**a, **change}.values())


INVALID, ALIGN, UNSUPPORTED = errors.INTENT_ERR_INVALID_ARGUMENT, errors.INTENT_ERR_ALIGNMENT, errors.INTENT_ERR_UNSUPPORTED


@pytest.mark.parametrize("entry,args,code,change", [
    ("intent_qk_norm_rope", _norm_args, INVALID, dict(T=-1)), ("intent_qk_norm_rope", _norm_args, INVALID, dict(q=None)),
    ("intent_qk_norm_rope", _norm_args, INVALID, dict(k_out=None)), ("intent_qk_norm_rope", _norm_args, INVALID, dict(q_ld=255)),
    ("intent_qk_norm_rope", _norm_args, INVALID, dict(k_out_ld=100)), ("intent_qk_norm_rope", _norm_args, INVALID, dict(R=80)),
    ("intent_qk_norm_rope", _norm_args, INVALID, dict(P=0)), ("intent_qk_norm_rope", _norm_args, INVALID, dict(pos=None)),
    ("intent_qk_norm_rope", _norm_args, INVALID, dict(cs_ld=32)), ("intent_qk_norm_rope", _norm_args, ALIGN, dict(q=FAKE + 8)),
    ("intent_qk_norm_rope", _norm_args, ALIGN, dict(qw=FAKE + 2)), ("intent_qk_norm_rope", _norm_args, ALIGN, dict(k_ld=132)),
    ("intent_qk_norm_rope", _norm_args, ALIGN, dict(cs_ld=66)), ("intent_qk_norm_rope", _norm_args, UNSUPPORTED, dict(R=24)),
    ("intent_qk_norm_rope", _norm_args, UNSUPPORTED, dict(D=68)), ("intent_qk_norm_rope", _norm_args, UNSUPPORTED, dict(D=520)),
    ("intent_qk_norm_rope", _norm_args, UNSUPPORTED, dict(T=1 << 25)),
    ("intent_paged_kv_append", _append_args, INVALID, dict(slots=None)),
    ("intent_paged_kv_append", _append_args, INVALID, dict(ks=None)), ("intent_paged_kv_append", _append_args, INVALID, dict(v=None)),
    ("intent_paged_kv_append", _append_args, INVALID, dict(kc_ld=2047)),
    ("intent_paged_kv_append", _append_args, INVALID, dict(vs_ld=31)),
    ("intent_paged_kv_append", _append_args, INVALID, dict(pages=1 << 30)),
    ("intent_paged_kv_append", _append_args, UNSUPPORTED, dict(page=12)),
    ("intent_paged_kv_append", _append_args, ALIGN, dict(vc=FAKE + 4)),
    ("intent_paged_kv_append", _append_args, ALIGN, dict(kc_ld=2056)),
    ("intent_paged_attention", _attention_args, INVALID, dict(S=-1)),
    ("intent_paged_attention", _attention_args, INVALID, dict(HQ=5, q_ld=400, out_ld=400)),
    ("intent_paged_attention", _attention_args, INVALID, dict(HK=0)),
    ("intent_paged_attention", _attention_args, INVALID, dict(window=-1)),
    ("intent_paged_attention", _attention_args, INVALID, dict(kv=None)),
    ("intent_paged_attention", _attention_args, INVALID, dict(scale=float("nan"))),
    ("intent_paged_attention", _attention_args, INVALID, dict(scale=float("-inf"))),
    ("intent_paged_attention", _attention_args, INVALID, dict(scale=3e38)),
    ("intent_paged_attention", _attention_args, INVALID, dict(vs=None)),
    ("intent_paged_attention", _attention_args, INVALID, dict(out_ld=128)),
    ("intent_paged_attention", _attention_args, INVALID, dict(table_ld=2)),
    ("intent_paged_attention", _attention_args, INVALID, dict(vc_ld=1024)),
    ("intent_paged_attention", _attention_args, UNSUPPORTED, dict(D=36)),
    ("intent_paged_attention", _attention_args, UNSUPPORTED, dict(page=10)),
    ("intent_paged_attention", _attention_args, UNSUPPORTED, dict(width=1 << 28, table_ld=1 << 28)),
    ("intent_paged_attention", _attention_args, UNSUPPORTED, dict(T=1 << 25)),
    ("intent_paged_attention", _attention_args, ALIGN, dict(q=FAKE + 2)),
    ("intent_paged_attention", _attention_args, ALIGN, dict(out_ld=260)),
    ("intent_paged_attention", _attention_args, ALIGN, dict(kc_ld=2052)),
])
def test_entries_refuse(entry, args, code, change):
    """Every call here fails before any HIP call."""
    assert status(entry, *args(**change)) == code, _native.last_error()
    assert _native.last_error()


def test_empty_calls_are_no_ops():
    assert status("intent_qk_norm_rope", *_norm_args(T=0)) == 0
    assert status("intent_qk_norm_rope", *_norm_args(HQ=0, HK=0)) == 0
    assert status("intent_paged_kv_append", *_append_args(T=0)) == 0
    assert status("intent_paged_attention", *_attention_args(T=0)) == 0
    assert status("intent_paged_attention", *_attention_args(S=0)) == 0
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_replayed_calls_are_checked():
    """A call kept as slots goes through its entry's own checks; a wrong record is refused."""
    with pytest.raises(ValueError, match="multiple of the HK"):
        _native.Record("intent_paged_attention", tuple(_attention_args(HK=3)[:-1]))(0)
    _native.Record("intent_paged_attention", tuple(_attention_args(T=0)[:-1]))(0)
    with pytest.raises(NotImplementedError, match="power of two"):
        _native.Record("intent_paged_kv_append", tuple(_append_args(page=12)[:-1]))(0)
    with pytest.raises(ValueError, match="16-byte"):
        _native.Record("intent_qk_norm_rope", tuple(_norm_args(q=FAKE + 8)[:-1]))(0)
    with pytest.raises(TypeError, match="takes"):
        _native.Record("intent_qk_norm_rope", tuple(_norm_args()))
    slots = (ctypes.c_int64 * 4)()
    assert status("intent_amd_replay", 0, slots, 4, None) == INVALID and "slots" in _native.last_error()
    assert status("intent_amd_replay", 9, slots, 4, None) == INVALID
    assert status("intent_amd_replay", 0, None, 22, None) == INVALID


def test_scalars_past_32_bits_are_refused():
    """A scale or epsilon that no f32 holds is refused like one that is not finite."""
    for scale in (1e39, -1e300):
        with pytest.raises(ValueError, match="intent_paged_attention"):
            _native.Record("intent_paged_attention", tuple(_attention_args(scale=scale)[:-1]))(0)
        with pytest.raises(ValueError, match="intent_paged_attention"):
            _native.call_packed("intent_paged_attention", tuple(a or 0 for a in _attention_args(scale=scale)[:-1]), 0)
    with pytest.raises(ValueError, match="intent_qk_norm_rope"):
        _native.Record("intent_qk_norm_rope", tuple(_norm_args(eps=1e40)[:-1]))
