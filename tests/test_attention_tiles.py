"""Attention through the kernels of many rows (tiles of 128 and 256) and of both lists of a mixture: values that are
not finite, sizes of scores, caps, distances and pages at their ends. Every case says which kernel it is for, and runs
with its tokens split and whole. Formulas and tolerances are those of test_attention_forms.py."""
import pytest
import torch

from intent_amd import _native
from test_attention import _close, _cuda, _gen, _heads
from test_attention_forms import _attend, _compile, _inputs, _prefixes, ref_attention

FORMATS = {"same": 0, "fp8": 1, "int4": 2}
# new tokens, query heads, cached heads: rows that 22 tiles of 128 and 384 of 256 hold; heads of 256 from 512 rows on
TILE, SHARED, HIGH = (360, 8, 1), (180, 16, 2), (800, 128, 1)
WIDE = (70, 8, 1)


def _kernel(rows, D):
    return f"D {D}, {rows} rows>"


def _whole(inputs, dt, cache, scale, causal=True, window=0, cap=0.0, slopes=None, prefix=None):
    """The same call without a workspace: (out, the kernel it ran)."""
    q, caches, table, offsets, lens = _cuda(inputs[0]) + [_cuda(*inputs[1])] + _cuda(*inputs[2:])
    out = torch.full_like(q, float("nan"))
    beside = [x for c in caches[2:] for x in (c.data_ptr(), c.stride(0))] or [None, 0, None, 0]
    more = [None if x is None else x.cuda() for x in (slopes, prefix)]
    T, HQ, D = q.shape
    pages, HK, page_size = caches[0].shape[:3]
    _native.call("intent_biased_paged_attention", q.data_ptr(), T, HQ, q.stride(0), int(dt == "bf16"), FORMATS[cache],
                 caches[0].data_ptr(), caches[0].stride(0), caches[1].data_ptr(), caches[1].stride(0), *beside, pages, HK,
                 page_size, D, table.data_ptr(), table.shape[0], table.shape[1], table.stride(0), offsets.data_ptr(),
                 lens.data_ptr(), scale, int(causal), window, cap, *(None if x is None else x.data_ptr() for x in more),
                 out.data_ptr(), out.stride(0), None, 0, torch.cuda.current_stream().cuda_stream)
    kernel = _native.last_kernel()
    torch.cuda.synchronize()
    return out.cpu(), kernel


def _some(HQ, HK):
    """First and last head of every group."""
    group = HQ // HK
    return [h * group + i for h in range(HK) for i in sorted({0, group - 1})]


def _check(inputs, dt, cache, scale, kernel, causal=True, window=0, more_tol=0.0, against=None, **forms):
    """Both ways by the formula, in the first and last head of every group (`against`: what the formula is taken of)."""
    heads = _some(inputs[0].shape[1], inputs[1][0].shape[1])
    q, caches, *rest = inputs if against is None else against
    few = {**forms, "slopes": None if forms.get("slopes") is None else forms["slopes"][heads]}
    want, tol = ref_attention(q[:, heads], caches, cache, *rest, scale, causal, window, fine=True, **few)
    whole, ran = _whole(inputs, dt, cache, scale, causal, window, **forms)
    assert kernel in ran, ran
    for got in (whole, _attend(inputs, dt, cache, scale, causal, window, **forms).cpu()):
        got = got[:, heads].double()
        finite = want.isfinite()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~finite].nan_to_num(0), want[~finite].nan_to_num(0))
        _close(got[finite], want[finite], (tol + more_tol)[finite], ran)


@pytest.mark.gpu
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("shape,D,rows", [(TILE, 64, 128), (SHARED, 96, 128), (TILE, 128, 128), (WIDE, 256, 128),
                                          (HIGH, 64, 256), (HIGH, 96, 256), (HIGH, 128, 256)], ids=str)
def test_int4_masked_values_do_not_reach_a_row(gpu, shape, D, rows, dt, biased):
    """Groups whose values are not finite, in the last tokens and in the middle of the chunk: rows that do not see them
    are as without them, those that do have them in those columns alone."""
    new, HQ, HK = shape
    kv, PAGE = new + 70, 16
    inputs = _inputs(26, dt, "int4", [(new, kv)], HQ, HK, D, PAGE, poison=False)
    pairs, table = inputs[1][3], inputs[2]
    for token, group, pair in ((kv - 1, 0, [0.0, float("nan")]), (kv - 2, 1, [0.0, float("inf")]),
                               (kv - new // 2, D // 32 - 1, [0.0, float("-inf")]), (kv - 40, 0, [8192.0, 60000.0])):
        pairs[int(table[0, token // PAGE]), :, token % PAGE, group] = torch.tensor(pair, dtype=torch.float16)
    # the last of them: finite, but no f16 holds the values of codes from one on, which are infinite then
    page, place = int(table[0, (kv - 40) // PAGE]), (kv - 40) % PAGE
    inputs[1][1][page, :, place, :16] = 0xff
    told = inputs[0], [*inputs[1][:3], pairs.clone()], *inputs[2:]
    told[1][3][page, :, place, 0] = torch.tensor([0.0, float("inf")], dtype=torch.float16)
    slopes = torch.full((HQ,), 0.001) if biased else None
    _check(inputs, dt, "int4", D ** -0.5, _kernel(rows, D), slopes=slopes, against=told)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,cache", [("f16", "same"), ("bf16", "same"), ("f16", "fp8"), ("bf16", "int4")])
def test_masked_values_of_a_mixture(gpu, dt, cache):
    """Both halves of one launch, values that are not finite in the last token of each sequence."""
    lens = [(1, 300), (700, 900), (2, 40), (3, 3)]
    inputs = _inputs(27, dt, cache, lens, 8, 2, 64, 16, poison=False)
    for s, (_, kv) in enumerate(lens):
        page, place = int(inputs[2][s, (kv - 1) // 16]), (kv - 1) % 16
        if cache == "same":
            inputs[1][1][page, :, place, 5] = float("inf")
        elif cache == "fp8":
            inputs[1][1].view(torch.uint8)[page, :, place, 5] = 0x7f
        else:
            inputs[1][3][page, :, place, 1] = torch.tensor([0.0, float("nan")], dtype=torch.float16)
    for forms in ({}, {"cap": 30.0}, {"slopes": torch.full((8,), 0.001)}):
        _check(inputs, dt, cache, 0.125, "attn_mixed_kernel", **forms)


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [2.0 ** -100, 0.01, 100.0, 4096.0])
@pytest.mark.parametrize("shape,D,rows", [(TILE, 64, 128), (SHARED, 128, 128), (HIGH, 64, 256)], ids=str)
@pytest.mark.parametrize("cache", ["same", "fp8", "int4"])
def test_caps_of_many_sizes(gpu, cap, shape, D, rows, cache):
    new, HQ, HK = shape
    inputs = _inputs(35, "f16", cache, [(new, new + 150)], HQ, HK, D, 16, q_std=4.0)
    for slopes in (None, torch.tensor([0.5, 0.0, 0.01, 1.0] * (HQ // 4))):
        _check(inputs, "f16", cache, D ** -0.5, _kernel(rows, D), cap=cap, slopes=slopes)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.2, 3e-36, 3.0])
@pytest.mark.parametrize("cache", ["same", "fp8", "int4"])
def test_scales(gpu, scale, cache):
    inputs = _inputs(36, "bf16", cache, [(180, 400)], 16, 2, 128, 16, q_std=0.5)
    slopes = torch.tensor([0.5, 0.0, 0.01, -0.02] * 4)
    for forms in ({}, {"cap": 7.0}, {"slopes": slopes},
                  {"cap": 2.0, "slopes": slopes, "prefix": torch.tensor([250], dtype=torch.int32)}):
        _check(inputs, "bf16", cache, scale, _kernel(128, 128), **forms)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("std", [1e-6, 3e3])
@pytest.mark.parametrize("shape,D,rows", [(TILE, 64, 128), (WIDE, 256, 128), (HIGH, 128, 256)], ids=str)
def test_int4_queries_of_many_sizes(gpu, dt, std, shape, D, rows):
    """Rows far below and above one, and a row that holds both ends."""
    new, HQ, HK = shape
    inputs = _inputs(25, dt, "int4", [(new, new + 60)], HQ, HK, D, 16, q_std=std)
    inputs[0][-1, :, ::3] *= 2.0 ** -9
    if dt == "bf16" and std < 1:
        inputs[0][-1] *= 2.0 ** -60
        inputs[0][0, 0] = 0
    _check(inputs, dt, "int4", 0.3 / max(std, 1.0), _kernel(rows, D))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_int4_queries_that_are_not_finite(gpu, dt):
    """A query that holds an infinity or NaN leaves the other rows alone."""
    inputs = _inputs(37, dt, "int4", [(360, 420)], 8, 1, 64, 16)
    want, tol = ref_attention(inputs[0], inputs[1], "int4", *inputs[2:], 0.125, True, 0, fine=True)
    inputs[0][0, 1, 5], inputs[0][-1, 7, 9] = float("inf"), float("nan")
    out, ran = _whole(inputs, dt, "int4", 0.125)
    assert _kernel(128, 64) in ran, ran
    bad = torch.zeros(360, 8, dtype=torch.bool)
    bad[0, 1], bad[-1, 7] = True, True
    assert bool(out[bad].isnan().any(-1).all())
    _close(out[~bad], want[~bad], tol[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("shape,rows", [(TILE, 128), (HIGH, 256)], ids=str)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_int4_pairs_of_many_sizes(gpu, dt, shape, rows):
    """Scales below zero, zero, of f16's subnormals and large ones; lowest values far off."""
    new, HQ, HK = shape
    inputs = _inputs(38, dt, "int4", [(new, new + 100)], HQ, HK, 128, 16)
    for i in (2, 3):
        pairs = inputs[1][i]
        pairs[..., 0, 0] = -pairs[..., 0, 0].abs()
        pairs[..., 1, 0] = 0
        pairs[..., 2, :] = torch.tensor([3 * 2.0 ** -24, -5 * 2.0 ** -24])
        pairs[..., 3, :] = torch.tensor([4096.0, -30720.0]) if i == 3 else torch.tensor([1.0, 32.0])
    _check(inputs, dt, "int4", 0.02, _kernel(rows, 128))


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "int4"])
def test_distances_past_24_bits(gpu, cache):
    """Positions that no f32 tells apart: with steep slopes the tokens behind 2^24 others give what they give alone
    (weights of tokens 1024 and more away are below 2^-1000)."""
    new, HQ, HK, D, PAGE, near = 360, 8, 1, 64, 256, 2048
    inputs = _inputs(39, "f16", cache, [(new, near)], HQ, HK, D, PAGE, poison=False)
    far = (1 << 24) + 3 * PAGE
    long = torch.cat((torch.zeros(1, far // PAGE, dtype=torch.int32), inputs[2]), 1)
    _check((*inputs[:2], long, inputs[3], torch.tensor([far + near], dtype=torch.int32)), "f16", cache, 0.125,
           _kernel(128, 64), slopes=torch.tensor([1.0, 2.0, 1.5, 30.0] * 2), against=inputs, more_tol=2.0 ** -20)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "fp8", "int4"])
@pytest.mark.parametrize("shape,D,rows,PAGE", [(TILE, 64, 128, 2), (SHARED, 96, 128, 8), (TILE, 128, 128, 4),
                                               (WIDE, 256, 128, 4), (HIGH, 64, 256, 8), (HIGH, 96, 256, 2),
                                               (HIGH, 128, 256, 1)], ids=str)
def test_pages_smaller_than_a_load(gpu, shape, D, rows, PAGE, cache):
    new, HQ, HK = shape
    lens = [(new, new + 130)]
    inputs = _inputs(40, "bf16", cache, lens, HQ, HK, D, PAGE)
    for forms in ({}, {"cap": 20.0, "slopes": torch.full((HQ,), 0.01), "prefix": _prefixes(lens, 1)}):
        _check(inputs, "bf16", cache, D ** -0.5, _kernel(rows, D), window=200 if forms else 0, **forms)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "fp8", "int4"])
def test_bad_pages_and_lengths(gpu, cache):
    """Page ids, lengths and prefixes outside the cache are clamped: the formula over the clamped ones."""
    inputs = list(_inputs(27, "f16", cache, [(180, 290), (180, 200)], 8, 1, 64, 16, poison=False))
    inputs[2][0, 1], inputs[2][1, 0] = 10 ** 6, -7
    inputs[4][1] = 10 ** 6
    for forms in ({}, {"prefix": torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32), "cap": 9.0}):
        _check(inputs, "f16", cache, 0.125, _kernel(128, 64), **forms)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "int4"])
@pytest.mark.parametrize("lens,HQ,kernel", [([(360, 430)], 8, "128 rows>"), ([(1, 130), (720, 800)], 4, "attn_mixed_kernel")],
                         ids=str)
def test_far_pages(gpu, lens, HQ, kernel, cache):
    """Pages past 2^31 bytes from the cache's start."""
    inputs = list(_inputs(34, "f16", cache, lens, HQ, 1, 64, 64, poison=False))
    caches, far = inputs[1], []
    pages = caches[0].shape[0]
    step = (1 << 31) // (pages - 1) // 16 * 16 + 4096
    for c in caches:  # the same rows, each page `step` elements behind the last
        flat = torch.zeros((pages - 1) * step + c[0].numel(), dtype=c.dtype, device="cuda")
        view = flat.as_strided(c.shape, (step, *c.contiguous().stride()[1:]))
        view.copy_(c)
        far.append(view)
    for forms in ({}, {"slopes": torch.full((HQ,), 0.01)}):
        _check(inputs, "f16", cache, 0.125, kernel, **forms)
        assert torch.equal(_attend([inputs[0], far, *inputs[2:]], "f16", cache, 0.125, **forms),
                           _attend(inputs, "f16", cache, 0.125, **forms))


@pytest.mark.gpu
@pytest.mark.parametrize("news,D", [((200, 200), 128), ((1, 700), 64)], ids=str)
def test_captured_and_replayed(gpu, news, D):
    """Append and attention of a chunk (tiles; both lists) in a graph, replayed over lengths, slots, slopes and prefixes
    that change in place, with eager calls of the same operators in between: every replay equals the eager step."""
    HQ, HK, PAGE, T = 8, 2, 16, sum(news)
    heads = list(_cuda(*_heads(41, "bf16", T, HQ, HK, D, D, "qk", length=1600)))
    inputs = _inputs(42, "bf16", "int4", [(n, 1500 - 100 * s) for s, n in enumerate(news)], HQ, HK, D, PAGE, poison=False)
    caches, (table, offsets, kv) = _cuda(*inputs[1]), _cuda(*inputs[2:])
    slots = torch.zeros(T, dtype=torch.int32, device="cuda")
    slopes, prefix = torch.ones(HQ, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    q_out, out = (torch.empty(T, HQ, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    calls = [_compile("paged_kv_append", "bf16", "int4").prepare(*heads, slots, *caches, outputs=(q_out,)),
             _compile("biased_paged_attention", "bf16", "int4", SOFTCAP=10.0).prepare(
                 q_out, *caches, table, offsets, kv, slopes, prefix, 0.0884, outputs=(out,))]

    def place(*ends):
        at = torch.cat([torch.arange(e - n, e) for n, e in zip(news, ends)])
        row = torch.arange(2).repeat_interleave(torch.tensor(news))
        slots.copy_((inputs[2][row, at // PAGE].long() * PAGE + at % PAGE).to(torch.int32))
        kv.copy_(torch.tensor(ends, dtype=torch.int32))
        prefix.copy_(torch.tensor([ends[0] // 2, ends[1]], dtype=torch.int32))
        slopes.copy_(torch.rand(HQ, generator=_gen(ends[0])) * 0.1)
        heads[6].copy_(at.to(torch.int32))

    place(1500, 1400)
    _, ran = _whole((torch.zeros(T, HQ, D, dtype=torch.bfloat16), [c.cpu() for c in caches], *inputs[2:]), "bf16", "int4", 0.0884, cap=10.0,
                    slopes=slopes.cpu(), prefix=prefix.cpu())
    assert "attn_mixed_kernel" in ran if D == 64 else _kernel(128, D) in ran, ran
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        [c.launch() for c in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        [c.launch() for c in calls]
    for ends in ((1500, 1400), (news[0], 1399), (756, news[1]), (1503, 1408)):
        place(*ends)
        [c.launch() for c in calls]
        kept = [t.clone() for t in (out, *caches)]
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, *caches), kept)), ends
