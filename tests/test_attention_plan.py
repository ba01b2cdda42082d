"""What the attention over a paged cache takes of the GPU and how it plans a batch, without one (CPU)."""
import re
import shutil
from pathlib import Path

import pytest
import torch

from intent_amd import _native
from intent_amd import build as B
from intent_amd import codeobj_check as C
from test_attention import runtime_for

LDS_OF_A_CU, LDS_STEP = 160 * 1024, 1280  # gfx950 gives LDS out in steps of 320 words

_MIXED = '#include "paged_attn_mfma.h"\ntemplate __global__ void intent::attn::attn_mixed_kernel<false, intent::%s, intent::kPlain>' \
         '(const intent::AttnArgs, const intent::AttnArgs, int);\n'


@pytest.mark.skipif(shutil.which(B.hipcc()) is None and not Path(B.hipcc()).exists(), reason="hipcc not available")
@pytest.mark.parametrize("cache", ["kCacheSame", "kCacheFp8"])
def test_three_workgroups_of_both_lists_share_a_cu(tmp_path, cache):
    """The kernel of both lists is bound to registers for three workgroups to a CU: its LDS lets in as many."""
    src = tmp_path / "mixed.hip"
    src.write_text(_MIXED % cache)
    code = C.extract_device_code(B._compile(src, tmp_path, (f"-I{B.CSRC}",)), tmp_path / "mixed.co")
    notes = C._run([C._tool("llvm-readelf"), "--notes", str(code)])
    sizes = [int(n) for n in re.findall(r"\.group_segment_fixed_size:\s+(\d+)", notes)]
    assert len(sizes) == 1 and 3 * (-(-sizes[0] // LDS_STEP) * LDS_STEP) <= LDS_OF_A_CU


def _scratch(T, S, HQ, HK, cache, tokens=4096):
    """Bytes for the parts of a batch of heads of 64: two lists of tiles need others than one."""
    return _native.library().intent_biased_paged_attention_workspace_size(T, HQ, HK, 64, S, tokens // 32, 32, cache)


@pytest.mark.parametrize("cache", [0, 1, 2])
@pytest.mark.parametrize("T,S,HQ,HK", [(301, 100, 32, 32), (101, 40, 128, 8), (301, 64, 32, 8), (561, 16, 32, 32),
                                       (841, 24, 12, 12), (363, 64, 32, 32), (231, 32, 64, 64)])
def test_batches_of_few_rows_take_one_list(T, S, HQ, HK, cache):
    """Drafts, and a small chunk beside decoding sequences: mean sequences of up to 64 rows and up to 2048 rows of a
    cached head in all take the same plan whether or not the sequences divide the tokens."""
    assert T % S and T * HQ // HK <= 2048 and T * HQ >= 8192
    even = T // S * S if -(-(T // S * HQ // HK) // 16) == -(-(-(-T * HQ // HK // S)) // 16) else -(-T // S) * S
    assert _scratch(T, S, HQ, HK, cache) == _scratch(even, S, HQ, HK, cache)


@pytest.mark.parametrize("cache", [0, 1, 2])
@pytest.mark.parametrize("T,S,HQ,HK", [(1925, 24, 12, 12), (929, 23, 16, 8), (1519, 13, 12, 12), (1921, 24, 14, 2)])
def test_chunks_beside_decoding_sequences_take_two(T, S, HQ, HK, cache):
    """Mean sequences of more than 64 rows, where the table holds more than 1024 tokens, or more than 2048 rows."""
    one = _scratch(T // S * S, S, HQ, HK, cache)
    assert _scratch(T, S, HQ, HK, cache) != one
    short = _scratch(T, S, HQ, HK, cache, 1024) != _scratch(T // S * S, S, HQ, HK, cache, 1024)
    assert short == (T * HQ // HK > 2048)


def test_a_layout_that_comes_once_is_not_made_out(monkeypatch):
    """The call of a layout is made out when it comes again: first calls of a program whose token count changes with
    every step do not pay for it."""
    rt = runtime_for("paged_kv_read")
    rt._home = torch.device("cpu")
    monkeypatch.setattr(_native, "call_packed", lambda entry, arguments, stream: None)
    monkeypatch.setattr("intent_amd.runtime._current_stream", lambda device: 0)
    calls = []
    monkeypatch.setattr(rt, "_template", lambda *a, make=rt._template: calls.append(a) or make(*a))
    caches = [torch.zeros(3, 2, 8, 64).half() for _ in range(2)]
    for n in range(1, 6):
        rt.run(*caches, torch.zeros(n, dtype=torch.int32))
    assert not calls
    for _ in range(3):
        bound = rt.rebind((*caches, torch.zeros(4, dtype=torch.int32)), False)
        assert bound.call is not None and bound.outputs[0].shape == (4, 2, 64)
    assert len(calls) == 1
