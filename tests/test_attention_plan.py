"""What the attention over a paged cache takes of the GPU and how it plans a batch, without one (CPU)."""
import re
import shutil
from pathlib import Path

import pytest

from intent_amd import build as B
from intent_amd import codeobj_check as C

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
