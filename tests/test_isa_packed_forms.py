"""Every instantiation of packed attention as it is built: the inline assembly that starts its DMA, and where registers are
spilled (no GPU needed)."""
import os
import re
import subprocess

import pytest

from test_build_flags import shipped_flags
from test_isa_schedule import CSRC, HIPCC

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not found")


@pytest.fixture(scope="module")
def text(tmp_path_factory):
    out = tmp_path_factory.mktemp("packed") / "attn_packed.s"
    subprocess.run([HIPCC, *shipped_flags("attn_packed.hip"), "-S", "--cuda-device-only", os.path.join(CSRC, "attn_packed.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    return out.read_text()


def inline_blocks(text):
    """instructions of each inline-assembly block, and all instructions outside of them"""
    inside, outside, block = [], [], None
    for ln in text.split("\n"):
        if "ASMSTART" in ln:
            block = []
        elif "ASMEND" in ln:
            inside.append(block)
            block = None
        else:
            ins = ln.split(";")[0].strip()
            if ins and not ins.startswith(".") and not ins.endswith(":"):
                (outside if block is None else block).append(ins)
    return inside, outside


def test_dma_blocks_wait_for_their_scalar_operands(text):
    """a vector instruction may have written the address pair (v_readlane of a spilled one, v_readfirstlane): a load may read
    it 5 wait states later, and the compiler does not look into the assembly to put them in"""
    inside, outside = inline_blocks(text)
    dma = [b for b in inside if any(i.startswith("global_load_lds") for i in b)]
    assert len(dma) > 100
    for block in dma:
        at = next(n for n, i in enumerate(block) if i.startswith("global_load_lds"))
        states = sum(1 + (int(i.split()[1]) if i.startswith("s_nop") else 0) for i in block[:at])
        assert states >= 5, block
        for n, i in enumerate(block[1:], 1):                 # m0 is read one wait state after its write
            assert not (i.startswith("global_load_lds") and re.search(r"\bm0,", block[n - 1])), block
        # m0 is this block's alone: written in front of the load, and used by nothing else in the file
        assert block[0].startswith("s_mov_b32 m0,")
    assert not [i for i in outside if re.search(r"\bm0\b", i)]


def test_no_form_but_one_spills(text):
    found = dict(re.findall(r"\.name:\s+(\S*attn_packed\S*).*?\.private_segment_fixed_size: (\d+)", text[text.index("amdhsa.kernels"):], re.S))
    assert len(found) == 26                                  # 2 head sizes x 4 launch forms x 3 caps, and the joins
    for name, scratch in found.items():
        # the four-wave form with split keys at head_dim 128 keeps about 70 values in scratch
        assert int(scratch) == 0 or "attn_packed_split_kernelILi128ELi4E" in name, (name, scratch)
