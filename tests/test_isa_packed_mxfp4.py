"""The loops of the MXFP4 product and of packed attention order LDS reads, DMA, counted waits, barriers and MFMAs by hand.
These tests compile the kernels to gfx950 assembly (no GPU needed) and check that the steady-state loops hold what they
are meant to: their MFMAs, no spill, and no wait for all DMA that the compiler put in by itself."""
import re

import pytest

from test_isa_schedule import CSRC, HIPCC

FLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def listing(src, tmp_path, *extra):
    import os
    import subprocess
    out = tmp_path / (src + ".s")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fno-gpu-rdc", "-S", "--cuda-device-only", *FLAGS,
                    *extra, os.path.join(CSRC, src), "-o", str(out)], check=True, capture_output=True)
    return out.read_text()


def kernels(text, name):
    """{mangled name: whole body} of the instantiations of `name`"""
    return {m.group(1): text[m.end():text.index(".end_amdhsa_kernel", m.end())]
            for m in re.finditer(r"^(_ZN\S*%s\S*):\s" % name, text, re.M)}


def blocks(body):
    """basic blocks of a kernel body: lists of instructions"""
    cur, out = [], []
    for ln in body.split("\n"):
        ln = ln.split(";")[0].strip()
        if ln.startswith(".LBB"):
            out.append(cur)
            cur = []
        elif ln and not ln.startswith("."):
            cur.append(ln)
    return out + [cur]


def count(block, start):
    return sum(i.startswith(start) for i in block)


@pytest.fixture(scope="module")
def mx(tmp_path_factory):
    return listing("mxfp4.hip", tmp_path_factory.mktemp("mx"))


def test_mxfp4_big_kernel_loop(mx):
    found = kernels(mx, "gemm_mxfp4_big_kernel")
    assert len(found) == 5                                         # one per epilogue
    for name, body in found.items():
        loop = next(b for b in blocks(body) if count(b, "v_mfma") == 64 and count(b, "global_load_lds") == 10)
        assert count(loop, "v_mfma_scale_f32_16x16x128_f8f6f4") == 64
        assert count(loop, "s_barrier") == 8
        waits = [i for i in loop if i.startswith("s_waitcnt") and "vmcnt" in i]
        assert len(waits) == 3 and all("vmcnt(10)" in w for w in waits), waits
        assert count(loop, "scratch_") == 0 and count(loop, "global_load_dword ") == 0


def test_no_packed_fp32(mx):
    assert not re.search(r"v_pk_(add|mul|fma)_f32", mx)


def test_packed_attention_loop(tmp_path):
    text = listing("attn_packed.hip", tmp_path, "-fno-slp-vectorize")
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
    for d, mfma in ((128, 32), (64, 16)):
        body = next(b for n, b in kernels(text, f"attn_packed_kernelILi{d}ELi8ELb0E").items())
        # the unmasked steps: S^T of the next tile and P V of this one, neither spilled nor masked
        steps = [b for b in blocks(body) if count(b, "v_exp_f32") >= 20 and count(b, "v_mfma") >= mfma - 4
                 and count(b, "v_cndmask") < 8 and count(b, "ds_read_b64_tr_b16") >= mfma // 2]
        assert steps, f"no steady-state step found for head_dim {d}"
        assert all(count(b, "scratch_") == 0 for b in steps)
        # the DMA of a step is waited for at its end, not ahead of the reads of V
        for b in steps:
            reads = [i for i, x in enumerate(b) if x.startswith("ds_read_b64_tr_b16")]
            assert not [x for x in b[:reads[-1]] if x.startswith("s_waitcnt") and "vmcnt" in x]
