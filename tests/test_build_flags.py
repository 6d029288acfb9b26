"""What is built, how, and what the tools and the assembly checks build: one list of objects, one set of flags."""
import os
import re
import subprocess

import pytest

import test_isa_schedule as schedule
from test_isa_schedule import CSRC, HIPCC, ROOT


def make_commands(target):
    """what `make` would run for `target` from scratch (file in the source folder, or the library)"""
    return subprocess.run(["make", "-C", CSRC, "-n", "-B", "HIPCC=hipcc", target], check=True, capture_output=True,
                          text=True).stdout


def flags_of(command, src):
    """a compile command's words without the compiler, the source, the output and the file's folder"""
    words = command.split()
    drop = {"-c", "-o", src, src[:-4] + ".o"}
    return [w for w in words[1:] if w not in drop and not w.endswith((".o", ".hip"))]


def shipped_flags(src):
    line = next(ln for ln in make_commands(src[:-4] + ".o").splitlines() if " -c " in ln)
    return flags_of(line, src)


@pytest.mark.parametrize("src", ["attn.hip", "attn_packed.hip", "sampler.hip", "rope.hip", "api.hip"])
def test_variant_tool_builds_what_make_builds(tmp_path, src):
    """tools/build_variant.sh with a compiler that only writes down how it was called"""
    fake, log = tmp_path / "hipcc", tmp_path / "calls"
    fake.write_text(f"#!/bin/sh\necho \"$@\" >> {log}\n")
    fake.chmod(0o755)
    env = dict(os.environ, HIPCC=str(fake), OUT=str(tmp_path / "out"))
    subprocess.run(["bash", os.path.join(ROOT, "tools", "build_variant.sh"), "v1", src, "-DVARIANT=1"], check=True, env=env,
                   capture_output=True)
    compile_line, link_line = log.read_text().splitlines()
    assert flags_of("hipcc " + compile_line, src) == shipped_flags(src) + ["-DVARIANT=1"]
    objs = re.search(r"^OBJS\s*=(.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1).split()
    linked = [w for w in link_line.split() if w.endswith(".o")]
    assert [os.path.basename(o).replace("_v1.o", ".o") for o in linked] == objs
    assert [o for o in linked if o.endswith("_v1.o")] == [str(tmp_path / "out" / (src[:-4] + "_v1.o"))]
    assert "--offload-arch=gfx950" in link_line and "-shared" in link_line


def test_every_kernel_file_is_built_without_packed_fp32():
    for src in sorted(f for f in os.listdir(CSRC) if f.endswith(".hip")):
        flags = shipped_flags(src)
        assert " ".join(flags).count("-Xclang -target-feature -Xclang -packed-fp32-ops") == 1, (src, flags)


@pytest.fixture
def shipped(monkeypatch, tmp_path):
    """the assembly checks of test_isa_schedule on the code as it is built"""
    def listing(src, where):
        out = where / (src + ".s")
        subprocess.run([HIPCC, *shipped_flags(src), "-S", "--cuda-device-only", os.path.join(CSRC, src), "-o", str(out)],
                       check=True, capture_output=True)
        text = out.read_text()
        assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
        return text
    monkeypatch.setattr(schedule, "listing", listing)
    return tmp_path


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not found")
def test_loops_as_built(shipped):
    schedule.test_phased_gemm_loop_keeps_its_order(shipped, "gemm256.hip", "gemm256_kernel", 16, 4)
    schedule.test_phased_gemm_loop_keeps_its_order(shipped, "fp8.hip", "gemm_fp8p_kernel", 4, 5)
    schedule.test_gemm_bias_loads_hidden_from_the_compiler_are_not_touched_before_their_wait(shipped)
    for src, kernel, count in (("attn.hip", "attn_pipe_kernel", 2), ("attn.hip", "attn_i8_kernel", 2),
                               ("vae.hip", "conv3d_cl_kernel", 8)):
        schedule.test_register_bound_loops_do_not_spill(shipped, src, kernel, count)
