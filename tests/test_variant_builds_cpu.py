"""The tools that build variants of the library compile every translation unit with the library's own flags (a different set of fused instructions rounds
differently, and byte comparisons with the variant would be void)."""
import os
import stat
import subprocess
import sys

import pytest

from propainter_amd import build as pbuild

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def fake_tree(tmp_path, tool):
    """a copy of the tool beside the package's flags and sources, with a compiler that writes down how it was called"""
    for d in ("tools", "propainter_amd/csrc", "propainter_amd/lib/obj", "bin"):
        os.makedirs(tmp_path / d)
    hipcc = tmp_path / "bin" / "hipcc"
    hipcc.write_text('#!/bin/bash\necho "$@" >> ' + str(tmp_path / "calls") + '\nwhile [ $# -gt 0 ]; do if [ "$1" = -o ]; then touch "$2"; fi; shift; done\n')
    hipcc.chmod(hipcc.stat().st_mode | stat.S_IXUSR)
    text = open(os.path.join(ROOT, "tools", tool)).read()
    assert "/opt/rocm/bin/hipcc" in text
    (tmp_path / "tools" / tool).write_text(text.replace("/opt/rocm/bin/hipcc", str(hipcc)))
    for f in ("__init__.py", "build.py"):
        (tmp_path / "propainter_amd" / f).write_text(open(os.path.join(ROOT, "propainter_amd", f)).read())
    for s in pbuild.sources():
        text = open(os.path.join(pbuild.CSRC, s)).read()
        (tmp_path / "propainter_amd" / "csrc" / s).write_text(text)
        (tmp_path / "propainter_amd" / "lib" / "obj" / s.replace(".hip", ".0.o")).write_text("")
    for h in os.listdir(pbuild.CSRC):
        if h.endswith(".h"):
            (tmp_path / "propainter_amd" / "csrc" / h).write_text(open(os.path.join(pbuild.CSRC, h)).read())


@pytest.mark.parametrize("tool,command,units", [("build_variant.sh", ["bash", "tools/build_variant.sh", "v"], None),
                                                ("build_h8_variant.sh", ["bash", "tools/build_h8_variant.sh", "v"], ["conv_gemm_v3.hip", "conv_gemm_v3s.hip"]),
                                                ("build_lds_variants.py", [sys.executable, "tools/build_lds_variants.py"], None)])
def test_variants_are_compiled_with_the_library_flags(tmp_path, tool, command, units):
    fake_tree(tmp_path, tool)
    subprocess.run(command, cwd=tmp_path, check=True, capture_output=True, timeout=100)
    calls = [c for c in open(tmp_path / "calls").read().splitlines() if " -c " in c]
    for s in units or pbuild.sources():
        mine = [c for c in calls if c.split(" -c ")[1].split()[0].endswith("/" + s)]
        assert mine, s
        assert all(c.startswith(" ".join(pbuild.flags(s)) + " ") for c in mine), (s, mine)


def test_flags_of_a_unit():
    assert pbuild.flags("conv_gemm_v3.hip")[-1] == "-fma-mix-insts" and "-fma-mix-insts" not in pbuild.flags("conv_gemm.hip") and "-packed-fp32-ops" in pbuild.flags("conv_gemm.hip")
