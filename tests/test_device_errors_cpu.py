"""The texts that tb_ctx_check_device reports: one for each word that a kernel may leave, and none that
names a kernel which other kernels share the word with (conv, linear and attention kernels all report a
bounded wait by the same one)."""
import os
import re
import shutil
import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include "tb_common.cuh"
int main() {
    for (int e = 0; e < 8; ++e) std::printf("%d|%s\n", e, tb_device_error_text(e));
    return 0;
}
"""


def test_texts(tb, tmp_path):
    from trellis_cpp_b200 import build
    if not os.path.exists(build.NVCC) and not shutil.which(build.NVCC):
        pytest.skip("nvcc not found")
    (tmp_path / "texts.cu").write_text(PROGRAM)
    b = subprocess.run([build.NVCC, "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I", build.CSRC,
                        str(tmp_path / "texts.cu"), "-o", str(tmp_path / "texts")], capture_output=True, text=True)
    assert b.returncode == 0, b.stderr
    r = subprocess.run([str(tmp_path / "texts")], capture_output=True, text=True, timeout=120)
    texts = dict(line.split("|") for line in r.stdout.splitlines())
    source = open(os.path.join(build.CSRC, "tb_common.cuh")).read()
    codes = {m[0]: m[1] for m in re.findall(r"(TB_DEVERR_\w+) = (\d+)", source) if m[1] != "0"}
    known = [texts[v] for v in codes.values()]
    assert len(set(known)) == len(known) and "unknown device error" not in known
    assert texts["7"] == "unknown device error"
    wait = texts[codes["TB_DEVERR_WAIT_TIMEOUT"]]
    assert "timed out" in wait and "conv" not in wait and "attention" not in wait
