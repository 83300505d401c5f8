"""Waits of the gated linear recurrence's kernels, without a GPU: one that gives up is the last one of its thread.

A lost message may cost one limit (2 s), not one per round (a column of 65536 steps has up to 128 rounds).  The class that
remembers it is compiled for the host and run there; that the kernels wait through nothing else is read from their source.
"""
import os
import re
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "sru_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "common.cuh"
int main() {
    srub::Patience patience;
    int tried = 0, gave_up = 0;
    auto round = [&](bool arrives) { patience.wait([&]() { ++tried; return arrives; }, [&]() { ++gave_up; }); };
    for (int i = 0; i < 5; ++i) round(true);
    if (tried != 5 || gave_up != 0 || patience.gone) return 1;
    for (int i = 0; i < 128; ++i) round(false);
    if (tried != 6 || gave_up != 1 || !patience.gone) return 2;
    round(true);
    return tried == 6 && gave_up == 1 ? 0 : 3;
}
"""


def test_the_first_wait_that_gives_up_is_the_last(tmp_path):
    src, exe = tmp_path / "patience.cu", tmp_path / "patience"
    src.write_text(PROGRAM)
    nvcc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    build = subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, str(src), "-o", str(exe)],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    assert subprocess.run([str(exe)], timeout=60).returncode == 0


def test_every_wait_of_the_recurrence_is_remembered():
    with open(os.path.join(CSRC, "linear_recurrence.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert code.count("mbar_wait_bounded(") == 1 and "mbar_try_wait" not in code
    helper = code[code.index("void wait_for("):]
    helper = helper[:helper.index("\n}")]
    assert "patience.wait(" in helper and "mbar_wait_bounded(bar, parity)" in helper
    assert code.count("wait_for(") >= 6            # both directions' rings, their asking warps, the exchange
