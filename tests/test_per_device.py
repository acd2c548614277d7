"""csrc/per_device.h: what a process sets once a device, of which a box with one GPU shows one. Built by the host compiler."""
import os
import subprocess

from tests.conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include "per_device.h"

int main() {
    ixg::OncePerDevice once;
    int calls = 0, answer = 7;
    auto on = [&](int dev) { return once(dev, [&] { ++calls; return answer; }); };
    // a failure is the call's, and is not kept
    if (on(0) != 7 || on(0) != 7 || calls != 2) return 1;
    answer = 0;
    if (on(0) != 0 || calls != 3) return 2;
    answer = 7;
    if (on(0) != 0 || calls != 3) return 3;
    // each device for itself, from the first to the last, and those beyond each time
    if (on(1) != 7 || on(63) != 7 || calls != 5) return 4;
    answer = 0;
    if (on(1) != 0 || on(63) != 0 || on(1) != 0 || on(63) != 0 || calls != 7) return 5;
    if (on(64) != 0 || on(64) != 0 || on(-1) != 0 || calls != 10) return 6;
    return 0;
}
"""


def test_once_per_device(tmp_path):
    (tmp_path / "once.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "baloon_amd", "csrc"), str(tmp_path / "once.cpp"), "-o",
                    str(tmp_path / "once")], check=True)
    assert subprocess.run([str(tmp_path / "once")]).returncode == 0


def test_no_kernel_is_set_up_once_a_process():
    """A static of hipFuncSetAttribute's answer holds the first call's device and error for good."""
    csrc = os.path.join(ROOT, "baloon_amd", "csrc")
    for f in sorted(os.listdir(csrc)):
        text = open(os.path.join(csrc, f)).read()
        assert "hipFuncSetAttribute" not in text or f == "gdn_common.h", f
