"""csrc/shared_list.h: every place of the list that block_kernel reads is written, also where groups overlap and have more items than
there are places. Built by the host compiler."""
import os
import subprocess

from tests.conftest import ROOT

PROGRAM = r"""
#include <vector>
#include "shared_list.h"

// The list as write_plan fills it: each group's items, then the places without one, of 32-bit numbers that may wrap.
static std::vector<int> filled(const std::vector<int>& groups, int room) {
    std::vector<int> list(room + 1, 7);               // 7: whatever the workspace held
    int base = 0;
    for (int items : groups) {
        for (int i = 0, n = ixg::items_listed(base, items, room); i < n; ++i) list.at(base + i) = 1;
        base = (int)((unsigned)base + (unsigned)items);
    }
    for (int i = ixg::list_end(base, room); i <= room; ++i) list.at(i) = -1;
    return list;
}

int main() {
    // room = n_shared / h_kv; n_shared is a multiple of the workgroups that the chip holds
    for (int n_shared : {256, 512, 768})
        for (int h_kv : {1, 2, 3, 5, 7, 8, 12, 300}) {
            const int room = n_shared / h_kv;
            for (int items : {0, 1, 40, 64, 300, 1 << 20, 0x7fffffff, -5})
                for (int n : {0, 1, 2, 3, 17, 700}) {
                    const std::vector<int> list = filled(std::vector<int>(n, items), room);
                    for (int x : list)
                        if (x != 1 && x != -1) return 1;
                    if (list[room] != -1) return 2;
                    // what is allowed: all items listed, and no others
                    if (items >= 0 && (long long)items * n <= room)
                        for (int i = 0; i <= room; ++i)
                            if (list[i] != (i < items * n ? 1 : -1)) return 3;
                }
        }
    return 0;
}
"""


def test_every_place_is_written(tmp_path):
    (tmp_path / "list.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "baloon_amd", "csrc"), str(tmp_path / "list.cpp"), "-o",
                    str(tmp_path / "list")], check=True)
    assert subprocess.run([str(tmp_path / "list")]).returncode == 0


def test_the_kernel_fills_it_so():
    text = open(os.path.join(ROOT, "baloon_amd", "csrc", "kv8_shared.hip")).read()
    assert "items_listed(" in text and "list_end(" in text and text.count("shared_items[") == 2
