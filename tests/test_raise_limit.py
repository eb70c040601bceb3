"""The record of a kernel's shared-memory limit under two host threads (no GPU): a thread that needs less
must not lower what another has set and recorded."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "mini-sglang-cpp_b200", "csrc")

PROGRAM = r"""
#include <stdio.h>

#include <chrono>
#include <thread>

#include "raise_limit.h"

static std::atomic<int> done, limit, sets;
static std::atomic<bool> entered, large_set;

int set(int want) {
    ++sets;
    if (want == 100) {  // the small one is overtaken here if it can be
        entered = true;
        for (int i = 0; i < 300 && !large_set; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
    }
    limit = want;
    if (want == 200) large_set = true;
    return 0;
}

int main() {
    std::thread small([] { msgl::raise_limit(done, 100, set); });
    while (!entered) std::this_thread::yield();
    std::thread large([] { msgl::raise_limit(done, 200, set); });
    small.join(), large.join();
    printf("limit %d recorded %d sets %d\n", limit.load(), done.load(), sets.load());
    if (limit != 200 || done != 200) return 1;
    msgl::raise_limit(done, 150, set), msgl::raise_limit(done, 200, set);  // nothing to do
    if (sets != 2 || limit != 200) return 2;
    if (msgl::raise_limit(done, 300, [](int) { return 5; }) != 5 || done != 200) return 3;  // a failure is not recorded
    return 0;
}
"""


def test_the_limit_is_never_lowered(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    r = subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I" + CSRC, str(src), "-o", str(exe),
                        "-lpthread"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr)
