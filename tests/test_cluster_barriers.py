"""Cluster barriers of the kernels (no GPU): the .aligned forms are undefined for a warp whose lanes are not
together, so they are issued in one place, each behind a __syncwarp()."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-sglang-cpp_b200", "csrc")


def test_every_aligned_cluster_barrier_follows_a_syncwarp():
    found = {}
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*")) + glob.glob(os.path.join(CSRC, "*.h"))):
        lines = open(path).read().split("\n")
        for i, line in enumerate(lines):
            for _ in re.findall(r"barrier\.cluster\.\w+[.\w]*", line):
                found.setdefault(os.path.basename(path), []).append(lines[i - 1].strip())
    assert found == {"common.cuh": ["__syncwarp();"] * 2}, found
