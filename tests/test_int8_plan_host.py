"""Which kernels int8 products take (csrc/gemm_i8_plan.h, compiled here on its own): the plan's properties over the
sizes, and that the GPU tests' sizes reach every kernel that any size reaches."""

from __future__ import annotations

import random
import shutil
import subprocess
from collections import namedtuple
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "ltx-2-mlx_amd" / "csrc"
Plan = namedtuple("Plan", "head head_bn bm bn splits k_split")
MAIN = """
#include "gemm_i8_plan.h"
#include <cinttypes>
#include <cstdio>
int main() {
  int64_t m, n, k;
  while (std::scanf("%" SCNd64 " %" SCNd64 " %" SCNd64, &m, &n, &k) == 3) {
    const ltx::I8Plan p = ltx::i8_plan(m, n, k);
    std::printf("%" PRId64 " %d %d %d %d %d\\n", p.head, p.head_bn, p.bm, p.bn, p.splits, p.k_split);
  }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    """f(sizes): their plans."""
    compiler = next((c for c in ("g++", "clang++", "/opt/rocm/llvm/bin/clang++") if shutil.which(c)), None)
    if compiler is None:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run([compiler, "-std=c++17", "-O1", f"-I{CSRC}", str(d / "main.cpp"), "-o", str(d / "plan")], check=True)

    def run(sizes):
        text = "".join(f"{m} {n} {k}\n" for m, n, k in sizes)
        out = subprocess.run([str(d / "plan")], input=text, capture_output=True, text=True, check=True).stdout
        return [Plan(*map(int, line.split())) for line in out.splitlines()]

    return run


def _sizes(count, seed=0):
    rng = random.Random(seed)

    def spread(hi):
        return int(hi ** rng.random())

    while count:
        m, n, k = spread(20000), 8 * spread(4096), 64 * spread(2046)
        if m * n * k <= 2e12:
            count -= 1
            yield m, n, k


def _kernels(plan):
    """The launches of a plan: (place, rows, columns of a tile or minus those of 16 of the few-row kernel, in K ranges)"""
    if plan.head:
        return {("head", 256, plan.head_bn, False), ("rest", plan.bm, plan.bn, False)}
    return {("whole", plan.bm, plan.bn, plan.splits > 1)}


def test_plans_are_ones_that_the_kernels_take(plans):
    sizes = [*_sizes(40000), (1, 8, 64), (1 << 27, 8, 64), (1, 1 << 27, 64), (33, 8, 131008), (1 << 17, 1 << 17, 4096)]
    for (m, n, k), p in zip(sizes, plans(sizes)):
        assert (p.bm, p.bn) in ((16, -1), (16, -2), (32, -1), (32, -2), (64, -1), (64, -2), (288, 256), (256, 256),
                                (256, 128), (128, 128), (64, 128)), (m, n, k, p)
        assert p.head % 256 == 0 and 0 <= p.head < m and p.head_bn in ((128, 256) if p.head else (0,)), (m, n, k, p)
        assert p.splits == 1 or not p.head, (m, n, k, p)
        if p.splits > 1:
            tiles = -(-m // p.bm) * -(-n // p.bn)
            assert p.bn > 0 and p.splits <= 16 and tiles * p.splits <= 256, (m, n, k, p)
            assert p.k_split % 128 == 0 and (p.splits - 1) * p.k_split < k <= p.splits * p.k_split, (m, n, k, p)


def test_the_library_has_these_plans(plans):
    from ltx_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("libltx_hip.so not built")
    sizes = list(_sizes(5000, seed=1))
    for (m, n, k), p in zip(sizes, plans(sizes)):
        assert _lib.lib().ltx_gemm_i8_workspace_bytes(m, n, k) == (4 * m * n * p.splits if p.splits > 1 else 0)


def test_the_gpu_tests_reach_every_kernel(plans):
    import test_gpu_int8
    import test_gpu_int8_plan as tests

    taken = set().union(*map(_kernels, plans(_sizes(200000, seed=2))))
    tested = set()
    for name, sizes in (("two", tests.TWO_LAUNCHES), ("ranges", tests.RANGES), ("one", tests.ONE_LAUNCH)):
        for size, p in zip(sizes, plans(sizes)):
            assert (p.head > 0) == (name == "two") and (p.splits > 1) == (name == "ranges"), (size, p)
            tested |= _kernels(p)
    tested |= set().union(*map(_kernels, plans(test_gpu_int8.SHAPES)))
    assert taken <= tested, sorted(taken - tested)
