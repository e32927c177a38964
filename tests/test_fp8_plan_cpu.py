"""Which kernel the 8-bit products run on, from the plan itself, compiled for the CPU with 256 compute units: that the GPU tests reach what they are for."""
import os
import shutil
import subprocess

import pytest

from test_gpu_fp8 import SECOND_CODES, SECOND_LINEAR, SECOND_PAIR

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-stu-2_amd", "csrc")
MAIN = """
static int fstu_cus() { return 256; }
#include "fstu_fp8_plan.h"
#include <cstdio>
int main() {
  int M, N, K, f32, glu, codes, slices;
  while (scanf("%d %d %d %d %d %d %d", &M, &N, &K, &f32, &glu, &codes, &slices) == 7) {
    const Plan p = plan(M, N, K, f32, glu, codes, slices);
    printf("%d %d\\n", (int)p.kind, p.slices);
  }
}
"""
SKINNY, TILE, LARGE = range(3)


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no compiler here")
    where = tmp_path_factory.mktemp("plan")
    (where / "plan.cpp").write_text(MAIN)
    subprocess.run([compiler, "-std=c++17", "-O1", "-I", CSRC, str(where / "plan.cpp"), "-o", str(where / "plan")], check=True)

    def ask(cases):
        out = subprocess.run([str(where / "plan")], input="\n".join(" ".join(str(int(v)) for v in c) for c in cases), capture_output=True, text=True, check=True)
        return [tuple(int(v) for v in line.split()) for line in out.stdout.splitlines()]
    return ask


def test_the_tests_of_several_rounds_reach_the_large_tiles(plans):
    for shapes, glu, codes, features in ((SECOND_LINEAR, 0, 0, 256), (SECOND_PAIR, 1, 0, 128), (SECOND_CODES, 1, 1, 128)):
        for (M, N, K), found in zip(shapes, plans([(M, N, K, 0, glu, codes, glu) for M, N, K in shapes])):
            assert found == (LARGE, 1), (M, N, K, glu, codes, found)
            assert -(-M // 256) * -(-N // features) > 256, "one round of tiles"
            assert K % 16 == 0                                         # others take another kernel
    assert any(K % 128 for _, _, K in SECOND_LINEAR) and any(K % 128 for _, _, K in SECOND_PAIR) and any(K % 128 for _, _, K in SECOND_CODES)


def test_every_product_has_a_plan_that_can_run(plans):
    """Slices that the entry point takes, few rows on their own kernel, the pair in one order of sums above 32 rows."""
    cases = [(M, N, K, f32, glu, codes, 0 if not glu else 1) for M in (1, 16, 17, 32, 33, 64, 65, 300, 4096, 100000) for N in (1, 100, 768, 24576) for K in (1, 129, 768, 24576)
             for f32, glu, codes in ((0, 0, 0), (1, 0, 0), (0, 1, 0), (1, 1, 0), (0, 1, 1))]
    for (M, N, K, f32, glu, codes, _), (kind, slices) in zip(cases, plans(cases)):
        assert 1 <= slices <= min(64, -(-K // 128))
        assert not (glu and slices > 1)
        if M <= (32 if glu else 64):
            assert kind == SKINNY
        elif glu:
            assert kind != SKINNY
        if kind == LARGE and not codes:
            assert K % 16 == 0 and not f32
