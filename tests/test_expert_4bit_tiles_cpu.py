"""CPU tests of how the 4-bit product is cut into tiles: a program of a few lines is compiled with the
kernels' own header and prints what the host side chooses (nvcc needs no GPU)."""
import os
import subprocess

import pytest

from efficient_linear_assignment_b200 import build as b200_build

PROGRAM = r"""
#include <cstdio>
#include "ela_expert_mma.cuh"
using namespace ela_expert;
int main() {
    int widest[5] = {}, fewest = 99;
    const int64_t few[] = {9, 13, 40, 128, 129, 500, 4000};
    for (int64_t E = 1; E <= ELA_EXPERT_MAX; ++E)
        for (int64_t share : few)
            for (int64_t F : {40, 264, 4096})
                for (int64_t K : {64, 1000}) {
                    const MmaParams p = row_pass(nullptr, E * share, E, F, K, true);
                    if (p.stages < fewest) fewest = p.stages;
                    if (p.ring % PACK_TURNS || p.ring > PACK_MAX_RING || p.stages > MMA_MAX_STAGES || p.bn % 32 || p.bn < 32 || p.bn > 256) return 2;
                    // the stages, the ring and the experts' tables fit, from a stage's boundary on
                    const int64_t bytes = 12 * E + 1023 + (int64_t)p.stages * 2 * (MMA_A_BYTES + p.bn / 2 * MMA_KB * 2) + p.ring * PACK_BLOCK;
                    if (bytes > MMA_SMEM - 1024) return 3;
                    int& w = widest[E <= 512 ? 0 : E <= 1536 ? 1 : E <= 2560 ? 2 : E <= 3584 ? 3 : 4];
                    if (p.bn > w) w = p.bn;
                }
    std::printf("%d", fewest);
    for (int w : widest) std::printf(" %d", w);
    return 0;
}
"""


@pytest.fixture(scope="module")
def chosen(tmp_path_factory):
    where = tmp_path_factory.mktemp("tiles")
    src, exe = where / "tiles.cu", where / "tiles"
    src.write_text(PROGRAM)
    subprocess.run([b200_build.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr", "-I", b200_build.INCLUDE,
                    "-I", b200_build.CSRC, "-o", str(exe), str(src)], check=True, env={**os.environ, "TMPDIR": str(where)})
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out
    return [int(v) for v in out.stdout.split()]


def test_every_group_of_unpacking_warps_has_a_stage(chosen):
    """The three groups take every third stage by a barrier's parity, which two stages do not tell apart."""
    assert chosen[0] >= 3


def test_tiles_are_as_wide_as_the_experts_tables_allow(chosen):
    assert chosen[1:] == [256, 224, 192, 160, 128]  # up to 512, 1536, 2560, 3584 and 4096 experts
