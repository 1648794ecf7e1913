"""The ring of the few-token layer's streaming kernels, from the header that the launcher itself uses (compiled here with the host
compiler): every stage has room for what any job of a call can put into it, and the ring for all stages.

A job is up to 32 slots of one expert. A token may name an expert more than once, so a call of T tokens with k slots each can
have jobs of up to min(32, T k) slots, whatever T is."""
import ctypes
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "scattermoe_b200", "csrc")
SHIM = r"""
#include "few_token_stages.h"
using namespace smoe::ft;
extern "C" int stages(int up, int ring, int box_bytes, int blocks, int T, int k, int turns, int* out) {
  Stages s;
  if (!make_stages(&s, up != 0, ring, box_bytes, blocks, T, k, turns)) return 0;
  *out++ = s.stages;
  *out++ = s.stage_bytes;
  for (int c = 0; c < 4; ++c)
    for (int g = 0; g < STAGE_GROUPS; ++g) *out++ = s.steps_of[c][g];
  return 1;
}
extern "C" int class_of(int boxes) { return width_class(boxes); }
extern "C" int slack() { return RING_SLACK; }
"""
GRID, MOST_SMEM = 148, 232448
PLAN, BARRIERS, MAX_R, CONSUMERS, TILE = 8208, (2 * 16 + 2) * 8, 1024, 8, 32


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    gxx = shutil.which("g++")
    assert gxx, "the host compiler that nvcc needs as well"
    at = tmp_path_factory.mktemp("stages")
    (at / "shim.cpp").write_text(SHIM)
    subprocess.run([gxx, "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(at / "shim.cpp"), "-o", str(at / "shim.so")], check=True)
    return ctypes.CDLL(str(at / "shim.so"))


def ceil(a, b):
    return -(-a // b)


def launch(up, k_major, K, d_out, T):
    """(bytes for the ring, bytes of a box, boxes a stage can be wide) as the launcher derives them."""
    rows = min(ceil(d_out, GRID), TILE) if k_major else 2 * TILE
    sums = MAX_R * 4 + (CONSUMERS * 32 * 32 * 4 if up else (CONSUMERS // 2 if rows > 16 else CONSUMERS) * T * (rows + 1) * 4)
    box_rows = (TILE if up else rows) if k_major else 2 * TILE
    widths = range(1, (CONSUMERS if k_major else CONSUMERS // 2) + 1) if up else [1]
    return MOST_SMEM - (PLAN + MAX_R + BARRIERS + sums + 1024 + 64), ceil(box_rows, 8) * 1024, widths


@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("k_major", [True, False])
def test_every_job_fits_its_stage(lib, up, k_major):
    turns = 2 if up else 4
    for T, k in [(1, 1), (1, 2), (1, 8), (1, 32), (2, 4), (2, 16), (4, 8), (7, 2), (8, 1), (8, 2), (8, 8), (9, 1), (9, 4), (16, 2), (16, 8), (24, 1),
                 (24, 8), (31, 1), (31, 4), (32, 1), (40, 2), (64, 2), (64, 16), (127, 8), (128, 1), (128, 8)]:
        for K in (8, 64, 72, 128, 192, 256, 320, 512, 768, 1024, 1536, 2880, 4096, 14336):
            for d_out in (8, 64, 152, 1000, 1184, 1192, 2048, 2368, 2880, 4096, 4736, 5120, 7168):
                ring, box, widths = launch(up, k_major, K, d_out, T)
                blocks = ceil(K, 64)
                out = (ctypes.c_int * 18)()
                what = dict(up=up, k_major=k_major, T=T, k=k, K=K, d_out=d_out)
                assert lib.stages(int(up), ring, box, blocks, T, k, turns, out), what
                stages, stage_bytes, steps_of = out[0], out[1], [out[2 + 4 * c:6 + 4 * c] for c in range(4)]
                assert turns <= stages <= 16 and stages % turns == 0 and stage_bytes % 1024 == 0, what
                assert stages * stage_bytes + lib.slack() <= ring, what
                for boxes in widths:
                    for groups in range(1, min(4, ceil(T * k, 8)) + 1):
                        steps = steps_of[lib.class_of(boxes)][groups - 1]
                        need = steps * (boxes * box + groups * 1024)
                        assert steps >= 1 and need <= stage_bytes, (what, boxes, groups, steps, need, stage_bytes)


def test_slots_of_few_tokens_on_one_expert(lib):
    """The smallest case by hand: 8 tokens x 8 slots, all on one expert, F = d_out = 64. A box of one output column's rows is 1 KB, 32
    slots' rows are 4 KB."""
    out = (ctypes.c_int * 18)()
    ring, box, _ = launch(False, True, 64, 64, 8)
    assert box == 1024 and lib.stages(0, ring, box, 1, 8, 8, 4, out)
    assert out[1] >= 1024 + 4 * 1024 and out[2 + 3] == 1


@pytest.mark.parametrize("k_major", [True, False])
def test_long_sums(lib, k_major):
    """The whole of K as bytes passes 32 bits long before K reaches its limit of 2^28: the stages are those of any other long K."""
    ring, box, _ = launch(False, k_major, 1 << 20, 64, 24)
    out, long = (ctypes.c_int * 18)(), (ctypes.c_int * 18)()
    assert lib.stages(0, ring, box, (1 << 20) // 64, 24, 2, 4, out)
    for K in ((1 << 25) + 8, 1 << 26, (1 << 27) + 64, (1 << 28) - 8):
        assert lib.stages(0, ring, box, ceil(K, 64), 24, 2, 4, long)
        assert list(long[:2]) == list(out[:2]), K
