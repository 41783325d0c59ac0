"""Which tiles the cross entropy's plan (csrc/vocab.h) takes at the sizes of the GPU tests: every kind of every product is among them, so that other
figures in its rules cannot take one out of the tests unseen.  ``plan_loss`` is compiled for the host; no GPU needed."""
import os
import shutil
import subprocess

import pytest

import test_vocab_gpu

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moda_amd", "csrc")
PROGRAM = """
#include <cstdio>
#include "vocab.h"
int main() {
  long long n, vocab, width;
  int fp32;
  while (scanf("%lld %lld %lld %d", &n, &vocab, &width, &fp32) == 4) {
    const bool grid = width % 8 == 0;
    const moda::LossPlan f = moda::plan_loss(n, vocab, width, fp32, grid, grid, false, true, true, true);
    const moda::LossPlan b = moda::plan_loss(n, vocab, width, fp32, grid, grid, true, true, true, true);
    printf("%d %d %d %d %d %d %d\\n", f.direct, f.logits.tile, b.logits.tile, b.grad_rows.tile, b.acc_rows, b.grad_weight.tile, b.grad_weight.splits > 1);
  }
}
"""
LARGE, MEDIUM, ROWS, SMALL = range(4)


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    if shutil.which("hipcc") is None:
        pytest.skip("hipcc not found")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.hip").write_text(PROGRAM)
    subprocess.run(["hipcc", "-x", "hip", "--cuda-host-only", "-std=c++17", "-I", CSRC, str(d / "plan.hip"), "-o", str(d / "plan")], check=True,
                   stdout=subprocess.PIPE, stderr=subprocess.PIPE)

    def run(sizes, fp32):
        text = "".join(f"{n} {v} {c} {int(fp32)}\n" for n, v, c in sizes)
        out = subprocess.run([str(d / "plan")], input=text, check=True, stdout=subprocess.PIPE, text=True).stdout
        return [tuple(int(x) for x in line.split()) for line in out.splitlines()]

    return run


@pytest.mark.parametrize("fp32", [False, True])
def test_every_tile_is_tested(plans, fp32):
    taken = plans(test_vocab_gpu.TILES, fp32)
    assert len(taken) == len(test_vocab_gpu.TILES)
    tiles = (LARGE, MEDIUM, ROWS, SMALL)
    assert {(p[0], p[1]) for p in taken} >= {(direct, tile) for direct in ((0,) if fp32 else (0, 1)) for tile in tiles}  # logits, rows in place or not
    assert {p[2] for p in taken} >= set(tiles)                                                                          # their gradient
    assert {(p[3], p[4]) for p in taken} >= {(tile, sums) for tile in tiles for sums in (0, 1)}                         # the rows'
    assert {(p[5], p[6]) for p in taken} >= {(tile, split) for tile in (LARGE, MEDIUM, SMALL) for split in (0, 1)}      # the weight's


def test_rows_in_place_are_few(plans):
    assert [p[0] for p in plans([(1, 50, 64), (512, 50, 64), (513, 50, 64), (512, 50, 65)], False)] == [1, 1, 0, 0]
    assert [p[0] for p in plans([(1, 50, 64)], True)] == [0]
