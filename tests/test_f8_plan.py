"""Which tile shape an 8-bit product takes: plan_for of csrc/f8_mm.cu, compiled
on the host as it stands.  The GPU tests that are there to reach every shape
have to go on reaching them when the rule changes."""
import os
import subprocess

import pytest

pytest.importorskip("torch")
import test_f8  # noqa: E402
import test_f8_scales  # noqa: E402
from test_f8_roles import SOURCE, between  # noqa: E402

MAIN = r"""
#include <stdint.h>
#include <stdio.h>
struct MmArgs { const void *offsets; int n_rows, n_experts, out, blocks_c; };
constexpr int kTileM = 128;
#include "plan.inc"
int main() {
    int rows, out, blocks, experts, sms;
    while (scanf("%d %d %d %d %d", &rows, &out, &blocks, &experts, &sms) == 5) {
        MmArgs a{experts ? &rows : nullptr, rows, experts ? experts : 1, out, blocks};
        const Plan p = plan_for(a, sms);
        printf("%d %d %d %lld\n", p.bn, p.pair, p.split, (long long)most_tiles(a, kTileM * p.pair, p.bn));
    }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.inc").write_text(between(open(SOURCE).read(), "int64_t most_tiles(", "template <int BN, int PAIR, bool SPLIT = false>"))
    (d / "main.cpp").write_text(MAIN)
    exe = str(d / "plan")
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", exe, str(d / "main.cpp")], check=True)

    def of(sizes, sms=148):
        """(columns of a tile, CTAs, parts, most tiles) for each (rows, outputs, contraction, experts)."""
        given = "".join(f"{r} {o} {-(-i // 128)} {e} {sms}\n" for r, o, i, e in sizes)
        said = subprocess.run([exe], input=given, capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in said.splitlines()]
    return of


def shapes(plans):
    return {p[:3] for p in plans}


def test_the_tests_reach_every_tile_shape(plans):
    every = {(128, 1, 1), (256, 1, 1), (256, 2, 1), (128, 1, 2), (128, 1, 4), (128, 1, 8)}
    alone = [s for s in test_f8.SHAPES_OF_TILES if not s[3]]
    grouped = [s for s in test_f8.SHAPES_OF_TILES if s[3]]
    assert shapes(plans(alone)) == every
    assert {(128, 1, 1), (256, 1, 1), (256, 2, 1)} < shapes(plans(grouped)) and any(p[2] > 1 for p in plans(grouped))
    of_scales = shapes(plans(test_f8_scales.SIZES))
    assert {(128, 1, 1), (256, 1, 1), (256, 2, 1)} < of_scales and any(p[2] > 1 for p in of_scales)


@pytest.mark.parametrize("sms", [148, 132, 64, 2, 1])
def test_a_shared_contraction_has_a_cluster_for_every_tile(plans, sms):
    """Its sums lie in the ring, so a cluster takes one tile only; and every part has a block."""
    sizes = [(r, o, i, e) for r in (1, 2, 100, 128, 129, 700, 5000) for o in (1, 128, 129, 1000, 4096) for i in (1, 128, 512, 2049, 14336)
             for e in (0, 1, 3, 64) if e == 0 or o * e <= 1 << 20]
    said = plans(sizes, sms)
    assert len(said) == len(sizes)
    for (rows, out, inner, experts), (bn, pair, split, tiles) in zip(sizes, said):
        if split > 1:
            assert (bn, pair) == (128, 1) and tiles * split <= sms and -(-inner // 128) >= split
