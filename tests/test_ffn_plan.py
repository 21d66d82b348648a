"""CPU: the rule that gives a feed-forward block's products their tile (csrc/ffn_plan.h, plain C++, built
here with g++): what it may choose, and that the sizes of the GPU tests take all of it."""
from __future__ import annotations

import ctypes as C
import subprocess

import pytest

from tests.conftest import ROOT
from tests.test_gpu_block import TILE_SHAPES

HARNESS = r"""
#include "see-ai_amd/csrc/ffn_plan.h"
using namespace seeai::ffn;
extern "C" {
// Up to three products of rows m[i] by columns n[i]; out: tile, tiles, whole, splits, stages a split.
void choose(int f32, int dual, int count, const size_t* m, const size_t* n, size_t K, int nseg, int* out) {
  const Plan p = count == 1 ? Choose(f32, dual, {{m[0], n[0]}}, K, nseg)
                            : Choose(f32, dual, {{m[0], n[0]}, {m[1], n[1]}, {m[2], n[2]}}, K, nseg);
  out[0] = p.tile, out[1] = p.tiles, out[2] = p.whole, out[3] = p.splits, out[4] = p.per_split;
}
size_t part_limit() { return kMostPart; }
int deep(int f32) { return Deep(f32); }
int rows(int f32, int dual, int tile) { return ShapeOf(f32, tile).bm(dual); }
int cols(int f32, int dual, int tile) { return ShapeOf(f32, tile).bn(dual); }
}
"""
TILES = {0: 3, 1: 2}  # of bf16, f32


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    d = tmp_path_factory.mktemp("ffn_plan")
    src, lib = d / "h.cc", d / "h.so"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-I{ROOT}", str(src), "-o", str(lib)], check=True)
    h = C.CDLL(str(lib))
    h.part_limit.restype = C.c_size_t
    return h


def products(M, D, F):
    """Name, whether two products run side by side, the outputs, K and segments of a block's launches."""
    return [("gate", 1, [(M, F)], D, 1), ("down", 0, [(M, D)], F, 1), ("grad", 0, [(M, F)], D, 1),
            ("dx", 0, [(M, D)], F, 2), ("dw", 0, [(D, F), (D, F), (F, D)], M, 1)]


def choose(rule, f32, dual, outs, K, nseg):
    m = (C.c_size_t * 3)(*[o[0] for o in outs])
    n = (C.c_size_t * 3)(*[o[1] for o in outs])
    out = (C.c_int * 5)()
    rule.choose(f32, dual, len(outs), m, n, C.c_size_t(K), nseg, out)
    return list(out)


@pytest.mark.parametrize("f32", [0, 1])
def test_plans_cover_their_products(rule, f32):
    """Every tile is counted, every stage of K lies in one split, no split is empty, and the shared
    sums stay within their limit."""
    sizes = (1, 63, 65, 200, 777, 1024, 2050, 4100, 8192)
    for M in sizes:
        for D in sizes:
            for F in sizes:
                for name, dual, outs, K, nseg in products(M, D, F):
                    tile, tiles, whole, splits, per = choose(rule, f32, dual, outs, K, nseg)
                    bm, bn = rule.rows(f32, dual, tile), rule.cols(f32, dual, tile)
                    assert tiles == sum(-(-m // bm) * -(-n // bn) for m, n in outs)
                    stages = -(-K // rule.deep(f32)) * nseg
                    assert 0 <= whole <= tiles and splits >= 1
                    if whole < tiles:
                        assert splits > 1 and (splits - 1) * per < stages <= splits * per
                        part = (tiles - whole) * splits * bm * bn * (8 if dual else 4)
                        assert part <= rule.part_limit()


def test_the_gpu_tests_sizes_take_every_tile_and_sharing(rule):
    """Each launch on each tile the rule gives it, over several stages of K, and each with K whole,
    shared out by all tiles, or by the tiles past whole rounds; ragged edges on the largest."""
    for f32 in (0, 1):
        tiles, shares, ragged = set(), set(), set()
        for M, D, F in TILE_SHAPES:
            for name, dual, outs, K, nseg in products(M, D, F):
                tile, n, whole, splits, per = choose(rule, f32, dual, outs, K, nseg)
                stages = -(-K // rule.deep(f32)) * nseg
                if min(stages, per) < 3:
                    continue
                tiles.add((name, tile))
                shares.add((name, "whole" if whole == n else "mixed" if whole else "shared"))
                bm, bn = rule.rows(f32, dual, tile), rule.cols(f32, dual, tile)
                if any(m % bm and c % bn and c % 8 for m, c in outs):
                    ragged.add((name, tile))
        names = [p[0] for p in products(1, 1, 1)]
        assert shares >= {(n, s) for n in names for s in ("whole", "mixed")} | {(n, "shared") for n in ("down", "dx")}
        want = {(n, t) for n in names for t in range(TILES[f32])}
        missing = want - tiles
        assert not missing, missing
        assert {(n, 0) for n in names} <= ragged, ragged
