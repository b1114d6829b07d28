"""How dense products are divided among clusters of blocks: the host's rules, compiled by themselves (no GPU, no CUDA)."""
import ctypes as C
import itertools
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "denno_beta_b200", "csrc")
SOURCE = """
#include "dense_plan.h"
extern "C" void pairs(const int* at_once, int tiles, int chunks, int* out) {
    int a[5];
    for (int i = 0; i < 5; ++i) a[i] = at_once[i];
    const dnb::PairPlan p = dnb::pair_plan(a, tiles, chunks);
    out[0] = p.parts; out[1] = p.whole; out[2] = p.pairs; out[3] = p.each; out[4] = p.more;
}
extern "C" int splits(const int* at_once, int sms, int stage, int tiles, int chunks) {
    int a[9];
    for (int i = 0; i < 9; ++i) a[i] = at_once[i];
    return dnb::best_splits(a, sms, stage, tiles, chunks);
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I" + CSRC, str(d / "plan.cpp"), "-o", str(d / "plan.so")])
    return C.CDLL(str(d / "plan.so"))


def pairs(plan, at_once, tiles, chunks):
    out = (C.c_int * 5)()
    plan.pairs((C.c_int * 5)(*at_once), tiles, chunks, out)
    return dict(zip(("parts", "whole", "pairs", "each", "more"), out))


WHOLE = [0, 74, 35, 22, 16]  # a device like a B200: GPCs leave some SMs over
COUNTS = [WHOLE, [0, 70, 33, 21, 14], [0, 74, 35, 22, 0], [0, 74, 0, 0, 0], [0, 74, 35, 0, 16], [0, 74, 0, 22, 16], [0, 1, 0, 0, 0], [0, 1, 1, 1, 1]]


@pytest.mark.parametrize("at_once", COUNTS)
def test_every_tile_belongs_to_one_place_that_exists(plan, at_once):
    for tiles, chunks in itertools.product([*range(1, 160), 296, 297, 1000, 4099], [1, 2, 3, 4, 16, 40, 64, 176]):
        p = pairs(plan, at_once, tiles, chunks)
        parts, clusters = p["parts"], p["pairs"] // p["parts"]
        assert at_once[parts] > 0 and clusters * parts == p["pairs"] and 1 <= clusters <= at_once[parts]
        shared = range(p["whole"], min(tiles, p["whole"] + clusters))
        owned = [first + i * p["pairs"] for first in range(p["pairs"]) for i in range(p["each"] + (first < p["more"]))]
        assert sorted([*owned, *shared]) == list(range(tiles))
        assert not shared or (parts > 1 and chunks >= parts)


def test_clusters_that_a_device_does_not_hold_are_not_used(plan):
    # one tile of a long sum: four pairs if there is such a cluster, fewer if there is not, one pair if no other is known
    assert pairs(plan, WHOLE, 1, 176)["parts"] == 4
    assert pairs(plan, [0, 74, 35, 22, 0], 1, 176)["parts"] == 3
    assert pairs(plan, [0, 74, 35, 0, 0], 1, 176)["parts"] == 2
    assert pairs(plan, [0, 74, 0, 0, 0], 1, 176) == dict(parts=1, whole=1, pairs=1, each=1, more=0)
    blocks = [0, 148, 66, 44, 33, 26, 22, 18, 15]
    held = lambda *none: (C.c_int * 9)(*(0 if s in none else n for s, n in enumerate(blocks)))  # noqa: E731
    assert plan.splits(held(), 148, 20480, 4, 64) == 8
    assert plan.splits(held(8), 148, 20480, 4, 64) < 8
    assert plan.splits(held(*range(2, 9)), 148, 20480, 4, 64) == 1
    for tiles, chunks, none in itertools.product([1, 17, 80, 500], [1, 3, 8, 16, 48], itertools.combinations(range(2, 9), 3)):
        s = plan.splits(held(*none), 148, 20480, tiles, chunks)
        assert 1 <= s <= min(8, chunks) and s not in none


def test_sizes_that_are_tested_take_the_paths_they_are_for(plan):
    """On any device with about a B200's clusters, whatever a change of the rules makes of them."""
    import dense_sizes as sizes

    for (nt, k, n), columns in [*((s, 256) for s in sizes.SPLIT_PRODUCTS), *((s, 128) for s in sizes.SPLIT_GATED)]:
        tiles = -(-nt // 256) * -(-n // columns)
        for at_once in ([0, *c] for c in itertools.product((70, 72, 74), (33, 35, 37), (20, 22, 24), (14, 16, 18))):
            p = pairs(plan, at_once, tiles, -(-k // 256))
            assert p["parts"] > 1 and p["whole"] < tiles and (p["whole"] > 0) == (tiles >= 74)
    for gated, listed in ((0, sizes.SEVERAL_A_BLOCK_PRODUCTS), (1, sizes.SEVERAL_A_BLOCK_GATED)):
        for nt, k, n in listed:
            tiles, per_sm, rows = -(-n // 128), 2 if nt <= 64 else 1, next(r for r in (16, 32, 64, 128) if nt <= r)
            assert tiles > 148 * per_sm
            stage16 = (1 + gated) * 16384 + rows * 128
            for stage, chunks in ((stage16 + (2 + gated) * 1024, -(-k // 256)), (stage16, -(-k // 64))):  # 4 bits, 16 bits
                held = [0, 148 * per_sm, *((148 * per_sm - 8) // s for s in range(2, 9))]
                assert plan.splits((C.c_int * 9)(*held), 148, stage, tiles, chunks) == 1
