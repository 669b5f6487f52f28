"""The forms (kernels, cuts) that the feed-forward block's plan chooses, and that the sizes of
tests/test_gpu_dense_plans.py reach all of them. No GPU needed: the plan is computed on the host."""
import ctypes
import math
import os
import random

import pytest

from tests.test_gpu_dense_plans import PLAN_SIZES

PRODUCTS = ("gate/up", "down", "gradient of gate/up", "dx", "gate/up weights", "down weight")
TILES = {0: "256x256", 1: "128x256", 2: "128x128", 3: "64x128"}


@pytest.fixture(scope="module")
def lib():
    from lazylora_amd import native
    if not os.path.exists(native.LIB_PATH):
        pytest.fail(f"{native.LIB_PATH} is not built: run __graft_entry__.build() first")
    return native._load_library()


def forms(lib, M, D, F, Do):
    """The forms of the six products of a step."""
    out, plan = set(), (ctypes.c_int * 6)()
    for i, product in enumerate(PRODUCTS):
        assert lib.mxfp4_ffn_plan(i, M, D, F, Do, plan) == 0
        kinds = []
        for rows, tile, runs in (plan[:3], plan[3:]):
            if rows and tile < 0:  # few rows: one or two blocks of weight rows, one to four of x
                out.add((product, f"few rows, {-tile} x {(rows + 15) // 16} blocks"))
                kinds.append("few rows")
            elif rows:
                kinds.append("runs" if runs > 1 else "one run")
                out.add((product, f"{TILES[tile]}, {kinds[-1]}"))
        if len(kinds) == 2:
            out.add((product, f"cut, the last rows: {kinds[1]}"))
    return out


def test_the_gpu_test_reaches_every_form(lib):
    reached = set().union(*(forms(lib, *s) for s in PLAN_SIZES))
    rng = random.Random(11)
    log = lambda lo, hi: max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    missed = {}
    for _ in range(40000):  # the rarest form known comes up in one of 2300 draws
        size = (log(1, 16384), *(8 * log(1, 1024) for _ in range(3)))
        for form in forms(lib, *size) - reached:
            missed.setdefault(form, size)
    assert not missed, "; ".join(f"{' '.join(f)} e.g. at {s}" for f, s in sorted(missed.items()))
    assert len(reached) >= 74  # nothing that was reached has left the plan unnoticed


def test_a_plan_covers_its_rows(lib):
    plan = (ctypes.c_int * 6)()
    for M, D, F, Do in PLAN_SIZES:
        for i, rows in enumerate((M, M, M, M, 2 * F, Do)):
            assert lib.mxfp4_ffn_plan(i, M, D, F, Do, plan) == 0
            assert plan[0] + plan[3] == rows and plan[0] > 0 and plan[2] >= 1
    assert lib.mxfp4_ffn_plan(0, 0, 8, 8, 8, plan) == 0 and not any(plan)


def test_plan_refusals(lib):
    plan = (ctypes.c_int * 6)()
    for args in ((-1, 4, 8, 8, 8), (6, 4, 8, 8, 8), (0, -1, 8, 8, 8), (0, 4, 12, 8, 8), (0, (1 << 24) + 1, 8, 8, 8),
                 (0, 4, 8, (1 << 20) + 8, 8)):
        assert lib.mxfp4_ffn_plan(*args, plan) == -1, args
    assert lib.mxfp4_ffn_plan(0, 4, 8, 8, 8, None) == -1
