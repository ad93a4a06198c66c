"""Both issuing warps of an attention kernel together (trinix_b200/csrc/attention_issue.cuh), run on the host:
items whose two Q tiles take the same K and V tiles, and items whose tiles take every second one each."""
from __future__ import annotations

import ctypes
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "trinix_b200", "csrc")
WRONG = ["", "a barrier was lapped", "a stage was overwritten", "a stage was released twice",
         "wrong order", "deadlock", "unfinished"]


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    lib = str(tmp_path_factory.mktemp("model") / "issue_pair.so")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-Wno-unknown-pragmas",
                           "-I", CSRC, "-o", lib, os.path.join(HERE, "attention_issue_pair_model.cpp")])
    return ctypes.CDLL(lib).issue_pair_model


def _item(rng, kind):
    """(visits, first and end of Q tile 0's and of Q tile 1's, mask): as the items of a launch have them."""
    if kind == "any":
        kind = rng.choice(["same", "ragged", "alternate", "odd", "empty"])
    n = rng.choice([1, 2, 3, 4, 5, 9])
    if kind == "same":
        return n, 0, n, 0, n, 0
    if kind == "ragged":  # a causal order: one tile sees less at either end, or nothing
        a, b = rng.choice([(0, n), (0, max(1, n - 1)), (min(1, n - 1), n), (0, 0)]), (0, n)
        return (n, *a, *b, 0) if rng.random() < 0.5 else (n, *b, *a, 0)
    if kind == "empty":
        return 0, 0, 0, 0, 0, 0
    if kind == "alternate":  # two heads: as many visits each
        return 2 * n, 0, 2 * n - 1, 1, 2 * n, 1
    # the keys of one head: as many or one less for the second tile, and none of a single one
    last = [t + 2 * ((n - t + 1) // 2 - 1) + 1 if n > t else 0 for t in (0, 1)]
    return n, 0, last[0], 1 if n > 1 else 0, last[1], 1


@pytest.mark.parametrize("kinds", [["same"], ["ragged"], ["alternate"], ["odd"], ["any"],
                                   ["alternate", "empty"], ["odd", "ragged"]], ids="-".join)
def test_issue_order_of_both(model, kinds):
    rng = random.Random(len(kinds[0]))
    for seed in range(2500):
        items = [_item(rng, rng.choice(kinds)) for _ in range(rng.randint(1, 5))]
        cols = [(ctypes.c_int * len(items))(*c) for c in zip(*items)]
        wrong = model(len(items), *cols, ctypes.c_uint64(seed))
        assert wrong == 0, (WRONG[wrong], items, seed)
