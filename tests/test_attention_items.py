"""How an attention kernel's CTAs come by their work items (trinix_b200/csrc/attention_issue.cuh), run on the host
against grids whose blocks are handed out in any order: cluster launch control promises none."""
from __future__ import annotations

import ctypes
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "trinix_b200", "csrc")
WRONG = ["", "an item was lost", "an item was taken twice", "a request behind a refusal",
         "the wrong answer was the last one", "giving up"]


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    lib = str(tmp_path_factory.mktemp("model") / "items.so")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-Wno-unknown-pragmas",
                           "-I", CSRC, "-o", lib, os.path.join(HERE, "attention_items_model.cpp")])
    return ctypes.CDLL(lib).items_model


# where the blocks without rows are: behind the last item (a launch that counts items), or anywhere (slots)
@pytest.mark.parametrize("spare", ["behind", "anywhere", "none", "all"])
@pytest.mark.parametrize("ordered", [True, False])
@pytest.mark.parametrize("give_up", [False, True])
def test_every_item_is_taken(model, spare, ordered, give_up):
    rng = random.Random(spare)
    for seed in range(1500):
        n = rng.choice([1, 2, 7, 30, 100])
        held = rng.randint(0, n)
        rows = {"behind": [i < held for i in range(n)], "anywhere": [rng.random() < 0.6 for _ in range(n)],
                "none": [True] * n, "all": [False] * n}[spare]
        resident = rng.choice([1, 2, 8, 40])
        stop = rng.randrange(n + 1) if give_up else -1
        wrong = model(n, bytes(rows), resident, int(ordered), stop, ctypes.c_uint64(seed))
        assert wrong == 0, (WRONG[wrong], rows, resident, stop, seed)
