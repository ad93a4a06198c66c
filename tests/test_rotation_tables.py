"""Rotation tables of the attention modules: what a model of many of them keeps."""
import copy
import gc

import torch

import trinix_b200 as T
from trinix_b200 import layers

CPU = torch.device("cpu")


def test_modules_share_their_tables():
    """One pair for all modules of a base and dim, as long as one of them lives."""
    a, b, other = T.FastRoPEPositionEmbedding(32, 24), T.FastRoPEPositionEmbedding(32, 24), T.FastRoPEPositionEmbedding(32, 24, base=500.0)
    pairs = [m.tables(100, CPU, half=True) for m in (a, b, other)]
    assert pairs[0] is pairs[1] and pairs[2][0] is not pairs[0][0]
    assert not torch.equal(pairs[0][0], pairs[2][0])
    ours = lambda: [k for k in layers._rotation_tables.keys() if k[0] == 32]  # noqa: E731
    assert len(ours()) == 2
    del a
    gc.collect()
    assert b.tables(128, CPU, half=True) is pairs[0]
    del b, other, pairs
    gc.collect()
    assert not ours()


def test_half_of_the_columns():
    rope = T.FastRoPEPositionEmbedding(48, 16)
    full, half = rope.tables(40, CPU), rope.tables(40, CPU, half=True)
    assert full[0].shape == (64, 48) and half[0].shape == (64, 24)
    for x, y in zip(full, half):
        assert torch.equal(x[:, :24], y) and torch.equal(x[:, 24:], y)
    assert rope.tables(64, CPU, half=True) is half and rope.tables(64, CPU) is full
    # a module of no other positions than its own: as many as it was told
    assert T.FastRoPEPositionEmbedding(48, 16).tables(3, CPU, half=True)[0].shape == (16, 24)


def test_a_copied_module_has_tables():
    rope = T.FastRoPEPositionEmbedding(40, 16)
    made = rope.tables(16, CPU, half=True)
    again = copy.deepcopy(rope)
    assert all(torch.equal(x, y) for x, y in zip(again.tables(16, CPU, half=True), made))
