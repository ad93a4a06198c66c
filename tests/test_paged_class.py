"""The host's part of PagedKVCache: places without a sequence, lengths that replays have taken too far."""
import pytest
import torch

import trinix_b200 as T


def cache(pages=6, batch=3, **how):
    return T.PagedKVCache(pages, 16, 2, 64, batch, device="cpu", **how)


def in_use(c):
    return (c.block_table >= 0).sum(1).tolist()


def test_an_idle_place_gets_no_pages():
    c = cache()
    c.reserve(20)
    c.release(1, idle=True)
    assert in_use(c) == [2, 0, 2] and c._in_use.tolist() == [1, 0, 1]
    c.reserve(30)  # the pool has pages for two more, not for three
    assert in_use(c) == [2, 0, 2]
    c.reserve(33)
    assert in_use(c) == [3, 0, 3]
    with pytest.raises(RuntimeError, match="pages"):
        c.reserve([0, 1, 0])
    assert c._idle == [False, True, False]
    c.release(0)
    c.reserve([0, 16, 0])
    assert in_use(c) == [0, 1, 3] and c._idle == [False] * 3 and c._in_use.tolist() == [0, 1, 1]
    c.reserve(1)
    assert in_use(c) == [1, 1, 3]


def test_lengths_behind_the_pages_are_not_taken():
    """Pages handed out for tokens that were never written would show what another sequence has left there."""
    c = cache()
    c.reserve(16)
    c._captured = True
    c.lengths.copy_(torch.tensor([16, 17, 3], dtype=torch.int32))
    for call in (c.sync, lambda: c.reserve(1)):
        with pytest.raises(RuntimeError, match=r"\[1\]"):
            call()
    assert in_use(c) == [1, 1, 1] and c._held == [0, 0, 0]
    c.release(1)
    c.reserve(1)
    assert in_use(c) == [2, 1, 1] and c._held == [16, 0, 3]


def test_release_keeps_what_it_did():
    c = cache()
    c.reserve(16)
    c.release(-1)
    assert in_use(c) == [1, 1, 0]
    c.reserve(16)
    assert in_use(c) == [1, 1, 1]
    with pytest.raises(IndexError):
        c.release(3)
