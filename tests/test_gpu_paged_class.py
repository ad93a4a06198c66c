"""PagedKVCache between captured steps, released places and the attention modules."""
import pytest
import torch

import trinix_b200 as T

pytestmark = pytest.mark.gpu
HQ, HK, D = 8, 2, 64


def tokens(cuda, *shape, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return [torch.randn(*shape, h, D, generator=g, device=cuda).bfloat16() for h in (HQ, HK, HK)]


def captured(step):
    """A graph of step(), and what it returned."""
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_pieces_behind_pages_reserved_later(cuda, bits):
    """Steps long enough for the packed kernel, replayed when the sequences have more pages, and other ones, than at the
    capture: the same as eager steps."""
    a, b = (T.PagedKVCache(20, 16, HK, D, 2, bits=bits) for _ in range(2))
    q, k, v = tokens(cuda, 2, 40)

    def step(c):
        c.append(k, v)
        return c.attend(q)

    step(T.PagedKVCache(20, 16, HK, D, 2, bits=bits))
    b.reserve(64)
    graph, out = captured(lambda: step(b))
    for i in range(5):
        if i == 1:
            b.reserve(80)
        if i == 2:
            for c in (a, b):
                c.release(0)
                c.reserve([120, 80])
        for t, s in zip((q, k, v), tokens(cuda, 2, 40, seed=i)):
            t.copy_(s)
        if i == 4:
            for c in (a, b):
                c.release(1)
                c.reserve([0, 100])
        graph.replay()
        want = step(a)
        assert torch.equal(a.lengths, b.lengths)
        assert torch.equal(out, want), i
    assert T.attention_status(cuda) == 0
