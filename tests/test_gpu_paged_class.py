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


def step(c, t, S=1):
    q, k, v = (x[:, :S] for x in t)
    c.append(k, v)
    return c.attend(q)


@pytest.mark.parametrize("S", [1, 3, 40])
def test_an_idle_place_takes_no_part(cuda, S):
    """The others' steps are what they were; its own queries see nothing; it costs no pages."""
    a, b = T.PagedKVCache(20, 16, HK, D, 3), T.PagedKVCache(18, 16, HK, D, 2)
    first = tokens(cuda, 3, 20)
    step(a, first, 20)
    step(b, [x[::2] for x in first], 20)
    a.release(1, idle=True)
    for i in range(3):
        t = tokens(cuda, 3, S, seed=i + 1)
        got, want = step(a, t, S), step(b, [x[::2] for x in t], S)
        assert torch.equal(got[::2], want) and not got[1].any()
    assert a.lengths.tolist() == [20 + 3 * S, 0, 20 + 3 * S]
    assert all(torch.equal(x, y) for x, y in zip(a.gather(), b.gather()))
    a.reserve([0, 1, 0])
    assert step(a, first).shape == (3, 1, HQ, D) and a.lengths.tolist()[1] == 1


def test_replays_pass_a_released_place_over(cuda):
    """Its length stays 0, what the next sequence there sees is its own."""
    a, b = (T.PagedKVCache(12, 16, HK, D, 2) for _ in range(2))
    t = tokens(cuda, 2, 1)
    step(T.PagedKVCache(4, 16, HK, D, 2), t)
    b.reserve(40)
    graph, out = captured(lambda: step(b, t))

    def both(seed):
        for x, y in zip(t, tokens(cuda, 2, 1, seed=seed)):
            x.copy_(y)
        graph.replay()
        return step(a, t)

    for i in range(5):
        assert torch.equal(out, both(i))
    for c in (a, b):
        c.release(0, idle=True)
    for i in range(5, 10):
        want = both(i)
        assert torch.equal(out, want) and not out[0].any()
        assert a.lengths.tolist() == b.lengths.tolist() == [0, i + 1]
    for c in (a, b):
        c.reserve([20, 20])
    for i in range(10, 14):
        assert torch.equal(out, both(i))
    assert a.lengths.tolist() == b.lengths.tolist() == [4, 14]
    assert all(torch.equal(x, y) for x, y in zip(a.gather(), b.gather()))


def test_replays_behind_what_was_reserved_are_told(cuda):
    c = T.PagedKVCache(4, 16, HK, D, 1)
    t = tokens(cuda, 1, 1)
    step(T.PagedKVCache(4, 16, HK, D, 1), t)
    c.reserve(16)
    graph, _ = captured(lambda: step(c, t))
    for _ in range(17):
        graph.replay()
    for call in (c.sync, lambda: c.reserve(1), lambda: step(c, t)):
        with pytest.raises(RuntimeError, match="lost"):
            call()
    c.lengths.fill_(16)
    step(c, t)
    assert c.lengths.tolist() == [17]
    assert T.attention_status(cuda) == 0


def test_a_module_with_dropout(cuda):
    """Refused while it trains, with the cache as it was; eval() does what a module without does."""
    torch.manual_seed(0)
    kw = dict(kernel_type="triton", causal=True, position_method="rope", head_dim=D)
    a, b = (T.FastGroupedQueryAttention(512, HQ, HK, dropout=p, **kw).to(cuda).bfloat16() for p in (0.0, 0.25))
    b.load_state_dict(a.state_dict())
    x = torch.randn(1, 3, 512, device=cuda).bfloat16()
    c, other = (T.PagedKVCache(2, 16, HK, D) for _ in range(2))
    with torch.no_grad():
        with pytest.raises(ValueError, match="eval"):
            b(x, past_key_value=c)
        assert c.lengths.tolist() == [0] and not c.k_pages.any()
        assert torch.equal(b.eval()(x, past_key_value=c)[0], a(x, past_key_value=other)[0])


def test_pages_do_not_change_hands_in_a_capture(cuda):
    """Refused, with the host's lists as they were: it would hold pages for given that the table never names."""
    c = T.PagedKVCache(4, 16, HK, D, 1)
    t = tokens(cuda, 1, 1)
    step(c, t)

    def try_all():
        for call in (lambda: c.reserve(30), lambda: c.release(0), c.sync):
            with pytest.raises(RuntimeError, match="capture"):
                call()
        return t[0] + 1

    graph, out = captured(try_all)
    graph.replay()
    assert torch.equal(out, t[0] + 1)
    assert "free=3" in repr(c) and c._tokens == [1] and c.lengths.tolist() == [1]
    c.reserve(30)
    assert (c.block_table >= 0).sum() == 2


def test_long_steps_of_idle_places_alone(cuda):
    c = T.PagedKVCache(4, 16, HK, D, 2)
    for b in range(2):
        c.release(b, idle=True)
    for S in (1, 40):
        assert not step(c, tokens(cuda, 2, S), S).any()
    assert c.lengths.tolist() == [0, 0] and "free=4" in repr(c)
