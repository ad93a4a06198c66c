"""The attention module over a paged cache, and with rotation and q / k norm as one kernel."""
import pytest
import torch

import trinix_b200 as T
from trinix_b200.decoder import params_to_bf16

pytestmark = pytest.mark.gpu
E, HQ, HK, D = 512, 8, 2, 64


def module(cuda, seed=0, **how):
    torch.manual_seed(seed)
    kw = dict(kernel_type="triton", causal=True, position_method="rope", head_dim=D, max_seq_len=256, tile_kv=False)
    m = T.FastGroupedQueryAttention(E, HQ, HK, **{**kw, **how}).to(cuda)
    if m.qk_norm:
        for norm in (m.q_norm, m.k_norm):
            norm.weight.data += 0.1 * torch.randn(D, device=cuda)
            if hasattr(norm, "bias"):
                norm.bias.data += 0.1 * torch.randn(D, device=cuda)
    return m


@pytest.mark.parametrize("norm", ["rmsnorm", "layernorm"])
def test_fused_qk_against_the_modules_of_it(cuda, norm):
    """In fp32 up to the attention's own type, so that both compute the same: forward of q and k, and gradients."""
    plain, fused = module(cuda, qk_norm=True, qk_norm_type=norm), module(cuda, qk_norm=True, qk_norm_type=norm, fused_qk=True)
    fused.load_state_dict(plain.state_dict())
    g = torch.Generator(device=cuda).manual_seed(0)
    q, k = (torch.randn(2, 40, h, D, generator=g, device=cuda) for h in (HQ, HK))
    grads = []
    for m, way in ((plain, "plain"), (fused, "fused")):
        a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
        if way == "plain":
            cos, sin = m.position_embedding(a, 40)
            x, y = m.position_embedding._apply_rope_pytorch(a, b, cos, sin)
            x, y = m.q_norm._pytorch_forward(x), m.k_norm._pytorch_forward(y)
        else:
            x, y = m._norm_and_rotate(a, b)
        (x.square().sum() + (y * torch.arange(D, device=cuda)).sum()).backward()
        params = [p for n in (m.q_norm, m.k_norm) for p in n.parameters()]
        grads.append([x, y, a.grad, b.grad, *(p.grad for p in params)])
    for x, y in zip(*grads):
        # fp32 both, sums of up to 640 terms: 640 roundings of 2^-24 of the largest, at most
        assert float((x - y).detach().abs().max()) <= 640 * 2.0 ** -24 * float(y.detach().abs().max())


def test_fused_qk_in_a_forward_and_backward_pass(cuda):
    """bf16, through the projections; the fused way has fewer roundings, so the two are compared as 16-bit results:
    three roundings of q and k (projection, rotation, norm) of 2^-9 to 2^-8 each change a score by less than 5 % of its
    size of some units, and an output, a mean of values, by less than a tenth of its largest."""
    a, b = (params_to_bf16(module(cuda, qk_norm=True, fused_qk=f)) for f in (False, True))
    b.load_state_dict(a.state_dict())
    x = torch.randn(2, 100, E, device=cuda).bfloat16()
    with torch.no_grad():
        y, z = a(x)[0], b(x)[0]
    assert float((y - z).abs().max()) <= 0.1 * float(y.abs().max())
    ids = torch.arange(100, device=cuda).expand(2, 100)
    with torch.no_grad():
        assert torch.equal(b(x, position_ids=ids)[0], z)
    assert a.extra_repr() == b.extra_repr()


@pytest.mark.parametrize("how", [dict(), dict(qk_norm=True), dict(qk_norm=True, qk_norm_type="layernorm"),
                                 dict(position_method="alibi"), dict(position_method="none", qk_norm=True),
                                 dict(use_sliding_window=True, sliding_window_size=20)], ids=str)
@pytest.mark.parametrize("bits", [16, 4])
def test_module_over_a_paged_cache(cuda, how, bits):
    """A prompt, a piece and single tokens through the cache against the whole sequence at once. 16 bits: the same
    values but for the order of roundings, as 16-bit results (see above). 4 bits: keys and values are off by half of a
    step, a 30th of their row's range, each; the output, a mean of values, by less than half of its largest."""
    m = params_to_bf16(module(cuda, fused_qk=True, **how))
    B, lengths = 3, [50, 7, 1, 1, 1]
    x = torch.randn(B, sum(lengths), E, device=cuda).bfloat16()
    cache = T.PagedKVCache(24, 16, HK, D, B, bits=bits, max_pages=8)
    got, at = [], 0
    with torch.no_grad():
        want = m(x)[0]
        for n in lengths:
            y, present = m(x[:, at:at + n], past_key_value=cache)
            assert present is cache
            got.append(y)
            at += n
    got = torch.cat(got, dim=1)
    assert cache.lengths.tolist() == [sum(lengths)] * B
    off = float((got - want).abs().max()) / float(want.abs().max())
    assert off <= (0.1 if bits == 16 else 0.5), off
    assert T.attention_status(cuda) == 0


@pytest.mark.parametrize("how", [dict(), dict(qk_norm=True)], ids=str)
def test_sequences_longer_than_the_module_was_told(cuda, how):
    """Positions go as far as the cache does."""
    a, b = (params_to_bf16(module(cuda, max_seq_len=n, **how)) for n in (256, 16))
    b.load_state_dict(a.state_dict())
    x = torch.randn(1, 40, E, device=cuda).bfloat16()
    with torch.no_grad():
        out = [[m(x[:, i:i + 8], past_key_value=c)[0] for i in range(0, 40, 8)]
               for m, c in ((a, T.PagedKVCache(4, 16, HK, D)), (b, T.PagedKVCache(4, 16, HK, D)))]
    assert all(torch.equal(y, z) for y, z in zip(*out)) and all(y.isfinite().all() for y in out[0])


def test_steps_as_a_graph(cuda):
    """Steps captured and replayed do what they do one by one."""
    m = params_to_bf16(module(cuda, qk_norm=True, fused_qk=True))
    x = torch.randn(2, 12, E, device=cuda).bfloat16()
    caches = [T.PagedKVCache(12, 16, HK, D, 2, bits=4) for _ in range(2)]
    tok = torch.zeros(2, 1, E, device=cuda).bfloat16()
    with torch.no_grad():
        for c in caches:
            m(x[:, :9], past_key_value=c)
        eager = [m(x[:, i:i + 1], past_key_value=caches[0])[0] for i in (9, 10, 11)]
        c = caches[1]
        c.reserve(8)
        saved = [t.clone() for t in (c.k_pages, c.v_pages, c.k_scales, c.v_scales, c.lengths)]
        m(tok, past_key_value=c)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(tok, past_key_value=c)[0]
        for t, s in zip((c.k_pages, c.v_pages, c.k_scales, c.v_scales, c.lengths), saved):
            t.copy_(s)
        for i, want in zip((9, 10, 11), eager):
            tok.copy_(x[:, i:i + 1])
            graph.replay()
            assert torch.equal(out, want)
        c.sync()
        assert c.lengths.tolist() == [12, 12] and c.gather()[0].shape[0] == 24
        # a piece long enough for the packed kernel, behind what the replays appended
        x = torch.randn(2, 40, E, device=cuda).bfloat16()
        for other in caches:
            other.lengths.fill_(12)
            other.sync()
        assert torch.equal(*(m(x, past_key_value=other)[0] for other in caches))


def test_pages_are_handed_out_and_taken_back(cuda):
    c = T.PagedKVCache(5, 16, HK, D, 3, max_pages=3)
    kv = torch.randn(3, 16, HK, D, device=cuda).bfloat16()
    c.append(kv, kv)
    assert "free=2" in repr(c) and c.lengths.tolist() == [16] * 3
    with pytest.raises(RuntimeError, match="pages"):
        c.append(kv[:, :1], kv[:, :1])
    assert c.lengths.tolist() == [16] * 3
    c.release(1)
    assert c.lengths.tolist() == [16, 0, 16] and "free=3" in repr(c)
    c.append(kv[:, :1], kv[:, :1])
    pages = [p for p in c.block_table.flatten().tolist() if p >= 0]
    assert len(pages) == len(set(pages)) == 5
    k, v = c.gather()
    assert k.shape == (17 + 1 + 17, HK, D)
    assert torch.equal(k[:16], kv[0]) and torch.equal(v[17], kv[1, 0]) and torch.equal(k[18:34], kv[2])


def test_refusals(cuda):
    c = T.PagedKVCache(4, 16, HK, D)
    m = params_to_bf16(module(cuda))
    x = torch.randn(1, 2, E, device=cuda).bfloat16()
    with pytest.raises(RuntimeError, match="no_grad"):
        m(x, past_key_value=c)
    with torch.no_grad():
        with pytest.raises(ValueError, match="mask"):
            m(x, attention_mask=torch.zeros(2, 2, device=cuda), past_key_value=c)
        with pytest.raises(ValueError, match="place"):
            m(x, position_ids=torch.zeros(1, 2, dtype=torch.int64, device=cuda), past_key_value=c)
        with pytest.raises(ValueError, match="causal"):
            params_to_bf16(module(cuda, causal=False))(x, past_key_value=c)
        with pytest.raises(ValueError, match="expected k"):
            m(x.expand(2, 2, E), past_key_value=c)
    assert c.lengths.tolist() == [0]


def test_steps_behind_replays(cuda):
    """A capture appends nothing; behind its replays, which the host does not see, steps find pages of their own."""
    m = params_to_bf16(module(cuda))
    x = torch.randn(1, 40, E, device=cuda).bfloat16()
    tok = x[:, :1].clone()
    a, b = (T.PagedKVCache(6, 16, HK, D) for _ in range(2))
    with torch.no_grad():
        m(tok, past_key_value=T.PagedKVCache(6, 16, HK, D))
        b.reserve(16)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(tok, past_key_value=b)[0]
        assert b.lengths.tolist() == [0]
        for i in range(16):
            tok.copy_(x[:, i:i + 1])
            graph.replay()
            assert torch.equal(out, m(x[:, i:i + 1], past_key_value=a)[0])
        for c in (a, b):
            for i in range(16, 20):
                y = m(x[:, i:i + 1], past_key_value=c)[0]
            c.last = y
    assert torch.equal(a.last, b.last) and b.lengths.tolist() == [20]
    assert all(torch.equal(s, t) for s, t in zip(a.gather(), b.gather()))


def test_a_captured_step_without_room_is_refused(cuda):
    m = params_to_bf16(module(cuda))
    tok = torch.randn(1, 1, E, device=cuda).bfloat16()
    c = T.PagedKVCache(1, 16, HK, D)
    with torch.no_grad():
        m(tok, past_key_value=T.PagedKVCache(1, 16, HK, D))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="reserve"):
                m(tok, past_key_value=c)
        assert c.lengths.tolist() == [0]
        m(tok, past_key_value=c)
    assert c.lengths.tolist() == [1]


def test_evaluated_then_trained(cuda):
    """Tables made in inference mode serve a training step."""
    m = params_to_bf16(module(cuda, qk_norm=True, fused_qk=True))
    q, k = (torch.randn(1, 4, h, D, device=cuda).bfloat16() for h in (HQ, HK))
    with torch.inference_mode():
        want = m._norm_and_rotate(q, k)
    a, b = m._norm_and_rotate(q.requires_grad_(), k.requires_grad_())
    (a.float().sum() + b.float().sum()).backward()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and q.grad.isfinite().all()


def test_generating(cuda):
    """A prompt through the packed kernel, then a token, into 4 bits; the lines of the README."""
    x = torch.randn(4, 501, 1024, device=cuda).bfloat16()
    attn = T.FastGroupedQueryAttention(1024, 8, 2, kernel_type="triton", causal=True,
                                       position_method="rope").to(cuda).bfloat16()
    cache = T.PagedKVCache(64, 64, 2, 128, batch_size=4, bits=4)
    with torch.no_grad():
        y, _ = attn(x[:4, :500], past_key_value=cache)
        z, _ = attn(x[:4, 500:501], past_key_value=cache)
    assert y.shape == (4, 500, 1024) and z.shape == (4, 1, 1024) and bool(y.isfinite().all() and z.isfinite().all())
    assert cache.lengths.tolist() == [501] * 4
