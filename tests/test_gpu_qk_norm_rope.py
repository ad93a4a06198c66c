"""Norms of queries and keys with the rotation in the same pass, forward and backward, against the definition in
64 bits.

Tolerances: the result is rounded once (half a step of its type); before that everything is fp32, where an error
of a few 2^-24 relative to the values that enter grows, in the norm, by max|x| * rstd (the mean of a LayerNorm is
taken from values that may be near each other). K counts those roundings: one per element for the products and
sums of the norm, the affine part and the rotation (about 16), the shuffles of a sum (up to 6) and its terms in a
thread (up to 32), the latter relative to a mean of them.
"""
import pytest
import torch

import trinix_b200 as T

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
K = 64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tables(rows, dim, device, dtype=torch.float32):
    rate = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * rate
    return angle.cos().to(device, dtype), angle.sin().to(device, dtype)


def rotate(x, c, s):
    h = x.shape[-1] // 2
    x1, x2 = x[..., :h], x[..., h:]
    c, s = c[..., :h], s[..., :h]
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)


def stats(x, eps, norm):
    if norm == "layernorm":
        x = x - x.mean(-1, keepdim=True)
    rstd = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return x * rstd, rstd


def definition(x, w, b, c, s, eps, norm, first):
    """y of one of the two, all in 64 bits; c, s (B | 1, S, 1, D/2)."""
    z = x if first else rotate(x, c, s)
    a = stats(z, eps, norm)[0] * w
    if b is not None:
        a = a + b
    return rotate(a, c, s) if first else a


def angles(cos, sin, S, positions):
    if positions is None:
        return cos.double()[None, :S, None], sin.double()[None, :S, None]
    p = positions.long().reshape(-1, S)
    return cos.double()[p][:, :, None], sin.double()[p][:, :, None]


def check_forward(y, x, w, b, c, s, eps, norm, first):
    x, w, b = x.double(), w.double(), None if b is None else b.double()
    ref = definition(x, w, b, c, s, eps, norm, first)
    n, rstd = stats(x if first else rotate(x, c, s), eps, norm)
    grown = x.abs().amax(-1, keepdim=True) * rstd + n.abs().amax(-1, keepdim=True)
    size = w.abs().max() * grown + (b.abs().max() if b is not None else 0.0)
    assert y.shape == x.shape
    tol = half_step(y.dtype) * ref.abs() + K * F32 * size + torch.finfo(y.dtype).tiny
    bad = (y.double() - ref).abs() > tol * 1.001
    assert not bad.any(), float(((y.double() - ref).abs() / tol).max())


def check_backward(got, dy, x, w, b, c, s, eps, norm, first):
    """got: dx, dw, db (or None)."""
    leaves = [t.double().detach().requires_grad_() for t in (x, w) + ((b,) if b is not None else ())]
    xx, ww, bb = (leaves + [None])[:3]
    grads = torch.autograd.grad(definition(xx, ww, bb, c, s, eps, norm, first), leaves, dy.double())
    xd, wd, g = x.double(), w.double(), dy.double()
    if first:
        g = rotate(g, c, -s)
    n, rstd = stats(xd if first else rotate(xd, c, s), eps, norm)
    grown = 1 + xd.abs().amax(-1, keepdim=True) * rstd + n.abs().amax(-1, keepdim=True)
    big = g.abs().amax(-1, keepdim=True)
    size = rstd * big * wd.abs().max() * (1 + n.abs().amax(-1, keepdim=True)) * grown
    tol = half_step(x.dtype) * grads[0].abs() + 2 * K * F32 * size + torch.finfo(x.dtype).tiny
    err = (got[0].double() - grads[0]).abs()
    assert not (err > tol * 1.001).any(), float((err / tol).max())
    # a thread adds up to some hundred terms one after the other, then 2 * 592 partial sums are added 37 to a thread
    terms = ((g.abs() * n.abs() + big * F32) * grown).sum((0, 1, 2)), g.abs().sum((0, 1, 2))
    for i in range(len(leaves) - 1):
        tol = half_step(w.dtype) * grads[i + 1].abs() + 8 * K * F32 * terms[i] + torch.finfo(w.dtype).tiny
        err = (got[i + 1].double() - grads[i + 1]).abs()
        assert not (err > tol * 1.001).any(), float((err / tol).max())


def make(B, S, Hq, Hk, D, dtype, cuda, norm, seed=0, w_dtype=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    q, k = (r(B, S, h, D).to(cuda, dtype) for h in (Hq, Hk))
    w = [(1 + 0.2 * r(D)).to(cuda, w_dtype or dtype) for _ in range(2)]
    b = [(0.3 * r(D)).to(cuda, w_dtype or dtype) if norm == "layernorm" else None for _ in range(2)]
    return q, k, w, b


CASES = [  # B, S, Hq, Hk, D
    (1, 1, 1, 1, 64), (2, 3, 5, 1, 128), (3, 17, 12, 4, 80), (1, 33, 9, 3, 96), (2, 5, 3, 3, 2), (2, 9, 4, 2, 6),
    (1, 7, 2, 1, 130), (2, 6, 8, 2, 256), (1, 4, 2, 2, 510), (1, 5, 3, 1, 512), (1, 700, 16, 2, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("norm", ["rmsnorm", "layernorm"])
@pytest.mark.parametrize("first", [True, False], ids=["first", "last"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_backward(cuda, case, first, norm, dtype):
    B, S, Hq, Hk, D = case
    eps = 1e-5 if norm == "layernorm" else 1e-6
    q, k, w, b = make(B, S, Hq, Hk, D, dtype, cuda, norm)
    cos, sin = tables(S + 3, D, cuda)
    how = dict(eps=eps, norm=norm, norm_first=first)
    y = T.qk_norm_rope(q, k, *w, cos, sin, q_bias=b[0], k_bias=b[1], **how)
    c, s = angles(cos, sin, S, None)
    for i, x in enumerate((q, k)):
        assert y[i].dtype == dtype and y[i].is_contiguous()
        check_forward(y[i], x, w[i], b[i], c, s, eps, norm, first)
    dy = [torch.randn(*x.shape, generator=torch.Generator().manual_seed(3)).to(cuda, dtype) for x in (q, k)]
    got = T.qk_norm_rope_backward(*dy, q, k, *w, cos, sin, need_db=norm == "layernorm", **how)
    again = T.qk_norm_rope_backward(*dy, q, k, *w, cos, sin, need_db=norm == "layernorm", **how)
    for x, z in zip(got, again):
        assert x is None and z is None or torch.equal(x, z)
    for i, x in enumerate((q, k)):
        check_backward(got[i::2], dy[i], x, w[i], b[i], c, s, eps, norm, first)


@pytest.mark.parametrize("first", [True, False], ids=["first", "last"])
@pytest.mark.parametrize("kind", ["per_token", "shared", "int32", "strided", "expanded"])
def test_positions(cuda, kind, first):
    B, S, D = 3, 11, 128
    q, k, w, _ = make(B, S, 4, 2, D, torch.bfloat16, cuda, "rmsnorm")
    cos, sin = tables(500, D, cuda)
    g = torch.Generator().manual_seed(1)
    pos = torch.randint(0, 500, (B, S), generator=g).to(cuda)
    if kind == "shared":
        pos = pos[0]
    elif kind == "int32":
        pos = pos.int()
    elif kind == "strided":
        pos = torch.randint(0, 500, (S, B, 2), generator=g).to(cuda)[..., 1].t()
    elif kind == "expanded":
        pos = pos[:1].expand(B, S)
    y = T.qk_norm_rope(q, k, *w, cos, sin, positions=pos, norm_first=first)
    dy = [torch.randn_like(t) for t in (q, k)]
    got = T.qk_norm_rope_backward(*dy, q, k, *w, cos, sin, positions=pos, norm_first=first)
    c, s = angles(cos, sin, S, pos)
    for i, x in enumerate((q, k)):
        check_forward(y[i], x, w[i], None, c, s, 1e-6, "rmsnorm", first)
        check_backward(got[i:4:2], dy[i], x, w[i], None, c, s, 1e-6, "rmsnorm", first)


def test_positions_outside_the_tables_are_nan(cuda):
    q, k, w, _ = make(2, 4, 3, 1, 80, torch.float16, cuda, "rmsnorm")
    cos, sin = tables(6, 80, cuda)
    pos = torch.tensor([[0, -1, 5, 6], [2, 3, 2 ** 40, -2 ** 40]], device=cuda)
    bad = ((pos < 0) | (pos > 5))[:, :, None, None]
    for first in (True, False):
        for x, y in zip((q, k), T.qk_norm_rope(q, k, *w, cos, sin, positions=pos, norm_first=first)):
            assert torch.equal(y.isnan(), bad.expand_as(x))


@pytest.mark.parametrize("D", [128, 80, 66])
def test_strides_tables_and_weights(cuda, D):
    """Views of one projection, transposed and expanded inputs, tables of the activation's type or wider ones,
    weights of another type."""
    B, S, Hq, Hk = 2, 19, 6, 2
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(B, S, (Hq + 2 * Hk) * D + 1, generator=g).to(cuda, torch.bfloat16)
    _, _, w, _ = make(1, 1, 1, 1, D, torch.bfloat16, cuda, "rmsnorm", w_dtype=torch.float32)
    cos, sin = tables(S, D, cuda, torch.bfloat16)
    wide = [torch.cat((t, t), dim=-1)[:, : D - 2] for t in tables(S, D, cuda)]
    one = qkv[..., :-1].view(B, S, -1, D)
    odd = qkv[..., 1:].view(B, S, -1, D)  # rows that start between two 16-byte boundaries
    heads = torch.randn(B, Hq, S, D, generator=g).to(cuda, torch.bfloat16).transpose(1, 2)
    for q, k in ((one[:, :, :Hq], one[:, :, Hq:Hq + Hk]), (odd[:, :, :Hq], odd[:, :, Hq:Hq + Hk]),
                 (heads, heads[:, :, :1].expand(B, S, Hk, D))):
        for c0, s0 in ((cos, sin), wide):
            y = T.qk_norm_rope(q, k, *w, c0, s0)
            dy = [torch.ones(1, 1, 1, D, device=cuda, dtype=q.dtype).expand_as(t) for t in (q, k)]
            got = T.qk_norm_rope_backward(*dy, q, k, *w, c0, s0)
            c, s = angles(c0, s0, S, None)
            c, s = c[..., : D // 2], s[..., : D // 2]
            for i, x in enumerate((q, k)):
                check_forward(y[i], x, w[i], None, c, s, 1e-6, "rmsnorm", True)
                check_backward(got[i:4:2], dy[i], x, w[i], None, c, s, 1e-6, "rmsnorm", True)


@pytest.mark.parametrize("norm", ["rmsnorm", "layernorm"])
@pytest.mark.parametrize("first", [True, False], ids=["first", "last"])
def test_gradient_against_differences(cuda, first, norm):
    """dx in a random direction against the difference of the definition, in 64 bits, at both sides: its own
    error is of the order h^2, the gradient's 2 K 2^-24 of its terms."""
    B, S, Hq, Hk, D, h = 1, 5, 3, 2, 16, 1e-4
    q, k, w, b = make(B, S, Hq, Hk, D, torch.float32, cuda, norm, seed=5)
    cos, sin = tables(S, D, cuda)
    c, s = angles(cos, sin, S, None)
    dy = [torch.randn_like(t) for t in (q, k)]
    got = T.qk_norm_rope_backward(*dy, q, k, *w, cos, sin, eps=1e-5, norm=norm, norm_first=first,
                                  need_db=norm == "layernorm")
    for i, x in enumerate((q, k)):
        for j, leaf in enumerate((x, w[i], b[i])):
            if leaf is None:
                continue
            v = torch.randn_like(leaf).double()
            at = lambda t: definition(*[(z.double() + t * v if n == j else z.double()) if z is not None else None  # noqa: E731,E501
                                        for n, z in enumerate((x, w[i], b[i]))], c, s, 1e-5, norm, first)
            change = ((at(h) - at(-h)) * dy[i].double()).sum() / (2 * h)
            terms = got[i + 2 * j].double() * v
            assert abs(float(terms.sum() - change)) <= 2 * K * F32 * 16 * float(terms.abs().sum()) + 1e-5


def test_rows_of_zeros_infinities_and_nan(cuda):
    """A row of zeros gives 0 (rstd is finite by eps); what is not finite stays in its own row."""
    q, k, w, _ = make(2, 8, 4, 2, 128, torch.bfloat16, cuda, "rmsnorm")
    cos, sin = tables(8, 128, cuda)
    clean = T.qk_norm_rope(q, k, *w, cos, sin)
    q[0, 1, 2] = 0
    q[1, 3, 0, 5] = float("nan")
    k[0, 2, 1, 7] = float("inf")
    y = T.qk_norm_rope(q, k, *w, cos, sin)
    assert not y[0][0, 1, 2].any()
    assert y[0][1, 3, 0].isnan().all() and not y[1][0, 2, 1].isfinite().all()
    for new, old, rows in ((y[0], clean[0], [(0, 1, 2), (1, 3, 0)]), (y[1], clean[1], [(0, 2, 1)])):
        for r in rows:
            new[r], old[r] = 0, 0
        assert torch.equal(new, old)


def test_nothing_to_do(cuda):
    cos, sin = tables(4, 64, cuda)
    w = torch.ones(64, device=cuda)
    for shape_q, shape_k in (((0, 4, 2, 64), (0, 4, 1, 64)), ((2, 0, 2, 64), (2, 0, 1, 64)),
                             ((2, 4, 2, 64), (2, 4, 0, 64)), ((2, 4, 0, 64), (2, 4, 3, 64))):
        q, k = torch.randn(shape_q, device=cuda), torch.randn(shape_k, device=cuda)
        y = T.qk_norm_rope(q, k, w, w, cos, sin)
        assert y[0].shape == q.shape and y[1].shape == k.shape
        got = T.qk_norm_rope_backward(q, k, q, k, w, w, cos, sin)
        for x, d, dw in ((q, got[0], got[2]), (k, got[1], got[3])):
            assert d.shape == x.shape and dw.shape == (64,)
            if x.numel() == 0:
                assert not dw.any()


def test_autograd(cuda):
    """Through the kernel class: gradients of every leaf, of shared heads and of broadcast inputs, with one of the
    two outputs unused, and accumulated over two passes."""
    B, S, Hq, Hk, D = 2, 6, 4, 2, 64
    q, k, w, b = make(B, S, Hq, Hk, D, torch.float32, cuda, "layernorm")
    cos, sin = tables(S, D, cuda)
    shared = torch.randn(1, 1, Hk, D, device=cuda, requires_grad=True)
    leaves = [t.clone().requires_grad_() for t in (q, *w, *b)]
    out = T.QKNormRoPEKernel.apply(leaves[0], shared.expand(B, S, Hk, D), leaves[1], leaves[2], cos, sin, leaves[3],
                                   leaves[4], 1e-5, "layernorm", False)
    c, s = angles(cos, sin, S, None)
    ref_leaves = [t.detach().double().requires_grad_() for t in (leaves[0], shared, *leaves[1:])]
    rq, rk, rw, rw2, rb, rb2 = ref_leaves
    ref = (definition(rq, rw, rb, c, s, 1e-5, "layernorm", False),
           definition(rk.expand(B, S, Hk, D), rw2, rb2, c, s, 1e-5, "layernorm", False))
    dy = [torch.randn_like(t) for t in out]
    for o, r, d in zip(out, ref, dy):
        (o * d).sum().backward(retain_graph=True)
        (r * d.double()).sum().backward(retain_graph=True)
    # fp32 sums of B * S * heads terms of order 1 .. 10, each off by 2 K 2^-24 of its size at most
    for got, want in zip((leaves[0], shared, *leaves[1:]), ref_leaves):
        assert got.grad.shape == want.grad.shape
        assert float((got.grad - want.grad).abs().max()) <= 2 * K * F32 * 10 * B * S * Hq


def test_weights_alone_need_gradients(cuda):
    q, k, w, _ = make(1, 4, 2, 2, 64, torch.bfloat16, cuda, "rmsnorm")
    cos, sin = tables(4, 64, cuda)
    kw = w[1].float().view(1, 64).requires_grad_()  # of another dtype and shape than the queries'
    y = T.QKNormRoPEKernel.apply(q, k, w[0], kw, cos, sin)
    y[1].float().sum().backward()
    assert kw.grad.shape == kw.shape and kw.grad.dtype == torch.float32 and kw.grad.isfinite().all()


def test_other_stream_and_captured(cuda):
    """On a stream of its own, and captured while an eager graph of the same leaves lives: replays follow the
    leaves' memory."""
    q, k, w, _ = make(2, 32, 8, 2, 128, torch.bfloat16, cuda, "rmsnorm")
    cos, sin = tables(32, 128, cuda)
    side = torch.cuda.Stream(cuda)
    want = T.qk_norm_rope(q, k, *w, cos, sin)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = T.qk_norm_rope(q, k, *w, cos, sin)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    dy = [torch.randn_like(t) for t in (q, k)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = (*T.qk_norm_rope(q, k, *w, cos, sin), *T.qk_norm_rope_backward(*dy, q, k, *w, cos, sin)[:4])
    for seed in (1, 2):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        now = (*T.qk_norm_rope(q, k, *w, cos, sin), *T.qk_norm_rope_backward(*dy, q, k, *w, cos, sin)[:4])
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(static, now))


@pytest.mark.parametrize("change,error", [
    (dict(norm="batchnorm"), "norm"), (dict(q_bias=True), "biases"), (dict(k=(2, 4, 2, 64)), "match"),
    (dict(k=(2, 5, 1, 128)), "match"), (dict(rows=3), "positions"), (dict(weight=127), "elements"),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), "positions"),
    (dict(positions=torch.zeros(4)), "int32"), (dict(columns=60), "tables"), (dict(q=(2, 4, 3, 7)), "head_dim"),
    (dict(q=(2, 4, 3, 514)), "head_dim"),
], ids=str)
def test_refusals(cuda, change, error):
    a = dict(q=(2, 4, 3, 128), k=None, rows=4, columns=64, weight=None, norm="rmsnorm", q_bias=None, positions=None)
    a.update(change)
    q = torch.zeros(a["q"], device=cuda)
    k = torch.zeros(a["k"] or (2, 4, 1, a["q"][3]), device=cuda)
    D = a["q"][3]
    w = torch.ones(a["weight"] or D, device=cuda)
    t = torch.zeros(a["rows"], max(a["columns"], D // 2) if D > 128 else a["columns"], device=cuda)
    pos = a["positions"].to(cuda) if a["positions"] is not None else None
    with pytest.raises((ValueError, TypeError), match=error):
        T.qk_norm_rope(q, k, w, w, t, t, norm=a["norm"], q_bias=w if a["q_bias"] else None, positions=pos)
