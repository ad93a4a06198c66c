"""Attention of one sequence from its definition, in 64 bits, and how far a kernel may be off it."""
from __future__ import annotations

import torch


def attend64(q, k, v, *, causal=False, window=None, slopes=None, scale=None):
    """q (Sq, Hq, D), k / v (Sk, Hk, D): (out, lse (Hq, Sq), allowed, allowed for lse), all but the
    first two elementwise bounds on the error of a 16-bit kernel with fp32 scores and sums.

    Query i stands at key position i + Sk - Sq. Let A = sum_j softmax_j |v_j|, u the half step of the
    type, and w the relative error of one weight exp(s_j - m):
      * the output is rounded once: u |out|; each probability is rounded once before the second
        product, the normaliser is not: u A;
      * w: D fp32 additions in the score, D 2^-24 sum_d |q_d k_d| scale; the scale, the bias and the
        maximum, three fp32 roundings of values up to |s| + |bias| + |m|; exp2 and the fp32 sums, 2^-21.
        Weights and their sum are off by at most w each: 2 w A, and log(1 + w) in the LSE;
      * fp16 probabilities below 2^-14 are subnormal and off by up to 2^-25 each: Sk 2^-25 max|v|, the
        reference maximum being at most the true one and the normaliser so at least 1.
    """
    sq, hq, d = q.shape
    sk, hk, _ = k.shape
    dev, half = q.device, torch.finfo(q.dtype).eps / 2
    scale = d ** -0.5 if scale is None else scale
    qq = q.double().transpose(0, 1)
    kk = k.double().transpose(0, 1).repeat_interleave(hq // hk, 0)
    vv = v.double().transpose(0, 1).repeat_interleave(hq // hk, 0)
    p = torch.arange(sq, device=dev)[:, None] + (sk - sq)
    j = torch.arange(sk, device=dev)[None]
    s = qq @ kk.transpose(1, 2) * scale
    size = (qq.abs() @ kk.abs().transpose(1, 2)) * abs(scale)
    bias = torch.zeros(hq, sq, sk, dtype=torch.float64, device=dev)
    if slopes is not None:
        bias = slopes.double().view(-1, 1, 1) * (p - j).abs()
    s = s - bias
    hidden = torch.zeros(sq, sk, dtype=torch.bool, device=dev)
    if causal:
        hidden |= j > p
    if window is not None:
        hidden |= (j < p - window[0]) | (j > p + window[1])
    s = s.masked_fill(hidden, float("-inf"))
    lse = torch.logsumexp(s, -1) if sk else torch.full((hq, sq), float("-inf"), dtype=torch.float64,
                                                       device=dev)
    w = torch.exp(s - lse[..., None]).masked_fill(hidden, 0.0)
    w = torch.where(torch.isfinite(lse)[..., None], w, torch.zeros_like(w))
    out = (w @ vv).transpose(0, 1)
    a = (w @ vv.abs()).transpose(0, 1)
    seen = ~hidden
    top = lambda t: (t.masked_fill(~seen, 0.0).amax(-1) if sk else  # noqa: E731
                     torch.zeros(hq, sq, dtype=torch.float64, device=dev))
    # the keys that carry weight decide: a bias of thousands belongs to weights of 0
    heavy = lambda t: (t * (w > 2 ** -30)).amax(-1) if sk else torch.zeros_like(lse)  # noqa: E731
    rel = d * 2.0 ** -24 * heavy(size) + 3 * 2.0 ** -24 * (
        2 * top(size) + heavy(bias) + lse.abs().masked_fill(~torch.isfinite(lse), 0.0)) + 2.0 ** -21
    if slopes is not None:  # ramps are counted from a tile's edge: 128 keys more
        rel = rel + 3 * 2.0 ** -24 * (128 * slopes.double().abs().view(-1, 1) + heavy(bias))
    allowed = half * (out.abs() + a) * 1.001 + 2 * rel.t()[..., None] * a
    if q.dtype == torch.float16:
        allowed = allowed + sk * 2.0 ** -25 * (vv.abs().max() if sk else 0.0)
    return out, lse, allowed, 2 * rel + 2.0 ** -22 * lse.abs().masked_fill(~torch.isfinite(lse), 0.0)


def assert_within(got, want, allowed, what=""):
    got = got.double()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite), f"{what}: other values are finite"
    assert torch.equal(got[~finite], want[~finite]), f"{what}: infinities"
    off = (got - want).abs()[finite]
    over = off - allowed[finite]
    if over.numel():
        worst = int(over.argmax())
        assert float(over.max()) <= 0, (
            f"{what}: off by {float(off[worst]):.3e}, allowed {float(allowed[finite][worst]):.3e}, "
            f"{float((over > 0).float().mean()):.2e} of the values beyond it")
