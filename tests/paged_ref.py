"""A paged cache by its definition, in 64 bits, and how far attention over 4-bit codes may be off it."""
from __future__ import annotations

import torch

FIFTEENTH = 0.06666667014360428  # 1 / 15 in 32 bits


def make_cache(lengths, heads, size, dim, bits, dtype, dev, seed=0, spare=3):
    """Pages of random values in random order; a dict of the cache's tensors by argument name."""
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-n // size) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device=dev).int()
    table = torch.full((len(lengths), max(need + [1])), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    c = {"block_table": table}
    for x in "kv":
        if bits == 16:
            c[x + "_pages"] = torch.randn(total, heads, size, dim, generator=g, device=dev).to(dtype)
        else:
            c[x + "_pages"] = torch.randint(0, 256, (total, heads, size, dim // 2), generator=g, device=dev,
                                            dtype=torch.uint8)
            step = 0.1 + 0.4 * torch.rand(total, heads, size, generator=g, device=dev)
            low = -step * (6.0 + 3.0 * torch.rand(total, heads, size, generator=g, device=dev))
            c[x + "_scales"] = torch.stack((step, low), dim=-1)
    return c


def scales_of(c):
    return {n: c[n] for n in ("k_scales", "v_scales") if n in c}


def codes_of(pages):
    return torch.stack((pages & 15, pages >> 4), dim=-1).flatten(-2)


def rows_of(c, x, b, n):
    """The first n rows of sequence b: (values, steps, lowest), (n, heads, dim) and (n, heads, 1) in 64 bits;
    pages outside the cache are zeros."""
    pages = c[x + "_pages"]
    size = pages.shape[2]
    table = c["block_table"][b].long()
    out, steps, lows = [], [], []
    for p in range(n):
        page = int(table[p // size]) if p // size < len(table) else -1
        there = 0 <= page < pages.shape[0]
        row = pages[page if there else 0, :, p % size]
        if x + "_scales" in c:
            s = c[x + "_scales"][page if there else 0, :, p % size].double()
            step, low = s[:, :1], s[:, 1:]
            row = low + codes_of(row).double() * step
        else:
            row, step, low = row.double(), row[:, :1].double() * 0, row[:, :1].double() * 0
        zero = 1.0 if there else 0.0
        out.append(row * zero if there else torch.zeros_like(row))
        steps.append(step if there else torch.zeros_like(step))
        lows.append(low if there else torch.zeros_like(low))
    if not out:
        heads = pages.shape[1]
        dim = pages.shape[3] * (2 if x + "_scales" in c else 1)
        empty = lambda d: torch.zeros(0, heads, d, dtype=torch.float64, device=pages.device)  # noqa: E731
        return empty(dim), empty(1), empty(1)
    return torch.stack(out), torch.stack(steps), torch.stack(lows)


def attend_codes(q, k, v, *, window=None, slopes=None, scale=None):
    """q (Sq, Hq, D); k, v: rows_of, (Sk, Hk, D). As ragged_ref.attend64, for codes:

      * the output is rounded once: u |out|, u the half step of its type;
      * a weight is p * step_v, rounded to 11 bits (2^-11) before it meets the codes: 2^-11 sum p step_v code, that
        is sum p |v - lowest|; one below 2^-14 of the row's largest to 2^-25 of that: 15 Sk 2^-25 max p step_v;
      * w, the relative error of a weight: D additions of the products q * code in the matrix unit's fp32, which
        may cut instead of round, 2 D 2^-24 step_k sum |q| code scale; the term of lowest_k, D 2^-24 of it; three
        fp32 roundings of the score, the bias and the maximum; log2 and the reciprocal of step_v, 2^-22
        (|log2 step_v| + 2); exp2 and the sums, 2^-21. Weights and their sum: 2 w sum p (|v - lowest| + |lowest|).
    """
    (kv, ks, kl), (vv, vs, vl) = k, v
    sq, hq, d = q.shape
    sk, hk, _ = kv.shape
    dev, half = q.device, torch.finfo(q.dtype).eps / 2
    scale = d ** -0.5 if scale is None else scale
    wide = lambda t: t.transpose(0, 1).repeat_interleave(hq // hk, 0)  # noqa: E731
    kv, ks, kl, vv, vs, vl = (wide(t) for t in (kv, ks, kl, vv, vs, vl))
    qq = q.double().transpose(0, 1)
    p = torch.arange(sq, device=dev)[:, None] + (sk - sq)
    j = torch.arange(sk, device=dev)[None]
    s = qq @ kv.transpose(1, 2) * scale
    spread = (kv - kl).abs()
    size = (2 * qq.abs() @ spread.transpose(1, 2) + qq.abs().sum(-1, keepdim=True) * kl.abs().transpose(1, 2)) * abs(scale)
    bias = torch.zeros(hq, sq, sk, dtype=torch.float64, device=dev)
    if slopes is not None:
        bias = slopes.double().view(-1, 1, 1) * (p - j).abs()
    s = s - bias
    hidden = j > p
    if window is not None:
        hidden = hidden | (j < p - window[0])
    s = s.masked_fill(hidden, float("-inf"))
    lse = torch.logsumexp(s, -1) if sk else torch.full((hq, sq), float("-inf"), dtype=torch.float64, device=dev)
    w = torch.exp(s - lse[..., None]).masked_fill(hidden, 0.0)
    w = torch.where(torch.isfinite(lse)[..., None], w, torch.zeros_like(w))
    out = (w @ vv).transpose(0, 1)
    codes = (w @ (vv - vl).abs()).transpose(0, 1)
    low = (w @ vl.abs()).transpose(0, 1)
    heavy = lambda t: (t * (w > 2 ** -30)).amax(-1) if sk else torch.zeros_like(lse)  # noqa: E731
    log_step = vs.clamp(min=2.0 ** -80).log2().abs().transpose(1, 2).expand(hq, sq, sk)
    rel = d * 2.0 ** -24 * heavy(size) + 3 * 2.0 ** -24 * (
        2 * heavy(size) + 2 * heavy(bias) + heavy(log_step) + lse.abs().masked_fill(~torch.isfinite(lse), 0.0)
    ) + 2.0 ** -22 * (heavy(log_step) + 4) + 2.0 ** -21
    rel = rel.t()[..., None]
    allowed = half * out.abs() * 1.001 + 2.0 ** -11 * codes * 1.001 + 2 * rel * (codes + low)
    if sk:
        allowed = allowed + 15 * sk * 2.0 ** -25 * (w * vs.transpose(1, 2)).amax(-1).t()[..., None]
    rel = rel[..., 0].t()
    return out, lse, allowed, 2 * rel + 2.0 ** -22 * lse.abs().masked_fill(~torch.isfinite(lse), 0.0)
