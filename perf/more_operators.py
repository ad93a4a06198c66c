"""Norms of queries and keys with their rotation, and a paged cache of keys and values in 16 or 4 bits, as
cases that can be timed.

`run` computes a case either in its plain form, with elementary torch operations in 32 bits, or (with
`own`) through the package's public entry points: QKNormRoPEKernel and `qk_norm_rope`, `append_paged`,
`gather_paged` and `attention_paged`. `exact` is the same from the definition, in 64 bits.

A cache of 4 bits holds, for each row of head_dim values, codes of 0 .. 15 (byte j: column 2 j in the low four
bits, 2 j + 1 in the high ones) and two 32-bit numbers, step and lowest: a value is lowest + code * step. The
lowest value has code 0, the highest 15, the others the nearest, of two as near the even one.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
FIFTEENTH = 0.06666667014360428  # 1 / 15 in 32 bits
LEAST_RANGE = 2.0 ** -120        # a row whose values are nearer to each other is held as one value

# Elements of queries and keys of a drawn case: the largest listed one has 42e6, forward and backward.
MOST_NORM = 40_000_000
# Rows of new keys, and of keys in the cache, times kv heads and head dim: the largest listed ones have 17e6 and 69e6.
MOST_NEW, MOST_CACHED = 12_000_000, 60_000_000
# Keys times kv heads and head dim of a drawn attention: the largest listed one has 268e6.
MOST_KEYS = 200_000_000
MOST_SCORES = 300_000_000


def listed():
    return [
        # One decoding step's tokens, each at a position of its own: call and launch latency.
        norm_case(16, 1, 32, 8, 128, "bf16", positions=True, name="norm_tokens"),
        # A training step of a block: forward and backward, all gradients.
        norm_case(4, 2048, 32, 8, 128, "bf16", backward=True, name="norm_train"),
        # The order of the attention modules here, rotation first, with LayerNorm and its biases; odd sizes.
        norm_case(3, 701, 20, 4, 80, "f16", norm="layernorm", first=False, backward=True,
                  name="norm_layernorm"),
        # One decoding step: a token of each sequence into its page, its queries rotated on the way.
        append_case(64, 1, 2048, 32, 8, 128, "bf16", 16, 16, rotate=True, queries=True,
                    name="append_tokens"),
        # The prompts that a server has collected, of very different lengths, packed.
        append_case(16, 2048, 0, 32, 8, 128, "bf16", 16, 64, packed=True, rotate=True, queries=True,
                    name="append_prompts"),
        # The same into a cache of 4 bits, and what attention over the prompts then reads; head dim 64, odd lengths.
        append_case(12, 1501, 0, 16, 4, 64, "f16", 4, 32, packed=True, rotate=True, name="append4_prompts"),
        # A piece of each prompt behind long cached keys of 4 bits, all read back.
        append_case(8, 256, 16384, 32, 8, 128, "bf16", 4, 64, rotate=True, name="append4_piece"),
        # A few users' next tokens: latency.
        paged_case(4, 1, 150, 16, 2, 128, "bf16", 16, 16, name="paged_small"),
        # A full batch's decoding step over a cache of 16 bits.
        paged_case(48, 1, 8192, 32, 8, 128, "bf16", 16, 64, name="paged_decode"),
        # The same, more sequences, over a cache of 4 bits.
        paged_case(64, 1, 8192, 32, 8, 128, "bf16", 4, 64, name="paged4_decode"),
        # Two users with a book each.
        paged_case(2, 1, 131072, 32, 8, 128, "bf16", 4, 64, lse=True, name="paged4_books"),
        # Drafted tokens checked in one go, head dim 64, ALiBi, a sliding window, odd lengths.
        paged_case(24, 5, 3001, 24, 4, 64, "f16", 4, 16, window=1000, alibi=True, lse=True,
                   name="paged4_draft"),
    ]


# ------------------------------------------------------------------------------ kinds of case
def norm_case(batch, seq, heads, kv_heads, dim, dtype, norm="rmsnorm", first=True, positions=False,
              backward=False, **more):
    """Queries and keys (batch, seq, heads, dim). first: the norm comes before the rotation."""
    return {"op": "norm", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "norm": norm, "first": first, "positions": positions, "backward": backward,
            **more}


def append_case(count, new, cached, heads, kv_heads, dim, dtype, bits, page, packed=False, rotate=False,
                queries=False, spread=1, **more):
    """`new` tokens for each of `count` sequences (packed: up to that many), each behind up to `cached`
    keys. With 4 bits, the whole of the sequences is read back in `dtype`."""
    return {"op": "append", "count": count, "new": new, "cached": cached, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "bits": bits, "page": page, "packed": packed,
            "rotate": rotate, "queries": queries, "spread": spread, **more}


def paged_case(count, seq, longest, heads, kv_heads, dim, dtype, bits, page, window=0, alibi=False,
               lse=False, spread=1, **more):
    """The last `seq` tokens of each of `count` sequences of up to `longest` keys in a paged cache."""
    return {"op": "paged", "count": count, "seq": seq, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "bits": bits, "page": page,
            "window": window, "alibi": alibi, "lse": lse, "spread": spread, **more}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    return min(64, kv * group) // kv * kv, kv


def draw(rng):
    heads, kv_heads = _heads(rng)
    kind = rng.choice(["norm", "append", "paged", "paged"])
    if kind == "norm":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        batch = _log(rng, 1, 64)
        seq = _log(rng, 1, max(1, min(8192, MOST_NORM // ((heads + kv_heads) * dim * batch))))
        return norm_case(batch, seq, heads, kv_heads, dim, rng.choice(["bf16", "bf16", "f16", "f32"]),
                         norm=rng.choice(["rmsnorm", "rmsnorm", "layernorm"]), first=rng.random() < 0.6,
                         positions=rng.random() < 0.4, backward=rng.random() < 0.6)
    dim, dtype = rng.choice([64, 128, 128]), rng.choice(["bf16", "bf16", "f16"])
    bits, page = rng.choice([16, 4, 4]), rng.choice([16, 32, 48, 64, 128])
    spread, row = rng.randrange(1 << 20), kv_heads * dim
    count = _log(rng, 1, 64)
    if kind == "append":
        packed = rng.random() < 0.5
        new = 1 if rng.random() < 0.3 else _log(rng, 1, min(4096, MOST_NEW // (row * count)))
        cached = 0 if rng.random() < 0.3 else _log(rng, 1, min(16384, MOST_CACHED // (row * count)))
        return append_case(count, new, cached, heads, kv_heads, dim, dtype, bits, page, packed=packed,
                           rotate=rng.random() < 0.8, queries=rng.random() < 0.5, spread=spread)
    seq = rng.choice([1, 1, 1, 1, 2, 5, 16, _log(rng, 17, 200)])
    longest = seq + _log(rng, 1, max(2, min(65536, MOST_KEYS // (row * count) - seq,
                                            MOST_SCORES // (count * seq * heads) - seq)))
    window = _log(rng, 1, longest) if rng.random() < 0.2 else 0
    return paged_case(count, seq, longest, heads, kv_heads, dim, dtype, bits, page, window=window,
                      alibi=rng.random() < 0.2, lse=rng.random() < 0.4, spread=spread)


def _spread(rng, count, least, most):
    """Lengths between the two, most of them short, one as long as any, in any order."""
    sizes = [_log(rng, max(least, most // 64, 1), most) for _ in range(count - 1)]
    sizes = [most] + [max(least, n) for n in sizes]
    rng.shuffle(sizes)
    return sizes


def _lengths(c):
    """append, paged: (new tokens, keys with these) of each sequence."""
    rng = random.Random(c["spread"])
    if c["op"] == "paged":
        return [(c["seq"], n) for n in _spread(rng, c["count"], c["seq"], c["longest"])]
    new = _spread(rng, c["count"], 1, c["new"]) if c["packed"] else [c["new"]] * c["count"]
    cached = _spread(rng, c["count"], 1, c["cached"]) if c["cached"] else [0] * c["count"]
    return [(n, n + m) for n, m in zip(new, cached)]


# --------------------------------------------------------------------------------- the inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _tables(rows, dim):
    """cos and sin (rows, dim / 2) in 32 bits, the angles in 64."""
    rate = 10000.0 ** (-torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim)
    angle = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def _norm_inputs(c, seed):
    g, t, d = _generator(seed), DTYPES[c["dtype"]], c["dim"]
    make = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    b, n = c["batch"], c["seq"]
    s = {"q": make(b, n, c["heads"], d).to(t), "k": make(b, n, c["kv_heads"], d).to(t),
         "q_weight": (1.0 + 0.1 * make(d)).to(t), "k_weight": (1.0 + 0.1 * make(d)).to(t)}
    if c["norm"] == "layernorm":
        s["q_bias"], s["k_bias"] = (0.1 * make(d)).to(t), (0.1 * make(d)).to(t)
    if c["backward"]:
        s["dq"], s["dk"] = make(*s["q"].shape).to(t), make(*s["k"].shape).to(t)
    rows = n
    if c["positions"]:
        rows = 8192
        s["positions"] = torch.randint(0, rows, (b, n), generator=g, device=DEV)
    s["cos"], s["sin"] = _tables(rows, d)
    return s


def _table_of_pages(c, g, sizes):
    """(sequences, most pages) page numbers, in any order, -1 behind a sequence's last; pages in all."""
    need = [-(-m // c["page"]) for _, m in sizes]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device=DEV, dtype=torch.int32)
    i = torch.arange(max(need), device=DEV)
    n = torch.tensor(need, device=DEV)
    at = (n.cumsum(0) - n)[:, None] + i
    return torch.where(i < n[:, None], order[at.clamp(max=total - 1)], -1), total


def _pages(c, g, total):
    hk, d, size = c["kv_heads"], c["dim"], c["page"]
    s = {}
    for x in "kv":
        if c["bits"] == 16:
            s[x + "_pages"] = torch.randn(total, hk, size, d, generator=g, device=DEV, dtype=torch.float32
                                          ).to(DTYPES[c["dtype"]])
        else:
            s[x + "_pages"] = torch.randint(0, 256, (total, hk, size, d // 2), generator=g, device=DEV,
                                            dtype=torch.uint8)
            step = 0.2 + 0.2 * torch.rand(total, hk, size, generator=g, device=DEV)
            low = -step * (6.5 + 2.0 * torch.rand(total, hk, size, generator=g, device=DEV))
            s[x + "_scales"] = torch.stack((step, low), dim=-1)
    return s


def _cache_inputs(c, seed):
    g, t, sizes = _generator(seed), DTYPES[c["dtype"]], _lengths(c)
    hq, hk, d = c["heads"], c["kv_heads"], c["dim"]
    make = lambda *shape: torch.randn(*shape, generator=g, device=DEV).to(t)  # noqa: E731
    s = {"lengths": torch.tensor([m for _, m in sizes], dtype=torch.int32, device=DEV)}
    s["block_table"], total = _table_of_pages(c, g, sizes)
    s |= _pages(c, g, total)
    if c["op"] == "paged":
        s["q"] = make(c["count"], c["seq"], hq, d)
        if c["alibi"]:
            s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEV) / hq)
        return s
    rows = (sum(n for n, _ in sizes),) if c["packed"] else (c["count"], c["new"])
    s["k"], s["v"] = make(*rows, hk, d), make(*rows, hk, d)
    if c["queries"]:
        s["q"] = make(*rows, hq, d)
    if c["packed"]:
        s["starts"] = _starts([n for n, _ in sizes])
    if c["rotate"]:
        s["cos"], s["sin"] = _tables(s["block_table"].shape[1] * c["page"], d)
    if c["bits"] == 4:
        s["starts_k"] = _starts([m for _, m in sizes])
    return s


def _starts(sizes):
    at = [0]
    for n in sizes:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def _inputs(c, seed):
    """The tensors of a case, by name: the same for `prepare` and `exact`."""
    return _norm_inputs(c, seed) if c["op"] == "norm" else _cache_inputs(c, seed)


def prepare(case, seed):
    s = {"case": dict(case), **_inputs(case, seed)}
    if case["op"] != "norm":
        # what the program that collects a batch knows of it
        sizes = _lengths(case)
        s["keys"], s["most_keys"] = sum(m for _, m in sizes), max(m for _, m in sizes)
    return s


# --------------------------------------------------------------------------------- the passes
def _turn(x, cos, sin, back=False):
    """The halves of the last dim rotated; cos and sin with a head dim."""
    h = x.shape[-1] // 2
    x1, x2 = x[..., :h], x[..., h:]
    if back:
        return torch.cat((x1 * cos + x2 * sin, x2 * cos - x1 * sin), dim=-1)
    return torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), dim=-1)


def _normed(x, eps, layer):
    """The normalised rows, and what a gradient is scaled by."""
    if layer:
        x = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    return x * rstd, rstd


def _norm_plain(c, s, x, w, b, dy):
    """y, and dx, dw, db where there is dy."""
    layer, t = c["norm"] == "layernorm", x.dtype
    rows = s["positions"] if c["positions"] else slice(0, c["seq"])
    cos, sin = s["cos"][rows].unsqueeze(-2), s["sin"][rows].unsqueeze(-2)
    x, wide = x.float(), w.float()
    n, rstd = _normed(x if c["first"] else _turn(x, cos, sin), _eps(c), layer)
    y = n * wide
    if b is not None:
        y = y + b.float()
    y = _turn(y, cos, sin) if c["first"] else y
    if dy is None:
        return (y.to(t),)
    g = dy.float()
    g = _turn(g, cos, sin, back=True) if c["first"] else g
    dn = g * wide
    dx = dn - n * (dn * n).mean(-1, keepdim=True)
    if layer:
        dx = dx - dn.mean(-1, keepdim=True)
    dx = dx * rstd
    dx = dx if c["first"] else _turn(dx, cos, sin, back=True)
    dw = (g * n).sum((0, 1, 2)).to(w.dtype)
    return y.to(t), dx.to(t), dw, g.sum((0, 1, 2)).to(w.dtype) if b is not None else None


def _eps(c):
    return 1e-5 if c["norm"] == "layernorm" else 1e-6


NORM_NAMES = ("", "d", "d_weight", "d_bias")


def _norm_run_plain(c, s):
    out = {}
    for x in "qk":
        got = _norm_plain(c, s, s[x], s[x + "_weight"], s.get(x + "_bias"), s.get("d" + x))
        out |= {x + "." + name: v for name, v in zip(NORM_NAMES, got) if v is not None}
    return out


def _norm_own(c, s):
    import trinix_b200 as T

    more = {"norm": c["norm"], "norm_first": c["first"], "eps": _eps(c), "positions": s.get("positions")}
    names = [n for n in ("q", "k", "q_weight", "k_weight", "q_bias", "k_bias") if n in s]
    if not c["backward"]:
        y = T.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"],
                           q_bias=s.get("q_bias"), k_bias=s.get("k_bias"), **more)
        return {"q.": y[0], "k.": y[1]}
    leaf = {n: s[n].detach().requires_grad_() for n in names}
    y = T.QKNormRoPEKernel.apply(leaf["q"], leaf["k"], leaf["q_weight"], leaf["k_weight"], s["cos"],
                                 s["sin"], leaf.get("q_bias"), leaf.get("k_bias"), **more)
    grads = torch.autograd.grad(y, list(leaf.values()), (s["dq"], s["dk"]))
    out = {"q.": y[0].detach(), "k.": y[1].detach()}
    for n, g in zip(leaf, grads):
        out[n[0] + ".d" + n[1:]] = g
    return out


def _quantised(x):
    """Codes (two in a byte) and (step, lowest) of rows in 32 bits."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    span = high - low
    none = span < LEAST_RANGE
    # 15 times a difference of 16-bit values, over another one: exact where the quotient is, so that a value
    # halfway between two codes goes to the even one here as in any other precision
    code = ((x - low) * 15.0 / span.masked_fill(none, 1.0)).round().masked_fill(none, 0.0).to(torch.uint8)
    step = (span * FIFTEENTH).masked_fill(none, 0.0)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat((step, low), dim=-1)


def _values(codes, scales):
    """The rows that codes stand for, in 32 bits."""
    code = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).float()
    return scales[..., 1:] + code * scales[..., :1]


def _places(c, s):
    """Sequence and position of each new token."""
    if c["packed"]:
        i = torch.arange(s["k"].shape[0], device=DEV, dtype=torch.int32)
        seq = torch.searchsorted(s["starts"][1:], i, right=True)
        return seq, s["lengths"][seq].long() - (s["starts"][seq + 1] - i)
    at = s["lengths"].long()[:, None] - c["new"] + torch.arange(c["new"], device=DEV)
    return torch.arange(c["count"], device=DEV)[:, None].expand_as(at), at


def _append_plain(c, s):
    seq, at = _places(c, s)
    out = {}
    rows = {"k": s["k"].float(), "v": s["v"].float()}
    if c["queries"]:
        q = s["q"].float()
    if c["rotate"]:
        cos, sin = s["cos"][at].unsqueeze(-2), s["sin"][at].unsqueeze(-2)
        rows["k"] = _turn(rows["k"], cos, sin)
        if c["queries"]:
            q = _turn(q, cos, sin)
    if c["queries"]:
        out["q"] = q.to(s["q"].dtype)
    page, slot = s["block_table"][seq, at // c["page"]].long(), at % c["page"]
    for x in "kv":
        if c["bits"] == 16:
            s[x + "_pages"][page, :, slot] = rows[x].to(s[x + "_pages"].dtype)
            out[x + "_pages"] = s[x + "_pages"]
        else:
            codes, scales = _quantised(rows[x])
            s[x + "_pages"][page, :, slot] = codes
            s[x + "_scales"][page, :, slot] = scales
    if c["bits"] == 4:
        i = torch.arange(s["keys"], device=DEV, dtype=torch.int32)
        seq = torch.searchsorted(s["starts_k"][1:], i, right=True)
        at = (i - s["starts_k"][seq]).long()
        page, slot = s["block_table"][seq, at // c["page"]].long(), at % c["page"]
        for x in "kv":
            rows = _values(s[x + "_pages"][page, :, slot], s[x + "_scales"][page, :, slot])
            out[x] = rows.to(DTYPES[c["dtype"]])
    return out


def _append_own(c, s):
    import trinix_b200 as T

    scales = {"k_scales": s.get("k_scales"), "v_scales": s.get("v_scales")}
    # without a rotation there is nothing to be done with queries
    q = T.append_paged(s["k"], s["v"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"],
                       cos=s.get("cos"), sin=s.get("sin"), q=s.get("q") if c["rotate"] else None,
                       cu_seqlens=s.get("starts"), **scales)
    out = {"q": q if c["rotate"] else s["q"]} if c["queries"] else {}
    if c["bits"] == 16:
        return out | {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    out["k"], out["v"] = T.gather_paged(s["k_pages"], s["v_pages"], s["block_table"], s["starts_k"],
                                        rows=s["keys"], dtype=DTYPES[c["dtype"]], **scales)
    return out


def _paged_plain(c, s):
    b, hq, hk, d, n = c["count"], c["heads"], c["kv_heads"], c["dim"], s["most_keys"]
    table = s["block_table"].long().clamp(min=0)
    rows = {}
    for x in "kv":  # (b, hk, keys, d) in 32 bits
        r = s[x + "_pages"][table]
        r = r.float() if c["bits"] == 16 else _values(r, s[x + "_scales"][table])
        rows[x] = r.transpose(1, 2).reshape(b, hk, -1, d)[:, :, :n]
    j = torch.arange(n, device=DEV)
    length = s["lengths"].long()[:, None]
    away = (length - c["seq"] + torch.arange(c["seq"], device=DEV))[:, :, None] - j  # (b, seq, n)
    hidden = away < 0
    if c["window"]:
        hidden = hidden | (away > c["window"])
    v = rows["v"].masked_fill((j >= length)[:, None, :, None], 0.0)
    q = s["q"].float().view(b, c["seq"], hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    x = (q.reshape(b, hk, -1, d) @ rows["k"].transpose(2, 3)).view(b, hk, hq // hk, c["seq"], n)
    x = x * d ** -0.5
    if c["alibi"]:
        x = x - s["slopes"].view(1, hk, hq // hk, 1, 1) * away[:, None, None].float()
    x = x.masked_fill(hidden[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = (x - top).exp()
    total = x.sum(-1, keepdim=True)
    out = (x.view(b, hk, -1, n) @ v).view(b, hk, hq // hk, c["seq"], d) / total
    out = {"out": out.permute(0, 3, 1, 2, 4).reshape(b, c["seq"], hq, d).to(s["q"].dtype)}
    if c["lse"]:
        out["lse"] = (top + total.log()).reshape(b, hq, c["seq"])
    return out


def _paged_own(c, s):
    import trinix_b200 as T

    r = T.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"],
                          k_scales=s.get("k_scales"), v_scales=s.get("v_scales"),
                          window=(c["window"], 0) if c["window"] else None, alibi_slopes=s.get("slopes"),
                          return_lse=c["lse"])
    return {"out": r[0], "lse": r[1]} if c["lse"] else {"out": r}


def run(state):
    c = state["case"]
    if own:
        return {"norm": _norm_own, "append": _append_own, "paged": _paged_own}[c["op"]](c, state)
    return {"norm": _norm_run_plain, "append": _append_plain, "paged": _paged_plain}[c["op"]](c, state)


# ------------------------------------------------------------------- what a pass cannot avoid
def work(case):
    c, size = case, 4 if case["dtype"] == "f32" else 2
    hq, hk, d = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "norm":
        n = c["batch"] * c["seq"] * (hq + hk) * d
        tokens = c["batch"] * c["seq"] if c["positions"] else c["seq"]
        passes = 4 if c["backward"] else 2  # q and k, their gradients, and both of the results
        weights = 2 * d * size * (2 if c["norm"] == "layernorm" else 1) * (2 if c["backward"] else 1)
        return {"bytes": passes * n * size + 4 * tokens * d + weights,
                "flops": n * (25 if c["backward"] else 8)}
    sizes = _lengths(c)
    row = 2 * d if c["bits"] == 16 else d // 2 + 8  # of the cache, in bytes
    if c["op"] == "append":
        new, keys = sum(n for n, _ in sizes), sum(m for _, m in sizes)
        moved = 2 * new * hk * (2 * d + row) + (4 * new * hq * d if c["queries"] else 0)
        if c["bits"] == 4:  # what was there is read, all of it written in 16 bits
            moved += 2 * hk * ((keys - new) * row + keys * 2 * d)
        values = new * d * (2 * hk + (hq if c["queries"] else 0))
        return {"bytes": moved + (4 * new * d if c["rotate"] else 0), "flops": 6 * values}
    pairs = seen = 0
    for n, m in sizes:
        first = 0 if not c["window"] else max(0, m - n - c["window"])
        seen += m - first
        pairs += sum(min(j, c["window"] + 1) if c["window"] else j for j in range(m - n + 1, m + 1))
    rows = c["count"] * c["seq"]
    return {"bytes": 4 * rows * hq * d + 2 * seen * hk * row + (4 * rows * hq if c["lse"] else 0),
            "flops": 4 * pairs * hq * d}


# --------------------------------------------------------------------------------- in 64 bits
def _norm_exact(c, s):
    """From the definition as a function, and the gradients by differentiating it."""
    cos, sin = s["cos"].double(), s["sin"].double()
    if c["positions"]:
        cos, sin = cos[s["positions"]], sin[s["positions"]]
    else:
        cos, sin = cos[None, :c["seq"]], sin[None, :c["seq"]]
    turn = torch.complex(cos, sin)[:, :, None]

    def rotated(x):
        z = torch.complex(*x.chunk(2, dim=-1)) * turn
        return torch.cat((z.real, z.imag), dim=-1)

    def normed(x, w, b):
        if b is not None:
            x = x - x.mean(-1, keepdim=True)
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _eps(c)) * w
        return x if b is None else x + b

    out = {}
    for n in "qk":
        leaves = [s[n].double().requires_grad_(), s[n + "_weight"].double().requires_grad_()]
        if c["norm"] == "layernorm":
            leaves.append(s[n + "_bias"].double().requires_grad_())
        x, w, b = (leaves + [None])[:3]
        y = rotated(normed(x, w, b)) if c["first"] else normed(rotated(x), w, b)
        out[n + "."] = y.detach()
        if c["backward"]:
            grads = torch.autograd.grad(y, leaves, s["d" + n].double())
            out |= {n + "." + name: g for name, g in zip(NORM_NAMES[1:], grads)}
    return out


def _append_exact(c, s):
    sizes, out = _lengths(c), {}
    k, v = s["k"].reshape(-1, c["kv_heads"], c["dim"]).double(), s["v"].reshape(-1, c["kv_heads"], c["dim"]).double()
    at = torch.cat([torch.arange(m - n, m, device=DEV) for n, m in sizes])
    if c["rotate"]:
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at][:, None]
        rotated = lambda x: torch.view_as_real(torch.complex(*x.chunk(2, dim=-1)) * turn).transpose(-1, -2).flatten(-2)  # noqa: E731,E501
    else:
        rotated = lambda x: x  # noqa: E731
    k = rotated(k)
    if c["queries"]:
        q = s["q"].reshape(-1, c["heads"], c["dim"]).double()
        out["q"] = rotated(q).view(s["q"].shape)

    def held(x):  # the values that 4 bits leave of rows
        low = x.min(dim=-1, keepdim=True).values
        span = x.max(dim=-1, keepdim=True).values - low
        code = torch.round((x - low) * 15 / torch.where(span > 0, span, 1.0))
        return low + code * span / 15

    whole, row = {"k": [], "v": []}, 0
    for x, new in (("k", k), ("v", v)):
        pages = s[x + "_pages"]
        if c["bits"] == 16:
            pages = pages.double()
            row = 0
            for b, (n, m) in enumerate(sizes):
                p = torch.arange(m - n, m, device=DEV)
                page = s["block_table"][b].long()[torch.div(p, c["page"], rounding_mode="floor")]
                pages[page, :, p.remainder(c["page"])] = new[row:row + n]
                row += n
            out[x + "_pages"] = pages
            continue
        row = 0
        for b, (n, m) in enumerate(sizes):
            whole[x] += [_cached(s, c, x, b, m - n), held(new[row:row + n])]
            row += n
        out[x] = torch.cat(whole[x])
    return out


def _cached(s, c, x, b, n):
    """The first n rows of sequence b in 64 bits, (n, heads, dim)."""
    pages = s["block_table"][b, :-(-n // c["page"])].long()
    r = s[x + "_pages"][pages].transpose(1, 2).flatten(0, 1)[:n]
    if c["bits"] == 16:
        return r.double()
    scales = s[x + "_scales"][pages].transpose(1, 2).flatten(0, 1)[:n].double()
    wide = torch.empty(*r.shape[:-1], c["dim"], dtype=torch.float64, device=DEV)
    wide[..., 0::2], wide[..., 1::2] = (r % 16).double(), torch.div(r, 16, rounding_mode="floor").double()
    return wide * scales[..., :1] + scales[..., 1:]


def _paged_exact(c, s):
    group, n, d = c["heads"] // c["kv_heads"], c["seq"], c["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(c["count"], c["heads"], n, dtype=torch.float64, device=DEV)
    for b, (_, m) in enumerate(_lengths(c)):
        k, v = _cached(s, c, "k", b, m), _cached(s, c, "v", b, m)
        i = torch.arange(m - n, m, device=DEV)[:, None]
        j = torch.arange(m, device=DEV)
        for h in range(c["heads"]):
            w = s["q"][b, :, h].double() @ k[:, h // group].t() * d ** -0.5
            if c["alibi"]:
                w = w - s["slopes"][h].double() * (i - j)
            w = torch.where(j > i, float("-inf"), w)
            if c["window"]:
                w = torch.where(i - j > c["window"], float("-inf"), w)
            lse[b, h] = torch.logsumexp(w, dim=-1)
            out[b, :, h] = torch.softmax(w, dim=-1) @ v[:, h // group]
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


def exact(case, seed):
    s = _inputs(case, seed)
    return {"norm": _norm_exact, "append": _append_exact, "paged": _paged_exact}[case["op"]](case, s)
