"""Attention over packed sequences and over a shared prefix, as cases that can be timed.

`run` computes a case either in its plain form, with elementary torch operations in 32 bits, or (with
`own`) through the package's public entry points `attention_packed` and `attention_shared_prefix`.
`exact` is the same from the definition, in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}

# Query-key pairs, padded to the longest, times heads, of a drawn case: at most the 5.5e11 operations
# of the largest listed one.
MOST_SCORES = 1_000_000_000
# Keys and values: the largest listed case has 276 MB.
MOST_KV_BYTES = 270_000_000


def listed():
    return [
        # A few short questions: nothing but call and launch latency.
        packed_case("causal", 4, 60, 16, 2, 128, "bf16", name="packed_small"),
        # The prompts that a server has collected, of very different lengths, prefilled together.
        packed_case("causal", 16, 2048, 32, 8, 128, "bf16", name="packed_prompts"),
        # Two documents: the largest call.
        packed_case("causal", 2, 8192, 32, 8, 128, "bf16", name="packed_long"),
        # One step of a server that mixes single tokens with pieces of prompts, each behind its cached
        # keys; the batch is padded to a fixed number of rows, as a captured graph wants it.
        packed_case("causal", 24, 500, 32, 8, 128, "bf16", cached=4096, spare=77, lse=True,
                    name="packed_mixed"),
        # An encoder over a packed batch of texts: no causal order, head dim 64.
        packed_case("full", 32, 509, 16, 16, 64, "f16", lse=True, name="packed_encoder"),
        # Sliding window and ALiBi, five query heads to a kv head.
        packed_case("window", 6, 1500, 40, 8, 128, "f16", window=256, alibi=True,
                    name="packed_window"),
        # One decoding step of sequences whose caches are packed.
        packed_case("causal", 48, 1, 32, 8, 128, "bf16", cached=8000, name="packed_decode"),
        # A few users behind a short system prompt.
        shared_case(4, 1, 150, 60, 16, 2, 128, "bf16", name="shared_small"),
        # A full batch behind a long system prompt, one token each.
        shared_case(64, 1, 8192, 1024, 32, 8, 128, "bf16", name="shared_decode"),
        # Questions about one book.
        shared_case(16, 1, 65536, 300, 32, 8, 128, "bf16", name="shared_book"),
        # Drafted tokens checked in one go, head dim 64, odd lengths.
        shared_case(32, 7, 3001, 801, 32, 4, 64, "f16", lse=True, name="shared_draft"),
        # The prompts of a batch behind the prefix that they share.
        shared_case(16, 320, 4096, 384, 32, 8, 128, "bf16", name="shared_prompts"),
    ]


# ------------------------------------------------------------------------------ kinds of case
def packed_case(kind, count, longest, heads, kv_heads, dim, dtype, cached=0, spare=0, window=0,
                alibi=False, lse=False, spread=1, **more):
    """`count` sequences of up to `longest` queries, each behind up to `cached` keys of its own;
    `spare` rows behind the last one. kind: "causal", "window" (the last `window` keys), "full"."""
    return {"op": "packed", "kind": kind, "count": count, "longest": longest, "cached": cached,
            "spare": spare, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "window": window, "alibi": alibi, "lse": lse, "spread": spread, **more}


def shared_case(batch, seq, prefix, capacity, heads, kv_heads, dim, dtype, alibi=False, lse=False,
                spread=1, **more):
    """`seq` new tokens each behind `prefix` shared keys and up to `capacity` of their own."""
    return {"op": "shared", "batch": batch, "seq": seq, "prefix": prefix, "capacity": capacity,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "alibi": alibi,
            "lse": lse, "spread": spread, **more}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    return min(64, kv * group) // kv * kv, kv


def draw(rng):
    heads, kv_heads = _heads(rng)
    dim, dtype = rng.choice([64, 128, 128]), rng.choice(["bf16", "bf16", "f16"])
    more = {"alibi": rng.random() < 0.2, "lse": rng.random() < 0.4, "spread": rng.randrange(1 << 20)}
    key_bytes = 4 * kv_heads * dim
    if rng.random() < 0.5:
        kind = rng.choice(["causal", "causal", "causal", "window", "full"])
        count = _log(rng, 1, 64)
        keys = MOST_KV_BYTES // (key_bytes * count)
        cached = _log(rng, 1, min(8192, keys // 2)) if rng.random() < 0.4 else 0
        most = min(8192, keys - cached)
        while most > 1 and count * heads * most * (most + cached) > MOST_SCORES:
            most = most * 7 // 8
        longest = 1 if cached and rng.random() < 0.3 else _log(rng, 1, most)
        window = _log(rng, 1, longest + cached) if kind == "window" else 0
        return packed_case(kind, count, longest, heads, kv_heads, dim, dtype, cached=cached,
                           spare=rng.choice([0, 0, 1, 50]), window=window, **more)
    batch, seq = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 5, 16, _log(rng, 17, 400)])
    capacity = seq + _log(rng, 1, max(2, min(2048, MOST_KV_BYTES // (2 * key_bytes * batch) - seq)))
    most = min(65536, MOST_KV_BYTES // (2 * key_bytes),
               MOST_SCORES // (batch * seq * heads) - capacity)
    return shared_case(batch, seq, _log(rng, 16, max(16, most)), capacity, heads, kv_heads, dim,
                       dtype, **more)


def _spread(rng, count, least, most):
    """Lengths between the two, most of them short, one as long as any, in any order."""
    sizes = [_log(rng, max(least, most // 64, 1), most) for _ in range(count - 1)]
    sizes = [most] + [max(least, n) for n in sizes]
    rng.shuffle(sizes)
    return sizes


def _lengths(c):
    """packed: (queries, keys) of each sequence; shared: (new tokens, own keys) of each."""
    rng = random.Random(c["spread"])
    if c["op"] == "shared":
        return [(c["seq"], n) for n in _spread(rng, c["batch"], c["seq"], c["capacity"])]
    queries = _spread(rng, c["count"], 1, c["longest"])
    cached = _spread(rng, c["count"], 1, c["cached"]) if c["cached"] else [0] * c["count"]
    return [(n, n + m) for n, m in zip(queries, cached)]


# --------------------------------------------------------------------------------- the inputs
def _starts(sizes):
    at = [0]
    for n in sizes:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def _inputs(c, seed):
    """The tensors of a case, by name: the same for `prepare` and `exact`."""
    g = torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)
    make = lambda *shape: torch.randn(*shape, generator=g, device=DEV).to(DTYPES[c["dtype"]])  # noqa: E731
    hq, hk, d = c["heads"], c["kv_heads"], c["dim"]
    sizes = _lengths(c)
    if c["op"] == "packed":
        rows, keys = sum(n for n, _ in sizes) + c["spare"], sum(m for _, m in sizes)
        s = {"q": make(rows, hq, d), "k": make(keys, hk, d), "v": make(keys, hk, d),
             "starts_q": _starts([n for n, _ in sizes]), "starts_k": _starts([m for _, m in sizes])}
    else:
        b, cap, p = c["batch"], c["capacity"], c["prefix"]
        s = {"q": make(b, c["seq"], hq, d), "prefix_k": make(p, hk, d), "prefix_v": make(p, hk, d),
             "k": make(b, cap, hk, d), "v": make(b, cap, hk, d),
             "lengths": torch.tensor([n for _, n in sizes], dtype=torch.int32, device=DEV)}
    if c["alibi"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEV) / hq)
    return s


def prepare(case, seed):
    sizes = _lengths(case)
    # the longest of each, as a program that makes the batch knows them
    return {"case": dict(case), "most_q": max(n for n, _ in sizes), "most_k": max(m for _, m in sizes),
            **_inputs(case, seed)}


# --------------------------------------------------------------------------------- the passes
def _attend(q, k, v, hidden, scale, slopes, distance):
    """q (n, Hk, G, Mq, D), k / v (n, Hk, Mk, D), hidden and distance (n, Mq, Mk): out, lse."""
    n, hk, g, mq, d = q.shape
    s = q.reshape(n, hk, g * mq, d) @ k.transpose(2, 3)
    s = s.view(n, hk, g, mq, -1).mul_(scale)
    if slopes is not None:
        s.addcmul_(slopes.view(1, hk, g, 1, 1), distance[:, None, None].float(), value=-1.0)
    s.masked_fill_(hidden[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = top.masked_fill(top == float("-inf"), 0.0)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    out = (s.view(n, hk, g * mq, -1) @ v).view(n, hk, g, mq, d)
    return out / total.masked_fill(total == 0, 1.0), (top + total.log()).squeeze(-1)


def _padded(x, starts, most):
    """(n, most, H, D) in 32 bits from packed rows, zeros behind each sequence."""
    at = starts[:-1, None] + torch.arange(most, device=DEV)
    there = at < starts[1:, None]
    return x[at.clamp(max=x.shape[0] - 1)].float().masked_fill_(~there[..., None, None], 0.0)


def _packed_plain(c, s):
    hq, hk, d = c["heads"], c["kv_heads"], c["dim"]
    len_q, len_k = s["starts_q"].diff(), s["starts_k"].diff()
    q = _padded(s["q"], s["starts_q"], s["most_q"]).view(-1, s["most_q"], hk, hq // hk, d)
    k = _padded(s["k"], s["starts_k"], s["most_k"]).transpose(1, 2)
    v = _padded(s["v"], s["starts_k"], s["most_k"]).transpose(1, 2)
    i = torch.arange(s["most_q"], device=DEV)[None] + (len_k - len_q)[:, None]
    away = i[:, :, None] - torch.arange(s["most_k"], device=DEV)  # positions back to the key
    hidden = (away <= i[:, :, None] - len_k[:, None, None])
    if c["kind"] != "full":
        hidden |= away < 0
    if c["kind"] == "window":
        hidden |= away > c["window"]
    out, lse = _attend(q.permute(0, 2, 3, 1, 4), k, v, hidden, d ** -0.5, s.get("slopes"), away.abs())
    rows = torch.arange(s["q"].shape[0], device=DEV, dtype=torch.int32)
    seq = torch.searchsorted(s["starts_q"][1:], rows, right=True)
    spare = seq >= c["count"]
    seq = seq.clamp(max=c["count"] - 1)
    at = (rows - s["starts_q"][seq]).clamp(max=s["most_q"] - 1)
    out = out.permute(0, 3, 1, 2, 4)[seq, at].masked_fill(spare[:, None, None, None], 0.0)
    lse = lse.permute(0, 3, 1, 2)[seq, at].masked_fill(spare[:, None, None], float("-inf"))
    return out.reshape(-1, hq, d).to(s["q"].dtype), lse.reshape(-1, hq).t().contiguous()


def _shared_plain(c, s):
    b, hq, hk, d, p = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["prefix"]
    n = s["lengths"][:, None]
    there = torch.arange(c["capacity"], device=DEV) < n
    k = torch.cat((s["prefix_k"].expand(b, -1, -1, -1), s["k"]), dim=1).float().transpose(1, 2)
    own_v = s["v"].masked_fill(~there[..., None, None], 0.0)
    v = torch.cat((s["prefix_v"].expand(b, -1, -1, -1), own_v), dim=1).float().transpose(1, 2)
    i = p + n - c["seq"] + torch.arange(c["seq"], device=DEV)[None]
    away = i[:, :, None] - torch.arange(p + c["capacity"], device=DEV)
    q = s["q"].float().view(b, c["seq"], hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    out, lse = _attend(q, k, v, away < 0, d ** -0.5, s.get("slopes"), away)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, c["seq"], hq, d).to(s["q"].dtype)
    return out, lse.reshape(b, hq, c["seq"])


def _packed_own(c, s):
    import trinix_b200 as T

    return T.attention_packed(
        s["q"], s["k"], s["v"], s["starts_q"], s["starts_k"], max_seqlen_q=s["most_q"],
        causal=c["kind"] == "causal", window=(c["window"], 0) if c["kind"] == "window" else None,
        alibi_slopes=s.get("slopes"), return_lse=c["lse"])


def _shared_own(c, s):
    import trinix_b200 as T

    return T.attention_shared_prefix(
        s["q"], s["prefix_k"], s["prefix_v"], s["k"], s["v"], s["lengths"],
        alibi_slopes=s.get("slopes"), return_lse=c["lse"])


def run(state):
    c = state["case"]
    if own:
        r = (_packed_own if c["op"] == "packed" else _shared_own)(c, state)
        return {"out": r[0], "lse": r[1]} if c["lse"] else {"out": r}
    out, lse = (_packed_plain if c["op"] == "packed" else _shared_plain)(c, state)
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


# ------------------------------------------------------------------- what a pass cannot avoid
def _seen(c, n, m):
    """Query-key pairs of one head of a sequence of n queries and m keys, n <= m."""
    if c.get("kind") == "full":
        return n * m
    keys = range(m - n + 1, m + 1)  # up to each query's own position
    if c.get("kind") == "window":
        return sum(min(j, c["window"] + 1) for j in keys)
    return n * (m - n) + n * (n + 1) // 2


def work(case):
    c = case
    sizes = _lengths(c)
    row, key = 4 * c["heads"] * c["dim"], 4 * c["kv_heads"] * c["dim"]
    if c["op"] == "packed":
        pairs = sum(_seen(c, n, m) for n, m in sizes)
        rows, keys = sum(n for n, _ in sizes), sum(m for _, m in sizes)
    else:
        pairs = sum(_seen(c, n, c["prefix"] + m) for n, m in sizes)
        rows, keys = c["batch"] * c["seq"], c["prefix"] + sum(m for _, m in sizes)
    lse = 4 * rows * c["heads"] if c["lse"] else 0
    return {"bytes": rows * row + keys * key + lse, "flops": 4 * pairs * c["heads"] * c["dim"]}


# --------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """A head of a sequence at a time, 1024 of its queries at a time."""
    c, s = case, _inputs(case, seed)
    shared, d, group = c["op"] == "shared", c["dim"], c["heads"] // c["kv_heads"]
    q = s["q"].reshape(-1, c["heads"], d)
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=DEV)
    row = key = 0
    for b, (n, m) in enumerate(_lengths(c)):
        if shared:
            keys, values = (torch.cat((s["prefix_" + x], s[x][b, :m])) for x in "kv")
        else:
            keys, values = s["k"][key:key + m], s["v"][key:key + m]
        j = torch.arange(keys.shape[0], device=DEV)
        for h in range(c["heads"]):
            kk, vv = keys[:, h // group].double(), values[:, h // group].double()
            for at in range(0, n, 1024):
                to = min(n, at + 1024)
                i = torch.arange(at, to, device=DEV)[:, None] + (keys.shape[0] - n)
                w = q[row + at:row + to, h].double() @ kk.t() * d ** -0.5
                if c["alibi"]:
                    w -= s["slopes"][h].double() * (i - j).abs()
                if shared or c["kind"] != "full":
                    w = torch.where(j > i, float("-inf"), w)
                if not shared and c["kind"] == "window":
                    w = torch.where(j < i - c["window"], float("-inf"), w)
                lse[row + at:row + to, h] = torch.logsumexp(w, dim=-1)
                out[row + at:row + to, h] = torch.softmax(w, dim=-1) @ vv
        row, key = row + n, key + m
    out = out.view(s["q"].shape)
    if not c["lse"]:
        return {"out": out}
    return {"out": out, "lse": lse.view(c["batch"], c["seq"], -1).transpose(1, 2) if shared
            else lse.t()}
