"""Attention of a batch behind a shared prefix against the definition in 64 bits, one sequence at a time."""
import pytest
import torch

import trinix_b200 as T
from tests.ragged_ref import assert_within, attend64
from tests.test_gpu_packed import make, slopes_of, starts

pytestmark = pytest.mark.gpu


def check(out, lse, q, pk, pv, k, v, lens, **how):
    for b, n in enumerate(lens):
        keys, values = torch.cat((pk, k[b, :n])), torch.cat((pv, v[b, :n]))
        want, want_lse, allowed, allowed_lse = attend64(q[b], keys, values, causal=True, **how)
        assert_within(out[b], want, allowed, f"sequence {b}")
        if lse is not None:
            assert_within(lse[b], want_lse, allowed_lse, f"lse of sequence {b}")


def inputs(dev, dtype, B, Sq, P, S, hq, hk, d, seed=1):
    q = make(seed, dev, dtype, B, Sq, hq, d)
    pk, pv = (make(seed + i, dev, dtype, P, hk, d) for i in (1, 2))
    k, v = (make(seed + i, dev, dtype, B, S, hk, d) for i in (3, 4))
    return q, pk, pv, k, v


def lengths(lens, dev):
    return torch.tensor(lens, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (8, 2), (6, 2), (5, 5)])
@pytest.mark.parametrize("Sq,lens", [(1, [1, 40, 7, 0, 130]), (3, [3, 5, 129, 1, 0]), (16, [16, 100, 260, 31, 128]),
                                     (17, [17, 128, 300, 4, 0]), (150, [150, 300, 151, 20])], ids=str)
@pytest.mark.parametrize("P", [0, 1, 127, 128, 300, 1500, 4097, 6500])
def test_lengths(cuda, P, Sq, lens, heads, kv):
    dtype, dim = (torch.bfloat16, 128) if heads % 2 else (torch.float16, 64)
    q, pk, pv, k, v = inputs(cuda, dtype, len(lens), Sq, P, max(lens) + 5, heads, kv, dim)
    for b, n in enumerate(lens):  # what lies behind a sequence's last key is never used
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    out, lse = T.attention_shared_prefix(q, pk, pv, k, v, lengths(lens, cuda), return_lse=True)
    check(out, lse, q, pk, pv, k, v, lens)


@pytest.mark.parametrize("heads,kv", [(3, 1), (7, 1), (32, 8), (48, 1), (71, 1), (130, 1), (16, 16)])
@pytest.mark.parametrize("Sq,P", [(1, 500), (2, 5000), (33, 500), (33, 5000)])
def test_groups(cuda, heads, kv, Sq, P):
    lens = [33, 50, 64]
    q, pk, pv, k, v = inputs(cuda, torch.bfloat16, 3, Sq, P, 64, heads, kv, 64, seed=20)
    out, lse = T.attention_shared_prefix(q, pk, pv, k, v, lengths(lens, cuda), return_lse=True)
    check(out, lse, q, pk, pv, k, v, lens)


@pytest.mark.parametrize("dim", [64, 128, 80, 16])
@pytest.mark.parametrize("Sq,P", [(1, 700), (4, 5555), (100, 700), (60, 9001)])
@pytest.mark.parametrize("how", [dict(alibi=True), dict(scale=0.4), dict(alibi=True, scale=0.01)], ids=str)
def test_biases(cuda, how, Sq, P, dim):
    how = dict(how)
    slopes = slopes_of(8, cuda) if how.pop("alibi", False) else None
    lens = [100, 333, 128]
    q, pk, pv, k, v = inputs(cuda, torch.bfloat16, 3, Sq, P, 333, 8, 2, dim, seed=30)
    out, lse = T.attention_shared_prefix(q, pk, pv, k, v, lengths(lens, cuda), alibi_slopes=slopes,
                                         return_lse=True, **how)
    check(out, lse, q, pk, pv, k, v, lens, slopes=slopes, **how)


@pytest.mark.parametrize("P", [129, 600, 9000, 20_000])
@pytest.mark.parametrize("heads,kv", [(4, 4), (32, 8), (5, 1)])
@pytest.mark.parametrize("alibi", [False, True])
def test_one_tile_of_rows(cuda, P, heads, kv, alibi):
    """All rows in one Q tile: the two have every second tile of a split's keys, an odd number among them."""
    slopes = slopes_of(heads, cuda) if alibi else None
    lens = [1, 20, 64, 5, 33]
    q, pk, pv, k, v = inputs(cuda, torch.bfloat16, 5, 2, P, 64, heads, kv, 128, seed=45)
    out, lse = T.attention_shared_prefix(q, pk, pv, k, v, lengths(lens, cuda), return_lse=True,
                                         alibi_slopes=slopes)
    check(out, lse, q, pk, pv, k, v, lens, slopes=slopes)


@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("B,Sq,P,heads,kv", [(5, 2, 3000, 160, 160), (1300, 1, 1500, 32, 8)])
def test_more_prefix_items_than_sms(cuda, B, Sq, P, heads, kv, alibi):
    """Many heads, all rows in one tile; many rows. The prefix's launch is of several items per CTA."""
    assert T._lib.load().trx_attn_shared_bytes(B, Sq, P, 40, heads, kv, 64) > 0
    slopes = slopes_of(heads, cuda) if alibi else None
    lens = [2 + (7 * b) % 39 for b in range(B)]
    q, pk, pv, k, v = inputs(cuda, torch.float16, B, Sq, P, 40, heads, kv, 64, seed=47)
    out, lse = T.attention_shared_prefix(q, pk, pv, k, v, lengths(lens, cuda), return_lse=True,
                                         alibi_slopes=slopes)
    some = torch.arange(0, B, max(1, B // 25), device=cuda)
    check(out[some], lse[some], q[some], pk, pv, k[some], v[some], [lens[b] for b in some.tolist()],
          slopes=slopes)
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("Sq,B", [(1, 100), (5, 60), (300, 12)])
@pytest.mark.parametrize("alibi", [False, True])
def test_many_rows(cuda, Sq, B, alibi):
    """Several tiles of rows against the prefix, and several items per CTA; no lengths: all keys in use."""
    slopes = slopes_of(32, cuda) if alibi else None
    q, pk, pv, k, v = inputs(cuda, torch.bfloat16, B, Sq, 1000, 320, 32, 8, 128, seed=40)
    out, lse = T.attention_shared_prefix(q, pk, pv, k, v, return_lse=True, alibi_slopes=slopes)
    check(out, lse, q, pk, pv, k, v, [320] * B, slopes=slopes)


@pytest.mark.parametrize("Sq,P", [(1, 200), (6, 200), (40, 200), (1, 5000), (6, 5000), (40, 9000)])
def test_views(cuda, Sq, P):
    """Caches of another layout (batch, heads, rows, head_dim), a prefix and queries that are slices."""
    B, S, hq, hk, d = 3, 60, 8, 2, 128
    lens = [40, 60, 51]
    qkv = make(50, cuda, torch.bfloat16, B, Sq, hq + 2 * hk, d)
    pre = make(51, cuda, torch.bfloat16, P, 2, hk, d)
    cache = make(52, cuda, torch.bfloat16, 2, B, hk, S, d)
    q, pk, pv = qkv[:, :, :hq], pre[:, 0], pre[:, 1]
    k, v = cache[0].transpose(1, 2), cache[1].transpose(1, 2)
    out = T.attention_shared_prefix(q, pk, pv, k, v, lengths(lens, cuda))
    check(out, None, q, pk, pv, k, v, lens)
    gap = make(53, cuda, torch.bfloat16, B, Sq + 2, hq, d)[:, 1:-1]  # rows that are not one run
    out = T.attention_shared_prefix(gap, pk, pv, k, v, lengths(lens, cuda))
    check(out, None, gap, pk, pv, k, v, lens)
    odd = make(54, cuda, torch.bfloat16, B, Sq, hq, d + 1)[..., 1:]
    one = make(55, cuda, torch.bfloat16, B, S, 1, d).expand(-1, -1, hk, -1)
    out = T.attention_shared_prefix(odd, pk, pv, one, one, lengths(lens, cuda))
    check(out, None, odd, pk, pv, one, one, lens)


def test_no_own_keys_and_empty_calls(cuda):
    q, pk, pv, k, v = inputs(cuda, torch.bfloat16, 2, 1, 77, 0, 4, 2, 64, seed=60)
    out, lse = T.attention_shared_prefix(q, pk, pv, k, v, return_lse=True)
    check(out, lse, q, pk, pv, k, v, [0, 0])
    out, lse = T.attention_shared_prefix(q, pk[:0], pv[:0], k, v, return_lse=True)
    assert not out.any() and torch.equal(lse, torch.full_like(lse, float("-inf")))
    assert T.attention_shared_prefix(q[:0], pk, pv, k[:0], v[:0]).shape == (0, 1, 4, 64)
    assert T.attention_shared_prefix(q[:, :0], pk, pv, k, v).shape == (2, 0, 4, 64)


def test_bad_lengths_are_cut(cuda):
    q, pk, pv, k, v = inputs(cuda, torch.bfloat16, 3, 1, 90, 50, 4, 2, 64, seed=61)
    got = T.attention_shared_prefix(q, pk, pv, k, v, lengths([-5, 1 << 30, 50], cuda))
    check(got, None, q, pk, pv, k, v, [0, 50, 50])


def test_long_offsets(cuda):
    """Element offsets beyond 32 bits in the caches."""
    B, S, hk, d = 70, 33_000, 8, 128
    k = torch.zeros(B, S, hk, d, dtype=torch.bfloat16, device=cuda)  # 4.7 GB
    k[-1, :40] = make(62, cuda, torch.bfloat16, 40, hk, d)
    k[-1, 40:] = float("nan")
    pk = make(63, cuda, torch.bfloat16, 100, hk, d)
    lens = [1] * (B - 1) + [40]
    for Sq in (1, 20):
        q = make(64, cuda, torch.bfloat16, B, Sq, hk, d)
        out = T.attention_shared_prefix(q, pk, pk, k, k, lengths(lens, cuda))
        check(out[-1:], None, q[-1:], pk, pk, k[-1:, :40], k[-1:, :40], [40])


def test_prompts_then_tokens(cuda):
    """As a server uses the two: the prefix's prompt and the users' prompts prefilled, then tokens."""
    hq, hk, d, P, S = 8, 2, 128, 333, 64
    prompts = [5, 17, 40, 1]
    B = len(prompts)
    pk, pv = make(70, cuda, torch.bfloat16, P, hk, d), make(71, cuda, torch.bfloat16, P, hk, d)
    k, v = (torch.full((B, S, hk, d), float("nan"), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    new_k, new_v = (make(s, cuda, torch.bfloat16, sum(prompts), hk, d) for s in (72, 73))
    q = make(74, cuda, torch.bfloat16, sum(prompts), hq, d)
    at = 0
    for b, n in enumerate(prompts):
        k[b, :n], v[b, :n] = new_k[at:at + n], new_v[at:at + n]
        at += n
    # prefill: every user's prompt behind the prefix, packed
    keys = torch.cat([torch.cat((pk, k[b, :n])) for b, n in enumerate(prompts)])
    values = torch.cat([torch.cat((pv, v[b, :n])) for b, n in enumerate(prompts)])
    packed, lse = T.attention_packed(q, keys, values, starts(prompts, cuda),
                                     starts([P + n for n in prompts], cuda), causal=True, return_lse=True)
    at = 0
    for b, n in enumerate(prompts):
        want, want_lse, allowed, allowed_lse = attend64(q[at:at + n], torch.cat((pk, k[b, :n])),
                                                        torch.cat((pv, v[b, :n])), causal=True)
        assert_within(packed[at:at + n], want, allowed)
        assert_within(lse[:, at:at + n], want_lse, allowed_lse)
        # the same rows through the other entry point, both within the bound of the definition
        one = T.attention_shared_prefix(q[None, at:at + n], pk, pv, k[b:b + 1], v[b:b + 1],
                                        lengths([n], cuda))
        assert_within(one[0], want, allowed)
        at += n
    lens = list(prompts)
    for step in range(3):  # tokens
        for b in range(B):
            k[b, lens[b]], v[b, lens[b]] = make(80 + 7 * step + b, cuda, torch.bfloat16, 2, hk, d)
            lens[b] += 1
        tok = make(90 + step, cuda, torch.bfloat16, B, 1, hq, d)
        out, lse = T.attention_shared_prefix(tok, pk, pv, k, v, lengths(lens, cuda), return_lse=True)
        check(out, lse, tok, pk, pv, k, v, lens)


def test_more_rows_than_a_grid_holds(cuda):
    """Rows of the batch in more blocks than the prefix's launch has room for: one pass, whatever a cost says."""
    B, Sq, P, hq = 50_000, 3, 6000, 128
    q, pk, pv, k, v = inputs(cuda, torch.bfloat16, 1, Sq, P, 8, hq, 1, 64, seed=70)
    many = [t.expand(B, -1, -1, -1).contiguous() for t in (q, k, v)]  # 2.5 GB of queries
    out = T.attention_shared_prefix(many[0], pk, pv, *many[1:])
    check(out[:1], None, q, pk, pv, k, v, [8])
    assert bool((out == out[:1]).all())


def test_more_rows_of_a_sequence_than_a_grid_holds(cuda):
    """One sequence whose rows, at 128 heads to a tile, are more blocks than one pass has room for."""
    Sq, P, n, hq = 131_075, 100, 150, 128
    q, pk, pv, k, v = inputs(cuda, torch.bfloat16, 1, Sq, P, 200, hq, 1, 64, seed=80)  # 2.1 GB of queries
    out, lse = T.attention_shared_prefix(q, pk, pv, k, v, lengths([n], cuda), return_lse=True)
    last = 300  # of which the first 50 stand in front of every key, as do all rows before them
    check(out[:, -last:], lse[:, :, -last:], q[:, -last:], pk, pv, k, v, [n])
    assert not out[:, :-last].any() and bool((lse[:, :, :-last] == float("-inf")).all())


@pytest.mark.parametrize("Sq,P", [(1, 40), (1, 5000), (30, 200)])
def test_strides_of_tensors_without_keys(cuda, Sq, P):
    """A prefix, or caches, without keys: whatever their strides are."""
    q, pk, pv, k, v = inputs(cuda, torch.bfloat16, 3, Sq, P, 50, 8, 2, 64, seed=90)
    nothing = make(95, cuda, torch.bfloat16, 7, 2, 68)[:0, :, :64]
    out, lse = T.attention_shared_prefix(q, nothing, nothing, k, v, return_lse=True)
    check(out, lse, q, pk[:0], pv[:0], k, v, [50] * 3)
    for empty in (make(96, cuda, torch.bfloat16, 3, 7, 2, 68)[:, :0, :, :64], k[:, :0, :1].expand(-1, -1, 2, -1)):
        out, lse = T.attention_shared_prefix(q, pk, pv, empty, empty, return_lse=True)
        check(out, lse, q, pk, pv, empty, empty, [0] * 3)
