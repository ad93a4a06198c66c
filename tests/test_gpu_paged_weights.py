"""Attention over a paged cache: what becomes of the weights between the two products, of keys that a query does not
see, and of calls at the borders of their arguments."""
import pytest
import torch

import trinix_b200 as T
from tests.paged_ref import make_cache
from tests.test_gpu_paged import check_attention

pytestmark = pytest.mark.gpu


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def two_kinds_of_keys(cuda, scores, n, bits, dtype, dim=64, big=1.0, heads=4):
    """A sequence to each of `scores`, of n keys: the first has score 0 for the query (1, 0, 0, ..), all others the
    sequence's own; the first value is 0 (column 1: `big`), the others `big` (column 1: 0)."""
    c = make_cache([n] * len(scores), 1, 16, dim, bits, dtype, cuda)
    exact = torch.tensor(scores, dtype=torch.float64).to(dtype).double()  # as the cache holds them
    for b, s in enumerate(exact.tolist()):
        pages = c["block_table"][b].long()
        place = lambda x, first, rest: (c[x].index_fill_(0, pages, rest), c[x][pages[0], :, 0].fill_(first))  # noqa: E731
        if bits == 16:
            place("k_pages", 0.0, s)
            place("v_pages", 0.0, big)
            c["v_pages"][pages, ..., 1] = 0.0
            c["v_pages"][pages[0], :, 0, 1] = big
        else:
            for x in "kv":
                c[x + "_pages"][pages] = 0
                c[x + "_scales"][pages] = 0.0
            c["k_scales"][pages, ..., 1] = s
            c["k_scales"][pages[0], :, 0] = 0.0
            c["v_scales"][pages, ..., 0] = big / 16
            c["v_pages"][pages] = 0xFF
            c["v_pages"][pages, ..., 0] = 0x0F       # column 1 in the high bits
            c["v_pages"][pages[0], :, 0] = 0
            c["v_pages"][pages[0], :, 0, 0] = 0xF0
    q = torch.zeros(len(scores), 1, heads, dim, device=cuda, dtype=dtype)
    q[..., 0] = 1.0
    out = T.attention_paged(q, **c, lengths=i32([n] * len(scores), cuda), scale=1.0)
    w = exact.to(cuda).exp()
    high = big if bits == 16 else 15 * big / 16
    rest, first = (high * t / (1 + (n - 1) * w) for t in ((n - 1) * w, torch.ones_like(w)))
    want = rest[:, None].expand(len(scores), dim).clone()
    want[:, 1] = first
    return out[:, 0], want[:, None]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("n,dim,heads", [(40, 64, 1), (40, 128, 4), (2000, 64, 4), (40, 128, 7), (2000, 64, 16)])
def test_weights_are_not_rounded_to_the_cache_s_type(cuda, n, dim, heads, dtype, bits):
    """The result is the definition's, rounded, but for fp32 errors: all of the keys but one have the same weight, so that
    a rounding of weights is an error of the result. With y the result before its rounding, |out - exact| is at most
    |round(exact) - exact| + 2 |y - exact|. The latter, relative to weights times values: a weight as two numbers of 16
    bits, 2^-16; the score, the maximum and their difference, up to 6 in size, and exp2, 32 2^-24; the fp32 sums, a lane's
    n / 32 terms and the matrix unit's n / 64 steps of two products, which may cut instead of round, and 32 more for
    the sums of lanes, warps and parts; the same again for the normaliser."""
    out, want = two_kinds_of_keys(cuda, [-i / 16 for i in range(64)], n, bits, dtype, dim, heads=heads)
    y = 2.0 ** -16 + 2 * (64 + n / 32 + 4 * n / 64) * 2.0 ** -24
    allowed = (want.to(dtype).double() - want).abs() + 2 * y * want.abs()
    off = (out.double() - want).abs()
    assert not (off > allowed).any(), float((off / allowed).max())
    assert T.attention_status(cuda) == 0


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_many_small_weights_count(cuda, dtype, bits):
    """4096 keys of weights around 2^-26 beside one of 1. fp16 operands lose what is below 2^-32 of a key, half of the
    smallest step of them below the scale of 2^7: 4096 2^-32 of the values. Errors as above, scores up to 20 in size."""
    n = 4097
    out, want = two_kinds_of_keys(cuda, [-17.0, -18.0, -18.5, -19.0], n, bits, dtype, big=1024.0)
    y = 2.0 ** -16 + 2 * (256 + n / 32 + 4 * n / 64) * 2.0 ** -24
    allowed = (want.to(dtype).double() - want).abs() + 2 * y * want.abs() + n * 2.0 ** -32 * 1024.0
    off = (out.double() - want).abs()
    assert not (off > allowed).any(), float((off / allowed).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("window", [None, (5, 0)], ids=str)
@pytest.mark.parametrize("Sq,heads,dim", [(3, 1, 64), (4, 2, 128), (9, 4, 64), (2, 4, 128), (5, 6, 128)])
def test_values_that_a_query_does_not_see_may_be_anything(cuda, Sq, heads, dim, window, dtype):
    """16 bits: an infinite value or one that is not a number counts for the queries that see its key, and for no other
    one of the same tile: those of earlier drafted tokens, those that a window has left it behind."""
    lengths, page = [50, 37, 16, 400], 16
    c = make_cache(lengths, 1, page, dim, 16, dtype, cuda)
    q = torch.randn(len(lengths), Sq, heads, dim, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(dtype)
    call = dict(lengths=i32(lengths, cuda), window=window)
    want = T.attention_paged(q, **c, **call)
    rows = torch.arange(Sq)
    for bad in (float("nan"), float("inf"), float("-inf")):
        for back in (1, 2, Sq + 4):  # the last key, the one before it, one that a window of 5 has left behind for the last query
            now = {n: t.clone() for n, t in c.items()}
            for b, n in enumerate(lengths):
                at = n - back
                now["v_pages"][int(c["block_table"][b, at // page]), 0, at % page, 3] = bad
            got = T.attention_paged(q, **now, **call)
            for b, n in enumerate(lengths):
                here = rows + n - Sq
                sees = (n - back <= here) & ((n - back >= here - 5) if window else True)
                assert torch.equal(got[b, ~sees], want[b, ~sees])
                assert torch.equal(got[b, sees][..., :3], want[b, sees][..., :3])
                hit = got[b, sees][..., 3]
                assert hit.isnan().all() if bad != bad else (hit == bad).all()
    assert T.attention_status(cuda) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("heads,n", [(1, 5), (4, 300), (7, 300), (24, 300), (4, 20000), (7, 20000)])
def test_infinite_values_stay_infinite(cuda, heads, n, dtype):
    c = make_cache([n], 1, 16, 64, 16, dtype, cuda)
    q = torch.randn(1, 1, heads, 64, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(dtype) / 8
    want = T.attention_paged(q, **c, lengths=i32([n], cuda))
    for bad, at in ((float("inf"), 0), (float("-inf"), n - 1), (float("inf"), n // 2)):
        v = c["v_pages"][int(c["block_table"][0, at // 16]), 0, at % 16]
        held = v.clone()
        v[7] = bad
        got = T.attention_paged(q, **c, lengths=i32([n], cuda))
        v.copy_(held)
        assert (got[..., 7] == bad).all()
        got[..., 7] = want[..., 7]
        assert torch.equal(got, want)


@pytest.mark.parametrize("bits", [16, 4])
def test_a_window_beyond_all_keys(cuda, bits):
    lengths = [9000, 3, 700]
    c = make_cache(lengths, 2, 64, 64, bits, torch.float16, cuda)
    q = torch.randn(3, 2, 4, 64, device=cuda).half()
    want = T.attention_paged(q, **c, lengths=i32(lengths, cuda))
    for left in (1 << 20, 1 << 40, 2 ** 63 - 1, 2 ** 64, 2 ** 64 + 1):
        assert torch.equal(T.attention_paged(q, **c, lengths=i32(lengths, cuda), window=(left, 0)), want)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("Sq,heads,dtype", [(1, 8, torch.bfloat16), (3, 12, torch.float16)], ids=str)
@pytest.mark.parametrize("B,width", [(3, 30), (3, 700), (3, 1 << 16), (16, 40), (16, 200), (16, 1000), (64, 60), (64, 512)])
def test_tables_wider_than_the_sequences(cuda, B, width, Sq, heads, dtype, bits):
    """How a call is cut goes by what the table has room for: short sequences in tables of all widths."""
    g = torch.Generator().manual_seed(B + width)
    lengths = torch.randint(0, 400, (B,), generator=g).tolist()
    lengths[1], lengths[2] = 0, 470
    c = make_cache(lengths, 2, 16, 64, bits, dtype, cuda)
    narrow = c["block_table"]
    c["block_table"] = torch.full((B, width), -1, dtype=torch.int32, device=cuda)
    c["block_table"][:, : narrow.shape[1]] = narrow
    q = torch.randn(B, Sq, heads, 64, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda).to(dtype)
    out, lse = T.attention_paged(q, **c, lengths=i32(lengths, cuda), return_lse=True)
    some = [0, 1, 2, B - 1]
    few = {**c, "block_table": narrow[some]}
    check_attention(out[some], lse[some], q[some], few, [lengths[b] for b in some], bits)
    assert T.attention_status(cuda) == 0
