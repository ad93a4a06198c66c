"""The paged cache of keys and values, in 16 and in 4 bits: appending, reading back, attention over it, and all of
it together, against the definition in 64 bits."""
import itertools

import pytest
import torch

import trinix_b200 as T
from tests.paged_ref import FIFTEENTH, attend_codes, codes_of, make_cache, rows_of, scales_of
from tests.ragged_ref import assert_within, attend64

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def starts(sizes, dev):
    return i32([0, *itertools.accumulate(sizes)], dev)


def tables(rows, dim, dev, dtype=torch.float32):
    rate = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * rate
    return angle.cos().to(dev, dtype), angle.sin().to(dev, dtype)


def turned(x, cos, sin):
    """fp32, as the elementwise formula rounds: x (rows, heads, D), cos and sin (rows, D / 2)."""
    x, h = x.float(), x.shape[-1] // 2
    x1, x2, c, s = x[..., :h], x[..., h:], cos.float()[:, None, :h], sin.float()[:, None, :h]
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)


def slopes_of(heads, dev):
    return 2.0 ** (-8.0 * torch.arange(1, heads + 1, device=dev) / heads)


def quantised(x):
    """(codes, step, lowest) of fp32 rows, with the divisions and products in fp32 that the format names."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    span = high - low
    bad, none = ~(span <= 2.0 ** 120), span < 2.0 ** -76
    code = ((x - low) * 15.0 / torch.where(none | bad, torch.ones_like(span), span)).round()
    code = torch.where(none | bad, torch.zeros_like(code), code)
    step = torch.where(none, torch.zeros_like(span), span * FIFTEENTH)
    nan = torch.full_like(span, float("nan"))
    return code.to(torch.uint8), torch.where(bad, nan, step), torch.where(bad, nan, low)


# ------------------------------------------------------------------------------- append
def check_append(c, before, k, v, new, lengths, cos, sin, bits, limit=None):
    """Every page of the cache after an append of `new` packed tokens of each sequence: written rows and all others."""
    size, pages = c["k_pages"].shape[2], c["k_pages"].shape[0]
    want = {n: t.clone() for n, t in before.items()}
    row = 0
    places = []
    for b, (n, m) in enumerate(zip(new, lengths)):
        for i in range(n):
            p = m - n + i
            if 0 <= p and p // size < c["block_table"].shape[1] and (limit is None or p < limit):
                page = int(c["block_table"][b, p // size])
                if 0 <= page < pages:
                    places.append((row + i, p, page, p % size))
        row += n
    if places:
        r, p, page, slot = (torch.tensor(t, device=k.device) for t in zip(*places))
        for x, rows in (("k", k), ("v", v)):
            rows = rows[r]
            rows = turned(rows, cos[p], sin[p]) if x == "k" and cos is not None else rows.float()
            if bits == 16:
                want[x + "_pages"][page, :, slot] = rows.to(k.dtype)
            else:
                code, step, low = quantised(rows)
                want[x + "_pages"][page, :, slot] = code[..., 0::2] | code[..., 1::2] << 4
                want[x + "_scales"][page, :, slot] = torch.cat((step, low), dim=-1)
    for n in want:
        if n != "block_table":
            same = (c[n] == want[n]) | (c[n].isnan() & want[n].isnan()) if c[n].is_floating_point() else c[n] == want[n]
            assert same.all(), (n, int((~same).sum()))


NEW = [([1], [1]), ([1], [33]), ([5], [5]), ([3, 3], [40, 3]), ([1] * 40, list(range(1, 41))), ([130], [300])]
PACKED = [([0, 5, 0, 1, 17], [9, 5, 0, 70, 17]), ([200, 1], [200, 90])]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("size", [16, 48, 256])
@pytest.mark.parametrize("new,lengths", NEW + PACKED, ids=str)
@pytest.mark.parametrize("heads,kv,dim,dtype", [(4, 1, 64, torch.float16), (10, 5, 128, torch.bfloat16),
                                                (32, 8, 128, torch.float16)])
def test_append(cuda, heads, kv, dim, dtype, new, lengths, size, bits):
    packed = len(set(new)) > 1 or len(new) == 1 and size == 48
    c = make_cache(lengths, kv, size, dim, bits, dtype, cuda)
    before = {n: t.clone() for n, t in c.items()}
    g = torch.Generator(device=cuda).manual_seed(7)
    make = lambda h: torch.randn(sum(new), h, dim, generator=g, device=cuda).to(dtype)  # noqa: E731
    q, k, v = make(heads), make(kv), make(kv)
    cos, sin = tables(max(lengths), dim, cuda)
    cu = starts(new, cuda) if packed else None
    shape = (lambda t: t) if packed else (lambda t: t.view(len(new), new[0], *t.shape[1:]))
    out = T.append_paged(shape(k), shape(v), **c, lengths=i32(lengths, cuda), cos=cos, sin=sin, q=shape(q), cu_seqlens=cu)
    check_append(c, before, k, v, new, lengths, cos, sin, bits)
    at = torch.cat([torch.arange(m - n, m) for n, m in zip(new, lengths)]).to(cuda)
    assert torch.equal(out.view_as(q), turned(q, cos[at], sin[at]).to(dtype))


@pytest.mark.parametrize("bits", [16, 4])
def test_append_without_rotation_and_queries(cuda, bits):
    c = make_cache([20, 7], 2, 32, 64, bits, torch.bfloat16, cuda)
    before = {n: t.clone() for n, t in c.items()}
    k, v = (torch.randn(2, 4, 2, 64, device=cuda).bfloat16() for _ in range(2))
    assert T.append_paged(k, v, **c, lengths=i32([20, 7], cuda)) is None
    check_append(c, before, k.flatten(0, 1), v.flatten(0, 1), [4, 4], [20, 7], None, None, bits)


@pytest.mark.parametrize("bits", [16, 4])
def test_append_of_tokens_without_a_place(cuda, bits):
    """Padded sequences, positions behind the block table, behind the rotation tables, pages that are none, rows
    behind the last packed sequence: nothing is written for them, and their queries are 0."""
    lengths, new = [0, 2, 70, 33, 64, 6], [1, 4, 3, 2, 2, 2]
    c = make_cache([1, 2, 48, 33, 64, 6], 2, 16, 64, bits, torch.float16, cuda)  # the table holds 64 positions
    c["block_table"][3, 2] = c["k_pages"].shape[0]
    c["block_table"][5, 0] = -7
    before = {n: t.clone() for n, t in c.items()}
    rows = sum(new) + 5
    g = torch.Generator(device=cuda).manual_seed(7)
    k, v, q = (torch.randn(rows, h, 64, generator=g, device=cuda).half() for h in (2, 2, 4))
    cos, sin = tables(63, 64, cuda)
    out = T.append_paged(k, v, **c, lengths=i32(lengths, cuda), cos=cos, sin=sin, q=q, cu_seqlens=starts(new, cuda))
    check_append(c, before, k, v, new, lengths, cos, sin, bits, limit=63)
    at = [m - n + i for n, m in zip(new, lengths) for i in range(n)]
    there = [0 <= p < 63 and 0 <= int(c["block_table"][b, p // 16]) < c["k_pages"].shape[0]
             for p, b in zip(at, [b for b, n in enumerate(new) for _ in range(n)])]
    assert sum(there) == 4  # positions 0, 1; none of 67 .. 69; 31; 62; none
    for i in range(rows):
        if i < len(at) and there[i]:
            assert torch.equal(out[i], turned(q[i:i + 1], cos[at[i]][None], sin[at[i]][None])[0].half())
        else:
            assert not out[i].any()


def test_four_bits_at_their_borders(cuda):
    """Halfway values, one value, neighbours of zero, the largest numbers, what is not finite; values are within half
    a step of what was put in, the smallest and the largest exactly codes 0 and 15."""
    rows = torch.zeros(14, 1, 64)
    rows[0] = torch.arange(64) % 31 / 2           # halves of a step of 1: to even
    rows[1] = -rows[0]
    rows[2] = 3.25                                # one value
    rows[4] = 2.0 ** -24 * (torch.arange(64) % 2)
    rows[5] = torch.linspace(-65000, 65000, 64)
    rows[6] = torch.randn(64, generator=torch.Generator().manual_seed(0))
    rows[7, 0, 63] = 1.0                          # one that differs
    rows[8, 0, 0] = -1.0
    rows[9] = torch.randn(64, generator=torch.Generator().manual_seed(1)) + 1000.0
    rows[10] = rows[6]
    rows[10, 0, 5] = float("nan")
    rows[11] = rows[6]
    rows[11, 0, 40] = float("inf")
    rows[12] = rows[6]
    rows[12, 0, 9] = float("-inf")
    rows[13] = float("inf")
    for dtype in (torch.float16, torch.bfloat16):
        x = rows.to(cuda, dtype)
        c = make_cache([14], 1, 16, 64, 4, dtype, cuda, spare=0)
        T.append_paged(x[None], x[None], **c, lengths=i32([14], cuda))
        code, step, low = quantised(x.float())
        page = int(c["block_table"][0, 0])
        for n in "kv":
            assert torch.equal(codes_of(c[n + "_pages"][page, 0, :14]), code[:, 0])
            held = c[n + "_scales"][page, 0, :14]
            assert torch.equal(held.nan_to_num(7.0), torch.cat((step, low), -1)[:, 0].nan_to_num(7.0))
            assert held[10:].isnan().all() and held[:10].isfinite().all()
        k, _ = T.gather_paged(**c, cu_seqlens=i32([0, 14], cuda), rows=14, dtype=dtype)
        assert k[10:].isnan().all()
        value = low + code.float() * step
        # half a step, its and the sum's roundings in 32 bits (4 2^-24 of 16 steps or of lowest), one to the type
        allowed = step / 2 + 64 * F32 * (step + low.abs()) + torch.finfo(dtype).eps / 2 * value.abs() + 2.0 ** -76
        assert ((k.float() - x.float()).abs() <= allowed)[:10].all()
        assert torch.equal(k[:10], value[:10].to(dtype))


def test_bf16_rows_beyond_the_format_are_nan(cuda):
    x = torch.zeros(3, 1, 64, device=cuda, dtype=torch.bfloat16)
    x[0, 0, 0], x[0, 0, 1], x[1, 0, 0], x[2, 0, 0] = 3e38, -3e38, 2.0 ** 121, 2.0 ** 120
    c = make_cache([3], 1, 16, 64, 4, x.dtype, cuda, spare=0)
    T.append_paged(x[None], x[None], **c, lengths=i32([3], cuda))
    k, _ = T.gather_paged(**c, cu_seqlens=i32([0, 3], cuda), rows=3)
    assert k[:2].isnan().all() and k[2, 0, 0] == 2.0 ** 120 and not k[2, 0, 1:].any()


def test_append_strides_and_tables(cuda):
    """Views of one projection, one tensor of keys' and values' pages, tables of the activation's type and odd rows,
    inputs that have to be copied, a block table wider than its rows."""
    B, S, Hq, Hk, D, size = 3, 5, 6, 2, 64, 32
    lengths = [5, 70, 33]
    for dtype, table_dtype, columns in ((torch.bfloat16, torch.bfloat16, D), (torch.float16, torch.float32, 33)):
        for odd in (0, 1):
            qkv = torch.randn(B, S, (Hq + 2 * Hk) * D + odd, device=cuda).to(dtype)[..., odd:].view(B, S, -1, D)
            q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
            both = torch.zeros(12, 2, Hk, size, D, device=cuda, dtype=dtype)
            wide = torch.full((B, 9), -1, dtype=torch.int32, device=cuda)
            wide[:, :3] = torch.arange(9, device=cuda).view(3, 3).int()
            c = {"k_pages": both[:, 0], "v_pages": both[:, 1], "block_table": wide[:, :3]}
            before = {n: t.clone() for n, t in c.items()}
            cos, sin = tables(96, D, cuda, table_dtype)
            cos, sin = (torch.cat((t, t), -1)[:, :columns] for t in (cos, sin))
            out = T.append_paged(k, v, **c, lengths=i32(lengths, cuda), cos=cos, sin=sin, q=q)
            check_append(c, before, k.flatten(0, 1), v.flatten(0, 1), [S] * B, lengths, cos, sin, 16)
            at = torch.cat([torch.arange(m - S, m) for m in lengths]).to(cuda)
            assert torch.equal(out.flatten(0, 1), turned(q.flatten(0, 1), cos[at], sin[at]).to(dtype))


def test_append_nothing(cuda):
    c = make_cache([3], 2, 16, 64, 16, torch.float16, cuda)
    before = {n: t.clone() for n, t in c.items()}
    cos, sin = tables(4, 64, cuda)
    empty = lambda *s: torch.zeros(*s, device=cuda, dtype=torch.float16)  # noqa: E731
    T.append_paged(empty(1, 0, 2, 64), empty(1, 0, 2, 64), **c, lengths=i32([3], cuda))
    none = {**c, "block_table": c["block_table"][:0]}
    T.append_paged(empty(0, 2, 2, 64), empty(0, 2, 2, 64), **none, lengths=i32([], cuda))
    out = T.append_paged(empty(4, 2, 64), empty(4, 2, 64), **none, lengths=i32([], cuda), cos=cos, sin=sin,
                         q=empty(4, 4, 64) + 1, cu_seqlens=i32([0], cuda))
    assert out.shape == (4, 4, 64) and not out.any()
    assert all(torch.equal(c[n], before[n]) for n in c)


# ------------------------------------------------------------------------------- gather
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,size,dim,lengths", [(1, 16, 64, [1]), (5, 48, 128, [0, 100, 0, 3, 48]),
                                                    (8, 64, 128, [700, 64, 65])], ids=str)
def test_gather(cuda, heads, size, dim, lengths, dtype, bits):
    c = make_cache(lengths, heads, size, dim, bits, dtype, cuda)
    c["block_table"][-1, 0] = -1  # rows of zeros
    rows = sum(lengths) + 4
    k, v = T.gather_paged(**c, cu_seqlens=starts(lengths, cuda), rows=rows, dtype=dtype)
    for x, got in (("k", k), ("v", v)):
        at = 0
        for b, n in enumerate(lengths):
            values, step, low = rows_of(c, x, b, n)
            if bits == 4:  # in fp32, as the format has it
                code = ((values - low) / step.clamp(min=1e-30)).round().float()
                values = low.float() + code * step.float()
            assert torch.equal(got[at:at + n], values.to(dtype))
            at += n
        assert not got[at:].any()


# ------------------------------------------------------------------------------- attention
def check_attention(out, lse, q, c, lengths, bits, **how):
    for b, n in enumerate(lengths):
        k, v = rows_of(c, "k", b, n), rows_of(c, "v", b, n)
        if bits == 4:
            want, want_lse, allowed, allowed_lse = attend_codes(q[b], k, v, **how)
        else:
            want, want_lse, allowed, allowed_lse = attend64(q[b], k[0].to(q.dtype), v[0].to(q.dtype), causal=True, **{
                **how, "window": (how["window"][0], 1 << 20) if how.get("window") else None})
        assert_within(out[b], want, allowed, f"sequence {b} of {n}")
        if lse is not None:
            assert_within(lse[b], want_lse, allowed_lse, f"lse of sequence {b} of {n}")


def attention_case(cuda, lengths, Sq, heads, kv, size, dim, bits, dtype, seed=0, **how):
    c = make_cache(lengths, kv, size, dim, bits, dtype, cuda, seed)
    g = torch.Generator(device=cuda).manual_seed(seed + 11)
    q = torch.randn(len(lengths), Sq, heads, dim, generator=g, device=cuda).to(dtype)
    out, lse = T.attention_paged(q, **c, lengths=i32(lengths, cuda), return_lse=True,
                                 **{n if n != "slopes" else "alibi_slopes": x for n, x in how.items()})
    assert T.attention_status(cuda) == 0
    check_attention(out, lse, q, c, lengths, bits, **how)
    return q, c, out, lse


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lengths", [[1], [15], [16], [17], [33], [127, 128, 129, 1, 31, 64, 200, 0], [700], [5] * 40,
                                     [1, 2000, 3]], ids=str)
@pytest.mark.parametrize("heads,kv,dim,dtype", [(1, 1, 128, torch.bfloat16), (8, 2, 64, torch.float16),
                                                (32, 8, 128, torch.bfloat16), (16, 1, 128, torch.float16),
                                                (10, 2, 64, torch.bfloat16)])
def test_attention_of_one_token(cuda, heads, kv, dim, dtype, lengths, bits):
    attention_case(cuda, lengths, 1, heads, kv, 16 if len(lengths) > 1 else 64, dim, bits, dtype)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("Sq", [2, 5, 8, 16, 33, 70])
@pytest.mark.parametrize("heads,kv", [(1, 1), (6, 2), (9, 1), (24, 1)])
def test_attention_of_several_tokens(cuda, heads, kv, Sq, bits):
    """Some sequences have fewer keys than queries: the first of these see none."""
    attention_case(cuda, [Sq, 3, 300, Sq + 31, 0, 97], Sq, heads, kv, 48, 64, bits, torch.bfloat16)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("Sq", [1, 7])
@pytest.mark.parametrize("how", [dict(window=(0, 0)), dict(window=(20, 5)), dict(window=(300, 0)), dict(alibi=True),
                                 dict(window=(100, 0), alibi=True), dict(scale=0.7), dict(scale=-0.05), dict(scale=0.0)],
                         ids=str)
def test_window_alibi_and_scale(cuda, how, Sq, dim, bits):
    how = dict(how)
    if how.pop("alibi", False):
        how["slopes"] = slopes_of(6, cuda)
    attention_case(cuda, [400, 7, 64, 150], Sq, 6, 2, 32, dim, bits, torch.float16, **how)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("batch,longest", [(1, 9000), (2, 20000), (3, 4097), (150, 300)])
def test_splits(cuda, batch, longest, bits):
    """Keys over all CTAs of a cluster, one sequence beside many."""
    lengths = [longest] + [max(1, longest // (i + 2) - i) for i in range(batch - 1)]
    c = make_cache(lengths, 2, 64, 128, bits, torch.bfloat16, cuda)
    q = torch.randn(batch, 1, 8, 128, device=cuda).bfloat16()
    out, lse = T.attention_paged(q, **c, lengths=i32(lengths, cuda), return_lse=True)
    cu = starts(lengths, cuda)
    k, v = T.gather_paged(**c, cu_seqlens=cu, rows=sum(lengths))
    at = cu.tolist()
    for b in range(0, batch, 1 if batch < 10 else 29):
        if bits == 16:
            want, want_lse, allowed, allowed_lse = attend64(q[b], k[at[b]:at[b + 1]], v[at[b]:at[b + 1]], causal=True)
        else:
            pages = c["block_table"][b, : -(-lengths[b] // 64)].long()
            def held(x):
                s = c[x + "_scales"][pages].transpose(1, 2).flatten(0, 1)[:lengths[b]].double()
                code = codes_of(c[x + "_pages"][pages].transpose(1, 2).flatten(0, 1)[:lengths[b]]).double()
                return s[..., 1:] + code * s[..., :1], s[..., :1], s[..., 1:]
            want, want_lse, allowed, allowed_lse = attend_codes(q[b], held("k"), held("v"))
        assert_within(out[b], want, allowed, f"sequence {b}")
        assert_within(lse[b], want_lse, allowed_lse, f"lse of sequence {b}")


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("Sq", [1, 4])
def test_what_lies_behind_the_last_key_is_not_used(cuda, Sq, bits):
    """Rows behind a sequence's last key, on its last page and beyond, may be NaN or infinite."""
    lengths = [5, 50, 31, 0]
    c = make_cache(lengths, 2, 32, 128, bits, torch.bfloat16, cuda)
    q = torch.randn(4, Sq, 8, 128, device=cuda).bfloat16()
    args = dict(lengths=i32(lengths, cuda), return_lse=True)
    want = T.attention_paged(q, **c, **args)
    for poison in (float("nan"), float("inf"), float("-inf")):
        for x in "kv":
            t = c[x + ("_scales" if bits == 4 else "_pages")]
            used = torch.zeros(t.shape[0], t.shape[2], dtype=torch.bool, device=cuda)
            for b, n in enumerate(lengths):
                for p in range(n):
                    used[int(c["block_table"][b, p // 32]), p % 32] = True
            t.masked_fill_(~used[:, None, :, None], poison)
        got = T.attention_paged(q, **c, **args)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert not want[0][3].any() and torch.isneginf(want[1][3]).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_pages_that_are_none(cuda, bits):
    """A page number outside the cache reads as zeros, wherever it stands; behind the window it does not matter."""
    lengths = [200, 70, 33]
    c = make_cache(lengths, 2, 16, 64, bits, torch.float16, cuda)
    c["block_table"][0, 3], c["block_table"][1, 0] = -1, c["k_pages"].shape[0]
    c["block_table"][2] = 2 ** 31 - 1
    q = torch.randn(3, 2, 4, 64, device=cuda).half()
    out, lse = T.attention_paged(q, **c, lengths=i32(lengths, cuda), return_lse=True)
    check_attention(out, lse, q, c, lengths, bits)
    full = make_cache(lengths, 2, 16, 64, bits, torch.float16, cuda, seed=4)
    want = T.attention_paged(q, **full, lengths=i32(lengths, cuda), window=(20, 0))
    for b, n in enumerate(lengths):
        full["block_table"][b, : max(0, n - 2 - 20) // 16] = -1
    assert torch.equal(T.attention_paged(q, **full, lengths=i32(lengths, cuda), window=(20, 0)), want)


@pytest.mark.parametrize("bits", [16, 4])
def test_lengths_beyond_the_table(cuda, bits):
    """Are cut to what the table holds; negative ones are 0."""
    lengths = [64, 20, 0]
    c = make_cache(lengths, 1, 16, 64, bits, torch.float16, cuda)
    q = torch.randn(3, 1, 2, 64, device=cuda).half()
    want = T.attention_paged(q, **c, lengths=i32(lengths, cuda))
    assert torch.equal(T.attention_paged(q, **c, lengths=i32([2 ** 31 - 1, 20, -5], cuda)), want)


def test_steps_of_very_different_sizes(cuda):
    """Values whose steps span 2^40, steps of 0 among them, keys of one value, queries of very different sizes."""
    c = make_cache([90, 40], 1, 16, 64, 4, torch.bfloat16, cuda)
    s = c["v_scales"]
    s.mul_(2.0 ** torch.randint(-20, 20, s.shape[:3], generator=torch.Generator().manual_seed(1)).float().to(cuda)[..., None])
    s[..., 0][:, :, ::5] = 0
    c["k_scales"][..., 0][:, :, ::7] = 0
    for zero in (s, c["k_scales"]):
        codes = c["v_pages"] if zero is s else c["k_pages"]
        codes.masked_fill_((zero[..., :1] == 0), 0)
    q = torch.randn(2, 3, 5, 64, device=cuda)
    q = (q * 2.0 ** torch.tensor([0, -30, 3, -100, 1.0], device=cuda)[:, None]).bfloat16()
    out, lse = T.attention_paged(q, **c, lengths=i32([90, 40], cuda), return_lse=True)
    check_attention(out, lse, q, c, [90, 40], 4)


def test_queries_and_keys_that_are_not_finite_stay_in_their_rows(cuda):
    for bits in (16, 4):
        c = make_cache([50, 60], 2, 16, 128, bits, torch.bfloat16, cuda)
        q = torch.randn(2, 2, 4, 128, device=cuda).bfloat16()
        want = T.attention_paged(q, **c, lengths=i32([50, 60], cuda))
        q[0, 1, 2, 5] = float("nan")
        got = T.attention_paged(q, **c, lengths=i32([50, 60], cuda))
        assert got[0, 1, 2].isnan().all()
        got[0, 1, 2] = want[0, 1, 2]
        assert torch.equal(got, want)
    # the last key's row of a 4-bit cache is not a number: the queries before it do not see it
    page, slot = int(c["block_table"][1, 59 // 16]), 59 % 16
    for x in "kv":
        held = c[x + "_scales"][page, 1, slot].clone()
        c[x + "_scales"][page, 1, slot] = float("nan")
        got = T.attention_paged(q, **c, lengths=i32([50, 60], cuda))
        assert got[1, 1, 2:].isnan().all()
        assert torch.equal(got[1, 0], want[1, 0]) and torch.equal(got[1, 1, :2], want[1, 1, :2])
        c[x + "_scales"][page, 1, slot] = held


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_strides(cuda, bits):
    """Keys' and values' pages in one tensor, queries as views, a wider block table, more pages than are used."""
    lengths = [70, 20]
    c = make_cache(lengths, 2, 16, 64, bits, torch.bfloat16, cuda)
    both = torch.stack((c["k_pages"], c["v_pages"]), dim=1)
    wide = torch.cat((c["block_table"], c["block_table"]), dim=1)
    view = {**c, "k_pages": both[:, 0], "v_pages": both[:, 1], "block_table": wide[:, :c["block_table"].shape[1]]}
    if bits == 4:
        scales = torch.stack((c["k_scales"], c["v_scales"]), dim=2)
        view |= {"k_scales": scales[:, :, 0], "v_scales": scales[:, :, 1]}
    q = torch.randn(2, 3, 8, 64, device=cuda).bfloat16()
    want = T.attention_paged(q, **c, lengths=i32(lengths, cuda))
    odd = torch.zeros(2, 3, 8, 65, device=cuda, dtype=q.dtype)[..., 1:].copy_(q)
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    for qq in (q, odd, swapped):
        assert torch.equal(T.attention_paged(qq, **view, lengths=i32(lengths, cuda)), want)


@pytest.mark.parametrize("bits", [16, 4])
def test_a_long_cache(cuda, bits):
    """Pages whose offsets pass 32 bits: 2^31 elements are before the last ones."""
    size, heads, dim = 4096, 8, 128
    pages = 2 ** 31 // (size * heads * (dim if bits == 16 else dim // 2)) + 3
    small = make_cache([300], heads, 4096, dim, bits, torch.bfloat16, cuda, spare=2)
    big = {"block_table": i32([[pages - 1]], cuda)}
    for n, t in small.items():
        if n != "block_table":
            big[n] = torch.empty(pages, *t.shape[1:], dtype=t.dtype, device=cuda)
            big[n][pages - 1] = t[int(small["block_table"][0, 0])]
    q = torch.randn(1, 1, 8, dim, device=cuda).bfloat16()
    k, v = (torch.randn(1, 1, heads, dim, device=cuda).bfloat16() for _ in range(2))
    for c in (small, big):
        T.append_paged(k, v, **c, lengths=i32([301], cuda))
    n = i32([301], cuda)
    assert torch.equal(T.attention_paged(q, **small, lengths=n), T.attention_paged(q, **big, lengths=n))
    cu = i32([0, 301], cuda)
    for x, y in zip(T.gather_paged(**small, cu_seqlens=cu, rows=301), T.gather_paged(**big, cu_seqlens=cu, rows=301)):
        assert torch.equal(x, y)


def test_nothing_to_attend_to(cuda):
    c = make_cache([3, 4], 2, 16, 64, 4, torch.float16, cuda)
    q = torch.randn(2, 0, 4, 64, device=cuda).half()
    assert T.attention_paged(q, **c, lengths=i32([3, 4], cuda)).shape == q.shape
    none = {**c, "block_table": c["block_table"][:0]}
    assert T.attention_paged(q[:0], **none, lengths=i32([], cuda)).shape == (0, 0, 4, 64)
    narrow = {**c, "block_table": c["block_table"][:, :0]}
    q = torch.randn(2, 1, 4, 64, device=cuda).half()
    out, lse = T.attention_paged(q, **narrow, lengths=i32([3, 4], cuda), return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()


# ------------------------------------------------------------------------------- together
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("captured", [False, True])
def test_a_batch_served_from_prompts_to_tokens(cuda, bits, captured):
    """Prompts appended packed, then token after token, as one graph replayed where captured: each step's attention is
    that over what the cache holds, and the cache holds what was appended."""
    Hq, Hk, D, size, steps, dtype = 8, 2, 128, 16, 6, torch.bfloat16
    prompts = [30, 1, 47]
    full = [n + steps for n in prompts]
    c = make_cache(full, Hk, size, D, bits, dtype, cuda)
    cos, sin = tables(max(full), D, cuda)
    g = torch.Generator(device=cuda).manual_seed(5)
    make = lambda *s: torch.randn(*s, D, generator=g, device=cuda).to(dtype)  # noqa: E731
    q, k, v = (make(sum(prompts), h) for h in (Hq, Hk, Hk))
    lengths = i32(prompts, cuda)
    turned_q = T.append_paged(k, v, **c, lengths=lengths, cos=cos, sin=sin, q=q, cu_seqlens=starts(prompts, cuda))
    cu = starts(prompts, cuda)
    out = T.attention_packed(turned_q, *T.gather_paged(**c, cu_seqlens=cu, rows=sum(prompts)), cu, causal=True)
    at = 0
    for b, n in enumerate(prompts):
        kk, vv = (rows_of(c, x, b, n)[0].to(dtype) for x in "kv")
        want, _, allowed, _ = attend64(turned_q[at:at + n], kk, vv, causal=True)
        assert_within(out[at:at + n], want, allowed, f"prompt {b}")
        at += n
    tok = [torch.zeros(3, 1, h, D, dtype=dtype, device=cuda) for h in (Hq, Hk, Hk)]

    def step():
        lengths.add_(1)
        rotated = T.append_paged(tok[1], tok[2], **c, lengths=lengths, cos=cos, sin=sin, q=tok[0])
        return rotated, T.attention_paged(rotated, **c, lengths=lengths)

    if captured:
        saved = {n: t.clone() for n, t in c.items()}, lengths.clone()
        step()  # once before it is captured
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            static = step()
        for n in c:
            c[n].copy_(saved[0][n])
        lengths.copy_(saved[1])
    for i in range(steps):
        new = [make(3, 1, h) for h in (Hq, Hk, Hk)]
        for t, x in zip(tok, new):
            t.copy_(x)
        if captured:
            graph.replay()
            rotated, out = static
        else:
            rotated, out = step()
        now = [n + i + 1 for n in prompts]
        assert lengths.tolist() == now
        check_attention(out, None, rotated, c, now, bits)
        last = torch.tensor([n - 1 for n in now], device=cuda)
        assert torch.equal(rotated[:, 0], turned(new[0][:, 0], cos[last], sin[last]).to(dtype))
    assert T.attention_status(cuda) == 0


@pytest.mark.parametrize("bits", [16, 4])
def test_streams_and_threads(cuda, bits):
    """Two streams at once, each with a cache of its own, and one that is not the current device's default."""
    lengths = [900, 40, 333]
    caches = [make_cache(lengths, 2, 32, 128, bits, torch.bfloat16, cuda, seed=i) for i in range(2)]
    q = torch.randn(3, 1, 8, 128, device=cuda).bfloat16()
    n = i32(lengths, cuda)
    want = [T.attention_paged(q, **c, lengths=n) for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in caches]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(T.attention_paged(q, **caches[i], lengths=n))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


@pytest.mark.parametrize("bits", [16, 4])
def test_long_caches_captured_and_on_two_streams(cuda, bits):
    """Calls whose keys are cut into pieces for the whole chip: captured, replayed with other lengths (short ones, none
    at all), and two at once on streams of their own."""
    lengths = [9000, 40, 20000, 333, 1]
    c = make_cache(lengths, 2, 64, 128, bits, torch.bfloat16, cuda)
    q = torch.randn(5, 1, 8, 128, device=cuda).bfloat16()
    n = i32(lengths, cuda)
    T.attention_paged(q, **c, lengths=n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = T.attention_paged(q, **c, lengths=n, return_lse=True)
    for now in (lengths, [0] * 5, [5, 40, 1, 0, 1], [9000, 0, 1, 333, 0], [64, 40, 20000, 333, 1]):
        n.copy_(i32(now, cuda))
        graph.replay()
        want, want_lse = T.attention_paged(q, **c, lengths=n, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        for b, m in enumerate(now):
            assert bool(out[b].any()) == (m > 0) and bool(torch.isneginf(lse[b]).all()) == (m == 0)
    n.copy_(i32(lengths, cuda))
    other = torch.randn_like(q)
    want = T.attention_paged(q, **c, lengths=n), T.attention_paged(other, **c, lengths=n)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(T.attention_paged((q, other)[i], **c, lengths=n))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)
    assert T.attention_status(cuda) == 0


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("Sq,heads,kv", [(1, 8, 2), (3, 12, 2), (16, 4, 4), (40, 6, 1)])
def test_many_sequences_of_all_lengths(cuda, bits, Sq, heads, kv):
    """More sequences than threads look at at once, most of them short, in a cache that some fill far: whole units,
    units cut once and many times, and row tiles."""
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 200, (300,), generator=g).tolist()
    lengths[7], lengths[150], lengths[299] = 3000, 1501, 2500
    c = make_cache(lengths, kv, 16, 64, bits, torch.float16, cuda)
    q = torch.randn(300, Sq, heads, 64, device=cuda).half()
    out, lse = T.attention_paged(q, **c, lengths=i32(lengths, cuda), return_lse=True)
    # one sequence at a time, which is a call of its own kind
    for b in (0, 1, 7, 8, 127, 128, 129, 150, 200, 256, 298, 299):
        one = {**c, "block_table": c["block_table"][b:b + 1, : max(1, -(-lengths[b] // 16))].contiguous()}
        k, v = T.gather_paged(**one, cu_seqlens=i32([0, lengths[b]], cuda), rows=lengths[b], dtype=torch.float16)
        if bits == 16:
            want, want_lse, allowed, allowed_lse = attend64(q[b], k, v, causal=True)
        else:
            pages = one["block_table"][0, : -(-lengths[b] // 16)].long()

            def held(x):
                s = c[x + "_scales"][pages].transpose(1, 2).flatten(0, 1)[:lengths[b]].double()
                code = codes_of(c[x + "_pages"][pages].transpose(1, 2).flatten(0, 1)[:lengths[b]]).double()
                return s[..., 1:] + code * s[..., :1], s[..., :1], s[..., 1:]
            want, want_lse, allowed, allowed_lse = attend_codes(q[b], held("k"), held("v"))
        assert_within(out[b], want, allowed, f"sequence {b} of {lengths[b]}")
        assert_within(lse[b], want_lse, allowed_lse, f"lse of sequence {b} of {lengths[b]}")


def test_a_later_backward_says_so(cuda):
    c = make_cache([5], 2, 16, 64, 16, torch.float16, cuda)
    q = torch.randn(1, 1, 4, 64, device=cuda).half().requires_grad_()
    out = T.PagedAttentionKernel.apply(q, **c, lengths=i32([5], cuda))
    with pytest.raises(NotImplementedError):
        out.float().sum().backward()
