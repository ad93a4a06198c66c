"""Attention over packed sequences against the definition in 64 bits, one sequence at a time."""
import itertools

import pytest
import torch

import trinix_b200 as T
from tests.ragged_ref import assert_within, attend64

pytestmark = pytest.mark.gpu


def starts(sizes, dev, dtype=torch.int32):
    return torch.tensor([0, *itertools.accumulate(sizes)], dtype=dtype, device=dev)


def make(seed, dev, dtype, *shape):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=dev).to(dtype)


def slopes_of(heads, dev):
    return 2.0 ** (-8.0 * torch.arange(1, heads + 1, device=dev) / heads)


def check(out, lse, q, k, v, len_q, len_k, **how):
    """Every sequence of a packed call, and the rows behind the last one."""
    row = key = 0
    for s, (n, m) in enumerate(zip(len_q, len_k)):
        want, want_lse, allowed, allowed_lse = attend64(q[row:row + n], k[key:key + m], v[key:key + m],
                                                        **how)
        assert_within(out[row:row + n], want, allowed, f"sequence {s} ({n}, {m})")
        if lse is not None:
            assert_within(lse[:, row:row + n], want_lse, allowed_lse, f"lse of sequence {s}")
        row, key = row + n, key + m
    assert not out[row:].any()
    if lse is not None:
        assert torch.equal(lse[:, row:], torch.full_like(lse[:, row:], float("-inf")))


LENGTHS = [
    ([1], None), ([17], None), ([128], None), ([129], None), ([257], None), ([700], None),
    ([0], None), ([0, 5, 0, 1, 0], None), ([127, 128, 129, 1, 31, 33, 64, 200], None),
    ([3] * 40, None), ([1, 2, 600, 1, 4], None),
    # behind cached keys; single tokens; no keys at all; fewer keys than queries
    ([1, 1, 1], [1, 300, 129]), ([5, 130, 1], [5 + 250, 130 + 1, 128]), ([4, 0, 7], [0, 9, 0]),
    ([9, 140], [3, 20]), ([260], [1000]),
]


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (8, 2), (6, 2), (5, 5)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(cuda, lengths, heads, kv, causal):
    len_q, len_k = lengths[0], lengths[1] or lengths[0]
    dtype, dim = (torch.bfloat16, 128) if heads % 2 else (torch.float16, 64)
    q = make(1, cuda, dtype, sum(len_q) + 3, heads, dim)
    k, v = (make(i, cuda, dtype, sum(len_k), kv, dim) for i in (2, 3))
    cu_q, cu_k = starts(len_q, cuda), starts(len_k, cuda)
    out, lse = T.attention_packed(q, k, v, cu_q, None if lengths[1] is None else cu_k, causal=causal,
                                  return_lse=True)
    check(out, lse, q, k, v, len_q, len_k, causal=causal)


# every group size that leaves a tile of another shape: 1 head, all of them, some of them
@pytest.mark.parametrize("heads,kv", [(2, 1), (3, 1), (7, 1), (10, 2), (16, 1), (24, 1), (32, 8), (48, 1),
                                      (71, 1), (128, 1), (130, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_groups(cuda, heads, kv, dtype):
    lens = [200, 3, 64, 65]
    q = make(4, cuda, dtype, sum(lens), heads, 64)
    k, v = (make(i, cuda, dtype, sum(lens), kv, 64) for i in (5, 6))
    out, lse = T.attention_packed(q, k, v, starts(lens, cuda), causal=True, return_lse=True)
    check(out, lse, q, k, v, lens, lens, causal=True)


@pytest.mark.parametrize("dim", [64, 128, 80, 16, 100])
@pytest.mark.parametrize("how", [
    dict(window=(40, 0)), dict(window=(0, 0)), dict(window=(130, 70)), dict(causal=True, window=(64, 64)),
    dict(causal=True, alibi=True), dict(alibi=True), dict(window=(50, 0), alibi=True),
    dict(causal=True, scale=0.3), dict(causal=True, scale=-0.05), dict(scale=0.0), dict(scale=-0.1, alibi=True),
], ids=str)
def test_masks_and_biases(cuda, how, dim):
    how = dict(how)
    len_q, len_k = [150, 1, 300, 20], [150, 200, 290, 160]
    slopes = slopes_of(8, cuda) if how.pop("alibi", False) else None
    q = make(7, cuda, torch.bfloat16, sum(len_q), 8, dim)
    k, v = (make(i, cuda, torch.bfloat16, sum(len_k), 2, dim) for i in (8, 9))
    out, lse = T.attention_packed(q, k, v, starts(len_q, cuda), starts(len_k, cuda), return_lse=True,
                                  alibi_slopes=slopes, **how)
    check(out, lse, q, k, v, len_q, len_k, slopes=slopes, **how)


# rows of up to 16, promised: the kernel for decoding
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 128), (8, 2, 128), (32, 8, 64), (3, 1, 128), (71, 1, 64), (5, 5, 80)])
@pytest.mark.parametrize("how", [
    dict(causal=True), dict(), dict(window=(300, 0)), dict(window=(0, 0)), dict(causal=True, alibi=True),
    dict(alibi=True), dict(window=(40, 20), alibi=True), dict(causal=True, scale=-0.2),
], ids=str)
def test_few_rows(cuda, how, heads, kv, dim):
    how = dict(how)
    slopes = slopes_of(heads, cuda) if how.pop("alibi", False) else None
    len_q = [1, 16, 0, 3, 1, 7, 1, 2, 5, 1] * 2
    len_k = [1, 16, 9, 700, 3000, 2, 0, 129, 5, 64] * 2
    dtype = torch.float16 if heads % 2 else torch.bfloat16
    q = make(50, cuda, dtype, sum(len_q) + 21, heads, dim)
    k, v = (make(i, cuda, dtype, sum(len_k) + 30, kv, dim) for i in (51, 52))
    k[sum(len_k):], v[sum(len_k):] = float("nan"), float("inf")
    out, lse = T.attention_packed(q, k, v, starts(len_q, cuda), starts(len_k, cuda), return_lse=True,
                                  alibi_slopes=slopes, max_seqlen_q=16, **how)
    check(out, lse, q, k, v, len_q, len_k, slopes=slopes, **how)
    held = q.clone()
    T.attention_packed(q, k, v, starts(len_q, cuda), starts(len_k, cuda), alibi_slopes=slopes,
                       max_seqlen_q=16, out=held, **how)
    n = sum(len_q)
    assert torch.equal(held[:n], out[:n]) and torch.equal(held[n:], q[n:])


@pytest.mark.parametrize("how", [dict(causal=True), dict(), dict(window=(20, 0)), dict(causal=True, alibi=True)],
                         ids=str)
@pytest.mark.parametrize("most,heads", [(1, 8), (3, 8), (16, 2)])
def test_rows_beyond_the_announced_ones(cuda, how, most, heads):
    """A sequence of more rows than max_seqlen_q: its first rows are those of the whole sequence, the others
    stay as they were."""
    how = dict(how)
    slopes = slopes_of(heads, cuda) if how.pop("alibi", False) else None
    len_q, len_k = [most + 1, 1, most, 40, most + 5], [60, 9, 300, 40, 3]
    q = make(56, cuda, torch.bfloat16, sum(len_q), heads, 64)
    k, v = (make(i, cuda, torch.bfloat16, sum(len_k), 2, 64) for i in (57, 58))
    held = make(59, cuda, torch.bfloat16, *q.shape)
    out, lse = T.attention_packed(q, k, v, starts(len_q, cuda), starts(len_k, cuda), max_seqlen_q=most,
                                  alibi_slopes=slopes, return_lse=True, out=held.clone(), **how)
    row = key = 0
    for n, m in zip(len_q, len_k):
        want, want_lse, allowed, allowed_lse = attend64(q[row:row + n], k[key:key + m], v[key:key + m],
                                                        slopes=slopes, **how)
        done = min(n, most)
        assert_within(out[row:row + done], want[:done], allowed[:done], f"{n} rows")
        assert_within(lse[:, row:row + done], want_lse[:, :done], allowed_lse[:, :done], f"lse of {n} rows")
        assert torch.equal(out[row + done:row + n], held[row + done:row + n])
        row, key = row + n, key + m


def test_scales_next_to_nothing(cuda):
    """A ramp divided by the scale would not be finite."""
    lens = [40, 300]
    q = make(53, cuda, torch.bfloat16, 340, 4, 64)
    k, v = make(54, cuda, torch.bfloat16, 340, 4, 64), make(55, cuda, torch.bfloat16, 340, 4, 64)
    for scale in (1e-37, 1e-31, 1e-20):
        out, lse = T.attention_packed(q, k, v, starts(lens, cuda), causal=True, scale=scale, return_lse=True,
                                      alibi_slopes=slopes_of(4, cuda))
        check(out, lse, q, k, v, lens, lens, causal=True, scale=scale, slopes=slopes_of(4, cuda))


@pytest.mark.parametrize("alibi", [False, True])
def test_several_items_per_cta(cuda, alibi):
    """More work items than SMs: the items that a CTA takes behind its first one, skipped slots."""
    lens = [1000, 1, 0, 333, 5, 5, 5, 2048, 64, 0, 0, 700]
    slopes = slopes_of(32, cuda) if alibi else None
    q = make(10, cuda, torch.bfloat16, sum(lens) + 40, 32, 128)
    k, v = (make(i, cuda, torch.bfloat16, sum(lens), 8, 128) for i in (11, 12))
    out, lse = T.attention_packed(q, k, v, starts(lens, cuda), causal=True, return_lse=True,
                                  alibi_slopes=slopes)
    check(out, lse, q, k, v, lens, lens, causal=True, slopes=slopes)


# two tiles of heads of one item, each with the K and V tiles of its own kv head (or of the same one)
@pytest.mark.parametrize("heads,kv", [(16, 16), (4, 2), (48, 1), (20, 4), (24, 2), (6, 2), (3, 3)])
@pytest.mark.parametrize("how", [dict(causal=True), dict(), dict(window=(30, 0)), dict(causal=True, alibi=True)],
                         ids=str)
def test_short_sequences_of_two_heads(cuda, heads, kv, how):
    how = dict(how)
    slopes = slopes_of(heads, cuda) if how.pop("alibi", False) else None
    g = torch.Generator().manual_seed(heads)
    most = 128 // (heads // kv)
    len_q = torch.randint(0, most + 1, (70,), generator=g).tolist() + [most + 1, 300, 1, most]
    len_k = [n + m for n, m in zip(len_q, torch.randint(0, 400, (74,), generator=g).tolist())]
    dtype, dim = (torch.bfloat16, 128) if heads % 3 else (torch.float16, 64)
    q = make(40, cuda, dtype, sum(len_q) + 9, heads, dim)
    k, v = (make(i, cuda, dtype, sum(len_k) + 100, kv, dim) for i in (41, 42))
    k[sum(len_k):], v[sum(len_k):] = float("nan"), float("nan")
    out, lse = T.attention_packed(q, k, v, starts(len_q, cuda), starts(len_k, cuda), return_lse=True,
                                  alibi_slopes=slopes, **how)
    check(out, lse, q, k, v, len_q, len_k, slopes=slopes, **how)


def test_many_sequences(cuda):
    """The search for a block's sequence: over 1024 of them, most of a few rows, many empty."""
    g = torch.Generator().manual_seed(3)
    lens = [int(n) for n in torch.randint(0, 9, (3000,), generator=g)]
    q = make(13, cuda, torch.float16, sum(lens), 2, 64)
    k, v = (make(i, cuda, torch.float16, sum(lens), 1, 64) for i in (14, 15))
    out = T.attention_packed(q, k, v, starts(lens, cuda), causal=True)
    # one sequence after the other would take minutes: a block-diagonal causal order instead
    rows = torch.arange(sum(lens), device=cuda)
    seq = torch.searchsorted(starts(lens, cuda)[1:].long(), rows, right=True)
    for at in range(0, sum(lens), 2000):
        r = slice(at, min(sum(lens), at + 2000))
        hidden = (seq[r, None] != seq[None]) | (rows[None] > rows[r, None])
        for h in range(2):
            s = (q[r, h].double() @ k[:, 0].double().t() * 0.125).masked_fill(hidden, float("-inf"))
            want = torch.softmax(s, -1) @ v[:, 0].double()
            # at most 8 keys: |out| and A are below max|v|, weights are off by far less than a rounding
            assert float((out[r, h].double() - want).abs().max()) <= 2.01 * 2 ** -11 * float(v.abs().max())


def test_strided_views_and_out(cuda):
    """q, k, v as views of one projection, and an output with rows that belong to no sequence."""
    lens, hq, hk, d = [70, 200, 1], 8, 2, 128
    qkv = make(16, cuda, torch.bfloat16, sum(lens) + 5, (hq + 2 * hk), d)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    buf = make(17, cuda, torch.bfloat16, sum(lens) + 5, hq + 1, d)
    held = buf.clone()
    res, lse = T.attention_packed(q, k, v, starts(lens, cuda), causal=True, return_lse=True, out=buf[:, 1:])
    assert res.data_ptr() == buf[:, 1:].data_ptr()
    n = sum(lens)
    check(buf[:n, 1:], lse[:, :n], q, k, v, lens, lens, causal=True)
    assert torch.equal(buf[n:], held[n:]) and torch.equal(buf[:, 0], held[:, 0])
    assert torch.equal(lse[:, n:], torch.full_like(lse[:, n:], float("-inf")))
    # a layout that the kernel cannot take as it is: head dim 40 at an odd offset, expanded kv heads
    odd = make(18, cuda, torch.bfloat16, n + 5, hq, 43)[..., 3:]
    one = make(19, cuda, torch.bfloat16, n, 1, 40)
    kx = one.expand(-1, 4, -1)
    out2 = make(20, cuda, torch.bfloat16, n + 5, hq, 41)
    held = out2.clone()
    T.attention_packed(odd, kx, kx, starts(lens, cuda), out=out2[..., :40])
    check(out2[:n, :, :40], None, odd, kx, kx, lens, lens)
    assert torch.equal(out2[n:], held[n:]) and torch.equal(out2[..., 40:], held[..., 40:])


@pytest.mark.parametrize("max_q", [None, 4])
def test_neighbours_and_rest_never_matter(cuda, max_q):
    """What lies behind a sequence's last key is NaN or infinite: the next sequence, or nothing."""
    len_q, len_k = [4, 3, 1, 4], [140, 33, 260, 17]
    q = make(21, cuda, torch.bfloat16, sum(len_q), 4, 128)
    k, v = (make(i, cuda, torch.bfloat16, sum(len_k) + 90, 2, 128) for i in (22, 23))
    cu_q, cu_k = starts(len_q, cuda), starts(len_k, cuda)
    want = T.attention_packed(q, k, v, cu_q, cu_k, causal=True, max_seqlen_q=max_q)
    check(want, None, q, k, v, len_q, len_k, causal=True)
    for s in range(4):
        for bad in (float("nan"), float("inf")):
            kk, vv = k.clone(), v.clone()
            lo, hi = int(cu_k[s]), int(cu_k[s + 1])
            for t in (kk, vv):
                t[:lo], t[hi:] = bad, bad
            a, b = int(cu_q[s]), int(cu_q[s + 1])
            qq = torch.full_like(q, bad)
            qq[a:b] = q[a:b]
            got = T.attention_packed(qq, kk, vv, cu_q, cu_k, causal=True, max_seqlen_q=max_q)
            assert torch.equal(got[a:b], want[a:b])


def test_long_offsets(cuda):
    """Element offsets beyond 32 bits in the keys and in the output."""
    rows, hk, d = 2_200_000, 8, 128
    kv = torch.zeros(rows, hk, d, dtype=torch.bfloat16, device=cuda)  # 4.5 GB
    kv[-500:] = make(24, cuda, torch.bfloat16, 500, hk, d)
    q = make(25, cuda, torch.bfloat16, 9, hk, d)
    cu_q = torch.tensor([0, 1, 9], dtype=torch.int32, device=cuda)
    cu_k = torch.tensor([0, rows - 300, rows], dtype=torch.int32, device=cuda)
    for most in (None, 8):
        got = T.attention_packed(q[1:], kv, kv, cu_q[1:] - 1, cu_k[1:], max_seqlen_q=most)
        check(got, None, q[1:], kv[-300:], kv[-300:], [8], [300])
    del kv
    hq, rows = 32, 540_000
    q = torch.zeros(rows, hq, d, dtype=torch.bfloat16, device=cuda)  # 4.4 GB
    q[-70:] = make(26, cuda, torch.bfloat16, 70, hq, d)
    k = make(27, cuda, torch.bfloat16, 70, hk, d)
    cu_q = torch.tensor([0, rows - 70, rows], dtype=torch.int32, device=cuda)
    cu_k = torch.tensor([0, 0, 70], dtype=torch.int32, device=cuda)
    got = T.attention_packed(q, k, k, cu_q, cu_k, causal=True)
    assert not got[:rows - 70].any()
    check(got[rows - 70:], None, q[rows - 70:], k, k, [70], [70], causal=True)


@pytest.mark.parametrize("few", [True, False])
def test_more_blocks_than_a_grid_dimension_holds(cuda, few):
    """Blocks counted along the grid's other dimension: a few long sequences, or 70000 of a row or two."""
    if few:
        lens = [100, 17_000_000, 300]
        q = torch.zeros(sum(lens), 2, 64, dtype=torch.bfloat16, device=cuda)  # 4.4 GB
        q[:100], q[-300:] = make(28, cuda, torch.bfloat16, 100, 2, 64), make(29, cuda, torch.bfloat16, 300, 2, 64)
        len_k = [100, 1, 300]
        k = make(30, cuda, torch.bfloat16, sum(len_k), 2, 64)
        out = T.attention_packed(q, k, k, starts(lens, cuda), starts(len_k, cuda))
        check(out[:100], None, q[:100], k[:100], k[:100], [100], [100])
        middle = out[100:-300]
        assert bool((middle == k[100]).all())  # a single key
        check(out[-300:], None, q[-300:], k[101:], k[101:], [300], [300])
        return
    lens = [1 + (i * 7919) % 2 for i in range(70_000)]
    q = make(31, cuda, torch.bfloat16, sum(lens), 1, 64)
    k, v = make(32, cuda, torch.bfloat16, sum(lens), 1, 64), make(33, cuda, torch.bfloat16, sum(lens), 1, 64)
    cu = starts(lens, cuda).long()
    for most in (None, 2):
        out = T.attention_packed(q, k, v, cu.int(), causal=True, max_seqlen_q=most)[:, 0]
        assert torch.equal(out[cu[:-1]], v[cu[:-1], 0])  # the first token of each sees itself
        two = cu[:-1][cu.diff() == 2]
        s = (q[two + 1, 0].double()[:, None] * torch.stack((k[two, 0], k[two + 1, 0]), 1).double()).sum(-1) / 8
        want = (torch.softmax(s, -1)[..., None] * torch.stack((v[two, 0], v[two + 1, 0]), 1).double()).sum(1)
        # one rounding of each of two probabilities and one of the result, weights far closer
        assert float((out[two + 1].double() - want).abs().max()) <= 2.01 * 2 ** -8 * float(v.abs().max())


@pytest.mark.parametrize("most", [None, 1])
def test_strides_of_one_row(cuda, most):
    """An output of one row, whatever the stride of its rows."""
    q, k, v = (make(60 + i, cuda, torch.bfloat16, n, h, 64) for i, (n, h) in enumerate([(1, 8), (50, 2), (50, 2)]))
    buf = make(64, cuda, torch.bfloat16, 3, 8 * 64 + 4)
    held = buf.clone()
    out = buf[:, :512].unflatten(1, (8, 64))[:1]
    assert out.stride(0) % 8
    got = T.attention_packed(q, k, v, starts([1], cuda), starts([50], cuda), causal=True, max_seqlen_q=most, out=out)
    assert got is out
    check(out, None, q, k, v, [1], [50], causal=True)
    assert torch.equal(buf[1:], held[1:]) and torch.equal(buf[0, 512:], held[0, 512:])


@pytest.mark.parametrize("most", [None, 1])
def test_strides_of_tensors_without_keys(cuda, most):
    """Keys and values without a row, whatever their strides are."""
    q, k = make(60, cuda, torch.bfloat16, 1, 8, 64), make(61, cuda, torch.bfloat16, 5, 2, 64)
    for empty in (make(65, cuda, torch.bfloat16, 7, 2, 68)[:0, :, :64], k[:0, :1].expand(-1, 4, -1)):
        got, lse = T.attention_packed(q, empty, empty, starts([1], cuda), starts([0], cuda), max_seqlen_q=most,
                                      return_lse=True)
        assert not got.any() and bool((lse == float("-inf")).all())


# the table of a launch of several items per CTA: its order within every 128 sequences, its sum over all threads,
# its last entry (1024 sequences, or 1023 and the rows behind them; one more takes the search)
@pytest.mark.parametrize("count", [127, 128, 129, 300, 1023, 1024, 1025])
@pytest.mark.parametrize("short", [True, False])  # items of two tiles of heads, or of one
@pytest.mark.parametrize("spare", [0, 5])
def test_table_of_items(cuda, count, short, spare):
    g = torch.Generator().manual_seed(count)
    most = 16 if short else 70  # 8 heads of a group: 16 tokens to a tile
    len_q = torch.randint(0, most + 1, (count,), generator=g).tolist()
    len_q[0], len_q[-1], len_q[count // 2] = 0, most, 3 * most
    len_k = [n + m for n, m in zip(len_q, torch.randint(0, 150, (count,), generator=g).tolist())]
    rows = sum(len_q)
    assert (16 * count >= rows) == short
    q = make(66, cuda, torch.bfloat16, rows + spare, 16, 64)
    k, v = (make(i, cuda, torch.bfloat16, sum(len_k), 2, 64) for i in (67, 68))
    cu = starts(len_q, cuda), starts(len_k, cuda)
    out, lse = T.attention_packed(q, k, v, *cu, causal=True, return_lse=True)
    check(out, lse, q, k, v, len_q, len_k, causal=True)
    held = make(69, cuda, torch.bfloat16, *q.shape)
    again, lse2 = T.attention_packed(q, k, v, *cu, causal=True, return_lse=True, out=held.clone())
    assert torch.equal(again[:rows], out[:rows]) and torch.equal(again[rows:], held[rows:])
    assert torch.equal(lse2, lse)


def test_hundreds_of_thousands_of_empty_sequences(cuda):
    """Blocks without rows by the million, between two that hold some: longer than any wait may last."""
    n, heads = 500_000, 64
    at = 1000
    cu = torch.zeros(n + 1, dtype=torch.int32, device=cuda)
    cu[at:] = 150
    cu[-1] = 350
    q, k, v = (make(70 + i, cuda, torch.bfloat16, 353, heads, 64) for i in range(3))
    out, lse = T.attention_packed(q, k[:350], v[:350], cu, causal=True, return_lse=True)
    check(out, lse, q, k[:350], v[:350], [150, 200], [150, 200], causal=True)
    assert T.attention_status(cuda) == 0


def test_hundreds_of_thousands_of_rows_without_keys(cuda):
    """Items that load nothing, for longer than any wait may last, behind one that does."""
    n, heads = 400_000, 64
    q = make(74, cuda, torch.bfloat16, n + 150, heads, 64)  # 3.3 GB
    k, v = (make(i, cuda, torch.bfloat16, 300, heads, 64) for i in (75, 76))
    cu_q = torch.arange(150, n + 151, dtype=torch.int32, device=cuda)
    cu_q[0] = 0
    cu_k = torch.full((n + 1,), 150, dtype=torch.int32, device=cuda)
    cu_k[0], cu_k[-1] = 0, 300
    out, lse = T.attention_packed(q, k, v, cu_q, cu_k, causal=True, return_lse=True)
    first, last = slice(0, 151), slice(n + 149, n + 150)
    check(out[first], lse[:, first], q[first], k[:150], v[:150], [151], [150], causal=True)
    check(out[last], lse[:, last], q[last], k[150:], v[150:], [1], [150], causal=True)
    assert not out[151:-1].any() and bool((lse[:, 151:-1] == float("-inf")).all())
    assert T.attention_status(cuda) == 0
