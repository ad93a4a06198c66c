"""How programs use the packed and the shared-prefix attention: streams, graphs, failures, autograd."""
import ctypes

import pytest
import torch

import trinix_b200 as T
from tests.test_gpu_packed import make, starts
from tests.test_gpu_packed import check as check_packed
from tests.test_gpu_shared_prefix import check as check_shared
from tests.test_gpu_shared_prefix import inputs, lengths

pytestmark = pytest.mark.gpu


def packed_state(dev, seed, lens=(70, 3, 260, 128), cached=(0, 500, 40, 7)):
    len_k = [n + m for n, m in zip(lens, cached)]
    q = make(seed, dev, torch.bfloat16, sum(lens), 8, 128)
    k, v = (make(seed + i, dev, torch.bfloat16, sum(len_k), 2, 128) for i in (1, 2))
    return q, k, v, starts(lens, dev), starts(len_k, dev)


def run_packed(s, **how):
    return T.attention_packed(*s, causal=True, return_lse=True, **how)


def shared_state(dev, seed, Sq=1, P=6000, lens=(30, 200, 77)):
    return (*inputs(dev, torch.bfloat16, len(lens), Sq, P, 200, 8, 2, 128, seed=seed), lengths(lens, dev))


def run_shared(s):
    return T.attention_shared_prefix(*s, return_lse=True)


# every kernel of the two: single items, several per CTA, few rows; prefix and decode, one pass
KINDS = {
    "packed": (packed_state, run_packed),
    "packed, many items": (lambda d, s: packed_state(d, s, [500, 30] * 20, [0, 300] * 20), run_packed),
    "packed, few rows": (lambda d, s: packed_state(d, s, (1, 1, 3, 1), (900, 5, 200, 0)),
                         lambda s: run_packed(s, max_seqlen_q=3)),
    "shared, in parts": (shared_state, run_shared),
    "shared, in parts of many rows": (lambda d, s: shared_state(d, s, 28, 20_000, (30, 200, 77) * 3), run_shared),
    "shared, one pass": (lambda d, s: shared_state(d, s, 25, 300), run_shared),
}


def test_kinds(cuda):
    """That the kinds take the ways they are named after."""
    size = T._lib.load().trx_attn_shared_bytes
    assert size(3, 1, 6000, 200, 8, 2, 128) > 0 and size(9, 28, 20_000, 200, 8, 2, 128) > 0
    assert size(3, 25, 300, 200, 8, 2, 128) == 0


@pytest.mark.parametrize("kind", KINDS)
def test_same_bits_every_time(cuda, kind):
    make_state, run = KINDS[kind]
    s = make_state(cuda, 1)
    first = run(s)
    for _ in range(20):
        again = run(s)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@pytest.mark.parametrize("kind", KINDS)
def test_two_streams_at_once(cuda, kind):
    make_state, run = KINDS[kind]
    states = [make_state(cuda, 10 * i) for i in range(2)]
    want = [run(s) for s in states]
    streams = [torch.cuda.Stream(cuda) for _ in states]
    torch.cuda.synchronize(cuda)
    for _ in range(15):
        got = []
        for s, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                got.append(run(s))
        torch.cuda.synchronize(cuda)
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


@pytest.mark.parametrize("kind", KINDS)
def test_captured_and_replayed(cuda, kind):
    """Two graphs, replayed beside each other, on inputs that change between the replays: values, and
    the lengths of the sequences, which only the device knows."""
    make_state, run = KINDS[kind]
    run(make_state(cuda, 5))  # first use outside of a capture
    graphs = []
    for i in range(2):
        s, g = make_state(cuda, 20 + i), torch.cuda.CUDAGraph()
        torch.cuda.synchronize(cuda)
        with torch.cuda.graph(g):
            out = run(s)
        graphs.append((s, g, out))
    streams = [torch.cuda.Stream(cuda) for _ in graphs]
    for turn in range(3):
        for s, _, _ in graphs:
            for t in s:
                if t.is_floating_point():
                    t.copy_(torch.randn(t.shape, device=cuda))
            if kind.startswith("packed") and turn:  # other sequences of the same rows, but for one
                lens = s[3].diff().tolist()
                lens = lens[1:] + lens[:1]
                lens[lens.index(max(lens))] -= 1
                s[3].copy_(starts(lens, cuda))
            elif turn:
                s[5].copy_(s[5].flip(0))
        torch.cuda.synchronize(cuda)
        for (_, g, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize(cuda)
        for s, _, out in graphs:
            want = run(s)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
            if kind.startswith("packed"):
                len_q, len_k = s[3].diff().tolist(), s[4].diff().tolist()
                check_packed(out[0], out[1], *s[:3], len_q, len_k, causal=True)
            else:
                check_shared(out[0], out[1], *s[:5], s[5].tolist())


@pytest.mark.parametrize("kind", KINDS)
def test_inputs_of_another_stream(cuda, kind):
    """Inputs made on one stream, the call on another that waits for it."""
    make_state, run = KINDS[kind]
    side = torch.cuda.Stream(cuda)
    want = run(make_state(cuda, 30))
    torch.cuda.synchronize(cuda)
    for _ in range(5):
        torch.cuda._sleep(200_000)
        s = make_state(cuda, 30)
        side.wait_stream(torch.cuda.current_stream(cuda))
        with torch.cuda.stream(side):
            got = run(s)
        torch.cuda.current_stream(cuda).wait_stream(side)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", KINDS)
def test_recorded_failure(cuda, kind):
    """Launches behind a recorded failure do no work; the next call raises once. Set from the host."""
    from trinix_b200 import ops
    make_state, run = KINDS[kind]
    s = make_state(cuda, 40)
    good = run(s)
    torch.cuda.synchronize(cuda)
    ops._workspace(cuda)[:4].view(torch.int32).fill_(4)
    run(s)
    torch.cuda.synchronize(cuda)
    assert int(ops._status_host[cuda.index or 0][0]) == 4
    with pytest.raises(T._lib.TrinixB200Error):
        run(s)
    again = run(s)
    assert torch.equal(again[0], good[0]) and torch.equal(again[1], good[1])
    assert T.attention_status(cuda) == 0


def call_packed(lib, s, out, lse, ws, max_rows=0):
    """The C entry, which zeroes rows behind the last sequence."""
    q, k, v, cu_q, cu_k = s
    strides = [(ctypes.c_int64 * 2)(*t.stride()[:2]) for t in (q, k, v, out)]
    return lib.trx_attn_fwd_packed(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), None, cu_q.data_ptr(),
        cu_k.data_ptr(), cu_q.numel() - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], *strides,
        q.shape[2] ** -0.5, 1, -1, -1, max_rows, 1, T._lib.TRX_BF16, ws.data_ptr(), ws.numel(),
        torch.cuda.current_stream(q.device).cuda_stream)


def call_shared(lib, s, out, lse, ws):
    q, pk, pv, k, v, n = s
    B, Sq, hq, d = q.shape
    sizes = B, Sq, pk.shape[0], k.shape[1], hq, k.shape[2], d
    size = lib.trx_attn_shared_bytes(*sizes)
    parts = torch.empty(max(size, 1), dtype=torch.uint8, device=q.device)
    st = [T._lib.I64x3(*t.stride()[:3]) for t in (q, k, v, out)]
    rows = [T._lib.I64x3(*t.stride()[:2], 0) for t in (pk, pv)]
    return lib.trx_attn_fwd_shared(
        q.data_ptr(), pk.data_ptr(), pv.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
        None, n.data_ptr(), *sizes, st[0], *rows, st[1], st[2], st[3], d ** -0.5, T._lib.TRX_BF16,
        parts.data_ptr(), size, ws.data_ptr(), ws.numel(), torch.cuda.current_stream(q.device).cuda_stream)


@pytest.mark.parametrize("kind", KINDS)
def test_nothing_is_written_behind_a_recorded_failure(cuda, kind):
    """Output and sums of a launch that finds one, rows behind the last sequence among them. Set from the host,
    in a workspace of its own."""
    lib = T._lib.load()
    s = KINDS[kind][0](cuda, 120)
    if kind.startswith("packed"):
        spare = torch.cat((s[0], s[0][:3]))  # three rows of no sequence
        s = (spare, *s[1:])
        shape, most = (s[0].shape[1], s[0].shape[0]), 3 if "few" in kind else 0
        call = lambda *a: call_packed(*a, max_rows=most)  # noqa: E731
    else:
        shape, call = (s[0].shape[0], s[0].shape[2], s[0].shape[1]), call_shared
    out, lse = torch.full_like(s[0], 7.0), torch.full(shape, 7.0, device=cuda)
    ws = torch.zeros(256, dtype=torch.uint8, device=cuda)
    ws[:4].view(torch.int32).fill_(4)
    assert call(lib, s, out, lse, ws) == 0
    torch.cuda.synchronize(cuda)
    assert bool((out == 7.0).all()) and bool((lse == 7.0).all())
    ws.zero_()
    assert call(lib, s, out, lse, ws) == 0
    if kind.startswith("packed"):
        check_packed(out, lse, *s[:3], s[3].diff().tolist(), s[4].diff().tolist(), causal=True)
    else:
        check_shared(out, lse, *s[:5], s[5].tolist())


def test_kernel_classes(cuda):
    assert T.PackedAttentionKernel.is_available() and T.SharedPrefixAttentionKernel.is_available()
    q, k, v, cu_q, cu_k = packed_state(cuda, 50)
    want = T.attention_packed(q, k, v, cu_q, cu_k, causal=True, window=(100, 0), scale=0.1)
    got = T.PackedAttentionKernel.apply(q, k, v, cu_q, cu_k, causal=True, window_size=(100, 0), scale=0.1)
    assert torch.equal(got, want)
    s = shared_state(cuda, 60)
    assert torch.equal(T.SharedPrefixAttentionKernel.apply(*s), T.attention_shared_prefix(*s))
    # forward only: the output is attached to the graph, and its backward says so
    out = T.PackedAttentionKernel.apply(q.clone().requires_grad_(), k, v, cu_q, cu_k)
    with pytest.raises(NotImplementedError):
        out.sum().backward()
    out = T.SharedPrefixAttentionKernel.apply(*s[:1], s[1].clone().requires_grad_(), *s[2:])
    with pytest.raises(NotImplementedError):
        out.sum().backward()
    with torch.no_grad():
        assert T.PackedAttentionKernel.apply(q.requires_grad_(), k, v, cu_q, cu_k).grad_fn is None


def test_refusals(cuda):
    q, k, v, cu_q, cu_k = packed_state(cuda, 70)
    bad = [
        (TypeError, (q.float(), k.float(), v.float(), cu_q, cu_k), {}),
        (TypeError, (q, k.half(), v, cu_q, cu_k), {}),
        (ValueError, (q[None], k, v, cu_q, cu_k), {}),
        (ValueError, (q, k[None], v[None], cu_q, cu_k), {}),
        (ValueError, (q, k, v[:-1], cu_q, cu_k), {}),
        (ValueError, (q[..., :64], k, v, cu_q, cu_k), {}),
        (ValueError, (q[:, :7], k, v, cu_q, cu_k), {}),
        (ValueError, (q, k[:, :0], v[:, :0], cu_q, cu_k), {}),
        (ValueError, (q, k, v, cu_q.long(), cu_k), {}),
        (ValueError, (q, k, v, cu_q, cu_k[:-1]), {}),
        (ValueError, (q, k, v, cu_q[None], cu_k), {}),
        (ValueError, (q, k, v, cu_q[:0], cu_k[:0]), {}),
        (ValueError, (q, k, v, cu_q.cpu(), cu_k), {}),
        (ValueError, (q, k, v, cu_q, cu_k), dict(window=(-1, 0))),
        (ValueError, (q, k, v, cu_q, cu_k), dict(max_seqlen_q=-1)),
        (ValueError, (q, k, v, cu_q, cu_k), dict(alibi_slopes=torch.ones(7, device=cuda))),
        (ValueError, (q, k, v, cu_q, cu_k), dict(out=q[:-1].clone())),
        (ValueError, (q, k, v, cu_q, cu_k), dict(out=q.half())),
        (ValueError, tuple(make(1, cuda, torch.bfloat16, 4, 2, 136) for _ in range(3)) + (cu_q, cu_k), {}),
    ]
    for error, args, how in bad:
        with pytest.raises(error):
            T.attention_packed(*args, **how)
    q, pk, pv, k, v, n = shared_state(cuda, 80)
    bad = [
        (TypeError, (q.float(), pk, pv, k, v, n), {}),
        (TypeError, (q, pk, pv, k.half(), v, n), {}),
        (ValueError, (q[0], pk, pv, k, v, n), {}),
        (ValueError, (q, pk[None], pv, k, v, n), {}),
        (ValueError, (q, pk, pv[:-1], k, v, n), {}),
        (ValueError, (q, pk, pv, k, v[:, :-1], n), {}),
        (ValueError, (q, pk, pv, k[:-1], v[:-1], n), {}),
        (ValueError, (q, pk[:, :1], pv[:, :1], k, v, n), {}),
        (ValueError, (q[:, :, :7], pk, pv, k, v, n), {}),
        (ValueError, (q, pk, pv, k, v, n.long()), {}),
        (ValueError, (q, pk, pv, k, v, n[:-1]), {}),
        (ValueError, (q, pk, pv, k, v, n.cpu()), {}),
        (ValueError, (q, pk, pv, k, v, n), dict(scale=0.0)),
        (ValueError, (q, pk, pv, k, v, n), dict(scale=-1.0)),
        (ValueError, (q, pk, pv, k, v, n), dict(alibi_slopes=torch.ones(3, device=cuda))),
    ]
    for error, args, how in bad:
        with pytest.raises(error):
            T.attention_shared_prefix(*args, **how)


def test_bounds_out_of_order_are_cut(cuda):
    """Bounds that no batch has: no fault, and sequences whose own bounds are right keep their results."""
    q, k, v, cu_q, cu_k = packed_state(cuda, 90)
    bad_k = cu_k.clone()
    bad_k[1] = 1 << 30  # the first two sequences' keys
    for how in ({}, dict(max_seqlen_q=16)):
        T.attention_packed(q, k, v, torch.full_like(cu_q, -7), cu_k, **how)
        T.attention_packed(q, k, v, cu_q.flip(0).contiguous(), cu_k.flip(0).contiguous(), **how)
        T.attention_packed(q, k, v, cu_q * 1000, cu_k * 1000, **how)
    want = T.attention_packed(q, k, v, cu_q, cu_k, causal=True)
    got = T.attention_packed(q, k, v, cu_q, bad_k, causal=True)
    assert torch.equal(got[73:], want[73:])
    assert T.attention_status(cuda) == 0


def test_no_sequences_and_no_rows(cuda):
    q, k, v, cu_q, cu_k = packed_state(cuda, 100)
    none = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = T.attention_packed(q, k, v, none, none, return_lse=True)
    assert not out.any() and torch.equal(lse, torch.full_like(lse, float("-inf")))
    held = q.clone()
    assert T.attention_packed(q, k, v, none, none, out=held) is held and torch.equal(held, q)
    assert T.attention_packed(q[:0], k, v, cu_q * 0, cu_k).shape == (0, 8, 128)
    out = T.attention_packed(q, k[:0], v[:0], cu_q, cu_k * 0)
    assert not out.any()


@pytest.mark.parametrize("B,Sq,P,hq,hk,d", [(3, 1, 6000, 8, 2, 128), (9, 28, 20_000, 8, 2, 64), (70, 2, 5000, 6, 2, 128),
                                            (5, 1, 3000, 160, 160, 64)])
def test_nothing_beside_the_outputs_is_written(cuda, B, Sq, P, hq, hk, d):
    """The space for the parts, the output and the sums, each in the middle of a larger buffer."""
    from trinix_b200 import ops
    lib = T._lib.load()
    q, pk, pv, k, v = inputs(cuda, torch.bfloat16, B, Sq, P, 64, hq, hk, d, seed=110)
    n = lengths([1 + (11 * b) % 64 for b in range(B)], cuda)
    want, want_lse = T.attention_shared_prefix(q, pk, pv, k, v, n, return_lse=True)
    size = lib.trx_attn_shared_bytes(B, Sq, P, 64, hq, hk, d)
    assert size > 0

    def guarded(numel, dtype):
        t = torch.full((numel + 512,), 7, dtype=dtype, device=cuda)
        return t, t[256:256 + numel]

    parts_all, parts = guarded(size, torch.uint8)
    out_all, out = guarded(q.numel(), torch.bfloat16)
    lse_all, lse = guarded(B * hq * Sq, torch.float32)
    strides = [T._lib.I64x3(*t.stride()[:3]) for t in (q, k, v)]
    rows = [T._lib.I64x3(*t.stride()[:2], 0) for t in (pk, pv)]
    ws = ops._workspace(cuda)
    rc = lib.trx_attn_fwd_shared(
        q.data_ptr(), pk.data_ptr(), pv.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
        None, n.data_ptr(), B, Sq, P, 64, hq, hk, d, strides[0], rows[0], rows[1], strides[1], strides[2],
        T._lib.I64x3(*q.stride()[:3]), d ** -0.5, T._lib.TRX_BF16, parts.data_ptr(), size, ws.data_ptr(),
        ws.numel(), torch.cuda.current_stream(cuda).cuda_stream)
    assert rc == 0
    torch.cuda.synchronize(cuda)
    for t in (parts_all, out_all, lse_all):
        assert bool((t[:256] == 7).all()) and bool((t[-256:] == 7).all())
    assert torch.equal(out.view(want.shape), want) and torch.equal(lse.view(want_lse.shape), want_lse)
