"""What the paged cache and the attention over it refuse, and the norms of queries and keys: at the C entries before
any launch, and in the tensor-level functions. Nothing here runs on a GPU."""
import ctypes

import pytest
import torch

import trinix_b200 as T

ONE, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4104)
ALL = 1 << 40


def block(*values):
    return (ctypes.c_int64 * len(values))(*values)


def cache_strides(bits=16, **change):
    s = dict(kp=8192, kh=2048, kr=128, vp=8192, vh=2048, vr=128, ksp=128, ksh=32, vsp=128, vsh=32, table=10)
    if bits == 4:
        s.update(kp=2048, kh=1024, kr=64, vp=2048, vh=1024, vr=64)
    s.update(change)
    return list(s.values())


def append(lib, cache=None, bits=16, **change):
    scales = ONE if bits == 4 else None
    a = dict(q=ONE, k=ONE, v=ONE, qo=ONE, kp=ONE, vp=ONE, ks=scales, vs=scales, table=ONE, lengths=ONE, cu=None, cos=ONE,
             sin=ONE, n=2, s=1, hq=4, hk=2, d=128, pages=20, size=16, width=10,
             strides=block(512, 512, 128, 256, 256, 128, 256, 256, 128, 512, 512, 128, *(cache or cache_strides(bits))),
             rows=160, row=64, tdtype=0, dtype=2, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return lib.trx_paged_append(*a.values())


CACHE = [
    (dict(d=96), -6), (dict(size=24), -6), (dict(hk=0), -3), (dict(n=-1), -3), (dict(pages=-1), -3), (dict(size=0), -3),
    (dict(size=8192), -3), (dict(width=-1), -3), (dict(width=1 << 26), -3), (dict(pages=1 << 31), -3),
    (dict(hk=1 << 17), -3), (dict(kp=None), -1), (dict(vp=None), -1), (dict(table=None), -1), (dict(vs=ONE), -1),
    (dict(kp=ODD), -4), (dict(vp=ODD), -4), (dict(table=ctypes.c_void_p(4098)), -4), (dict(dtype=0), -2),
]


@pytest.mark.parametrize("change,code", CACHE + [
    (dict(tdtype=1), -2), (dict(s=-1), -3), (dict(hq=-1), -3), (dict(s=1 << 30), -3), (dict(k=None), -1),
    (dict(v=None), -1), (dict(lengths=None), -1), (dict(qo=None), -1), (dict(cos=None), -1), (dict(sin=None), -1),
    (dict(cos=None, sin=None), -1), (dict(strides=None), -1), (dict(k=ODD), -4), (dict(q=ODD), -4), (dict(qo=ODD), -4),
    (dict(lengths=ctypes.c_void_p(4098)), -4), (dict(cos=ODD), -4), (dict(row=63), -5), (dict(row=65), -4),
    (dict(rows=-1), -3), (dict(cu=ctypes.c_void_p(4098)), -4), (dict(n=0, cu=ONE, s=5), -3),
], ids=str)
def test_append_refuses(lib, change, code):
    assert append(lib, **change) == code


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("change,code", [(dict(kp=8), -5), (dict(kh=-2048), -5), (dict(kr=60), -5), (dict(vr=0), -5),
                                         (dict(kp=8196), -4), (dict(vh=2052), -4), (dict(table=-10), -5)], ids=str)
def test_cache_strides_are_refused(lib, bits, change, code):
    assert append(lib, bits=bits, cache=cache_strides(bits, **change)) == code


@pytest.mark.parametrize("change,code", [(dict(kr=80), -5), (dict(ksp=16), -5), (dict(vsh=0), -5), (dict(ksh=33), -4)], ids=str)
def test_code_strides_are_refused(lib, change, code):
    assert append(lib, bits=4, cache=cache_strides(4, **change)) == code


def test_append_has_nothing_to_do(lib):
    assert append(lib, s=0) == 0
    assert append(lib, n=0) == 0
    assert append(lib, n=0, cu=ONE, s=5, q=None) == 0


def gather(lib, bits=16, **change):
    scales = ONE if bits == 4 else None
    a = dict(kp=ONE, vp=ONE, ks=scales, vs=scales, table=ONE, cu=ONE, ko=ONE, vo=ONE, n=2, rows=30, hk=2, d=128, pages=20,
             size=16, width=10, strides=block(*cache_strides(bits)), rest=1, dtype=2, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return lib.trx_paged_gather(*a.values())


@pytest.mark.parametrize("change,code", CACHE + [
    (dict(rows=-1), -3), (dict(rows=1 << 30), -3), (dict(n=1 << 30), -3), (dict(ko=None), -1), (dict(vo=None), -1),
    (dict(cu=None), -1), (dict(ko=ODD), -4), (dict(vo=ODD), -4), (dict(cu=ctypes.c_void_p(4098)), -4),
    (dict(strides=None), -1),
], ids=str)
def test_gather_refuses(lib, change, code):
    assert gather(lib, **change) == code


def test_gather_has_nothing_to_do(lib):
    assert gather(lib, rows=0) == 0


def attend(lib, bits=16, **change):
    scales = ONE if bits == 4 else None
    a = dict(q=ONE, kp=ONE, vp=ONE, ks=scales, vs=scales, out=ONE, lse=None, slopes=None, table=ONE, lengths=ONE, n=2, sq=1,
             hq=4, hk=2, d=128, pages=20, size=16, width=10,
             strides=block(512, 512, 128, 512, 512, 128, *cache_strides(bits)), scale=1.0, left=-1, dtype=2, parts=ONE, pb=ALL,
             ws=ONE, wsb=256, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return lib.trx_attn_fwd_paged(*a.values())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("change,code", [x for x in CACHE if x[0] != dict(vs=ONE)] + [
    (dict(hk=3), -3), (dict(hq=0), -3), (dict(sq=-1), -3), (dict(q=None), -1), (dict(out=None), -1),
    (dict(lengths=None), -1), (dict(strides=None), -1), (dict(ws=None), -9), (dict(wsb=8), -9),
    (dict(ws=ctypes.c_void_p(4100)), -9), (dict(pages=0), -3), (dict(n=1 << 17), -3), (dict(sq=1 << 28), -3),
    (dict(sq=1 << 20), -3), (dict(scale=float("nan")), -6), (dict(scale=float("inf")), -6), (dict(q=ODD), -4),
    (dict(out=ODD), -4), (dict(lengths=ctypes.c_void_p(4098)), -4),
    (dict(strides=block(516, 512, 128, 512, 512, 128, *cache_strides())), -4),
    (dict(strides=block(-8, 512, 128, 512, 512, 128, *cache_strides())), -5),
    (dict(strides=block(512, 512, 128, 512, 516, 128, *cache_strides())), -4),
], ids=str)
def test_attention_refuses(lib, bits, change, code):
    if bits == 4 and "strides" in change and change["strides"] is not None:
        change = {"strides": block(*list(change["strides"])[:6], *cache_strides(4))}
    assert attend(lib, bits, **change) == code


def test_attention_refuses_too_little_room(lib):
    size = lambda width, left=-1, bits=16: lib.trx_attn_paged_bytes(2, 1, 4, 2, 128, 16 * width, left, int(bits == 4))  # noqa: E731
    for bits in (16, 4):
        assert size(10, bits=bits) == 0 and size(1000, 100, bits=bits) == 0  # a CTA to a sequence and head
        assert size(1000, bits=bits) > 0
        for change in (dict(parts=None), dict(pb=size(1000, bits=bits) - 1), dict(parts=ODD)):
            assert attend(lib, bits, width=1000, **change) == -9
    for bad in ((0, 1, 4, 2, 128), (2, 0, 4, 2, 128), (2, 1, 4, 3, 128), (2, 1, 4, 2, 96), (1 << 17, 1, 4, 2, 64)):
        assert lib.trx_attn_paged_bytes(*bad, 1 << 20, -1, 0) == 0


def test_attention_has_nothing_to_do(lib):
    assert attend(lib, n=0) == 0
    assert attend(lib, sq=0) == 0


def norms(lib, steps=None, **change):
    a = dict(q=ONE, k=ONE, qw=ONE, kw=ONE, qb=None, kb=None, cos=ONE, sin=ONE, pos=None, qo=ONE, ko=ONE, b=2, s=4, hq=3, hk=1,
             d=64, strides=block(*(steps or [768, 192, 64, 256, 64, 64] * 2), 0, 0), rows=4, row=32, eps=1e-6, norm=0,
             first=1, wide=0, tdtype=0, wdtype=2, dtype=2, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return lib.trx_qk_norm_rope_fwd(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), -2), (dict(tdtype=1), -2), (dict(wdtype=5), -2), (dict(norm=2), -6), (dict(d=63), -3), (dict(d=0), -3),
    (dict(d=514), -6), (dict(b=-1), -3), (dict(s=-1), -3), (dict(hq=-1), -3), (dict(hq=1 << 17), -3), (dict(rows=3), -3),
    (dict(rows=-1), -3), (dict(row=31), -5), (dict(q=None), -1), (dict(k=None), -1), (dict(qw=None), -1),
    (dict(kw=None), -1), (dict(cos=None), -1), (dict(sin=None), -1), (dict(qo=None), -1), (dict(ko=None), -1),
    (dict(strides=None), -1), (dict(eps=-1.0), -6), (dict(eps=float("nan")), -6), (dict(b=1 << 20, s=1 << 12), -3),
    (dict(b=1 << 14, s=1 << 14, hq=64), -3), (dict(pos=ctypes.c_void_p(4098)), -4), (dict(pos=ctypes.c_void_p(4100), wide=1), -4),
], ids=str)
def test_norms_refuse(lib, change, code):
    assert norms(lib, **change) == code


def test_norms_refuse_strides(lib):
    assert norms(lib, steps=[-768, 192, 64, 256, 64, 64] * 2) == -5
    assert norms(lib, steps=[768, 192, 64, 256, 64, 64, 768, 192, 64, 256, -64, 64]) == -5


def test_norms_have_nothing_to_do(lib):
    assert norms(lib, b=0) == 0 and norms(lib, s=0) == 0 and norms(lib, hq=0, hk=0) == 0


def test_norm_gradients_refuse(lib):
    f = lib.trx_qk_norm_rope_bwd
    size = lib.trx_qk_norm_rope_bwd_workspace_bytes
    assert size(0) == 0 and size(514) == 0 and size(64) > 0
    s = block(*[768, 192, 64, 256, 64, 64] * 3, 0, 0)
    args = lambda dy=ONE, db=None, norm=0, ws=ONE, n=ALL: (  # noqa: E731
        dy, ONE, ONE, ONE, ONE, ONE, ONE, ONE, None, ONE, ONE, ONE, ONE, db, db, 2, 4, 3, 1, 64, s, 4, 32, 1e-6, norm, 1, 0,
        0, 2, 2, ws, n, None)
    assert f(*args(dy=None)) == -1
    assert f(*args(db=ONE)) == -6
    assert f(*args(ws=None)) == -9 and f(*args(n=size(64) - 1)) == -9 and f(*args(ws=ODD)) == -9


# ------------------------------------------------------------------- tensors: all on the CPU, refused as such at last
def tensors(bits=16, B=2, S=1, Hk=2, D=64, size=16, pages=5, dtype=torch.bfloat16):
    k = torch.zeros(B, S, Hk, D, dtype=dtype)
    held = torch.zeros(pages, Hk, size, D // 2 if bits == 4 else D, dtype=torch.uint8 if bits == 4 else dtype)
    c = dict(k_pages=held, v_pages=held.clone(), block_table=torch.zeros(B, 3, dtype=torch.int32))
    if bits == 4:
        c |= dict(k_scales=torch.zeros(pages, Hk, size, 2), v_scales=torch.zeros(pages, Hk, size, 2))
    return k, c, torch.ones(B, dtype=torch.int32)


@pytest.mark.parametrize("bits", [16, 4])
def test_cpu_tensors_are_refused(bits):
    k, c, lengths = tensors(bits)
    with pytest.raises(ValueError, match="CUDA"):
        T.append_paged(k, k, **c, lengths=lengths)
    with pytest.raises(ValueError, match="CUDA"):
        T.gather_paged(**c, cu_seqlens=torch.zeros(3, dtype=torch.int32), rows=4)
    with pytest.raises(ValueError, match="CUDA"):
        T.attention_paged(k, **c, lengths=lengths)
    with pytest.raises(ValueError, match="CUDA"):
        T.qk_norm_rope(k, k, k[0, 0, 0], k[0, 0, 0], k[0, 0], k[0, 0])


@pytest.mark.parametrize("change,error", [(dict(bits=8), ValueError), (dict(dtype=torch.float32), TypeError),
                                          (dict(page_size=24), ValueError), (dict(num_pages=0), ValueError),
                                          (dict(head_dim=96), ValueError), (dict(page_size=8192), ValueError)], ids=str)
def test_cache_refuses(change, error):
    a = dict(num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, batch_size=2, device="cpu")
    with pytest.raises(error):
        T.PagedKVCache(**{**a, **change})


def test_cache_reserves_pages():
    c = T.PagedKVCache(6, 16, 2, 64, 2, max_pages=4, device="cpu")
    c.reserve([17, 3])
    assert sorted(c.block_table.flatten().tolist()) == [-1] * 5 + [0, 1, 2]
    c.reserve(16)  # less than one has, as much as the other
    assert (c.block_table >= 0).sum(1).tolist() == [2, 1]
    for bad in (65, [0, 80]):
        before = c.block_table.clone()
        with pytest.raises(RuntimeError, match="pages"):
            c.reserve(bad)
        assert torch.equal(c.block_table, before)
    for bad in ([1], [-1, 0]):
        with pytest.raises(ValueError):
            c.reserve(bad)
    c.release(0)
    c.reserve([0, 64])
    assert (c.block_table >= 0).sum(1).tolist() == [0, 4]


@pytest.mark.parametrize("kv,error", [(torch.zeros(2, 1, 2, 64, dtype=torch.float16), TypeError),
                                      (torch.zeros(2, 1, 3, 64, dtype=torch.bfloat16), ValueError),
                                      (torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16), ValueError),  # not on CUDA
                                      (torch.zeros(2), ValueError)], ids=lambda x: str(getattr(x, "shape", x)))
def test_a_refused_append_leaves_the_cache_as_it_was(kv, error):
    c = T.PagedKVCache(6, 16, 2, 64, 2, device="cpu", bits=4)
    with pytest.raises(error):
        c.append(kv, kv)
    assert c.lengths.tolist() == [0, 0] and c._held == [0, 0]


def test_cache_reads_the_lengths_once_a_step_was_captured():
    c = T.PagedKVCache(6, 16, 2, 64, 2, device="cpu")
    c.reserve(16)
    c.lengths.fill_(16)  # what replays did
    c._captured = True
    c.reserve(1)
    assert (c.block_table >= 0).sum(1).tolist() == [2, 2]


def test_long_tables_are_kept():
    """A captured graph may read tables that later ones are longer than."""
    rope = T.FastRoPEPositionEmbedding(64, 16)
    cpu = torch.device("cpu")
    with torch.inference_mode():
        short = rope.tables(5, cpu)
    long = rope.tables(40, cpu)
    assert short[0].shape == (16, 64) and long[0].shape == (64, 64) and not short[0].is_inference()
    assert torch.equal(short[0], long[0][:16]) and torch.equal(short[1], long[1][:16])
    assert rope.tables(16, cpu) is short and rope.tables(50, cpu) is long
    cos, sin = rope(torch.zeros(1, 64), 40)
    assert torch.equal(cos, long[0][:40]) and torch.equal(sin, long[1][:40])
