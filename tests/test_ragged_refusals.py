"""What the packed and shared-prefix attention refuse: at the C entries before any launch, and in the
tensor-level functions. Nothing here runs on a GPU."""
import ctypes

import pytest
import torch

import trinix_b200 as T
from trinix_b200 import _lib

I64x2 = ctypes.c_int64 * 2
ONE = ctypes.c_void_p(4096)


def packed(lib, **change):
    a = dict(q=ONE, k=ONE, v=ONE, out=ONE, lse=None, slopes=None, cu_q=ONE, cu_k=ONE, n=2, tq=8, tk=8, hq=4,
             hk=2, d=128, qs=I64x2(512, 128), ks=I64x2(256, 128), vs=I64x2(256, 128), os=I64x2(512, 128),
             scale=1.0, causal=1, wl=-1, wr=-1, most=0, rest=1, dtype=2, ws=ONE, wsb=256, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return lib.trx_attn_fwd_packed(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(dtype=0), -2), (dict(hk=3), -3), (dict(n=-1), -3), (dict(tq=-1), -3), (dict(most=-1), -3),
    (dict(d=96), -6), (dict(wl=4), -3), (dict(wr=4), -3), (dict(q=None), -1), (dict(out=None), -1),
    (dict(k=None), -1), (dict(v=None), -1), (dict(cu_q=None), -1), (dict(cu_k=None), -1),
    (dict(ws=None), -9), (dict(wsb=8), -9), (dict(ws=ctypes.c_void_p(4100)), -9),
    (dict(tq=1 << 30), -3), (dict(tk=1 << 30), -3), (dict(hq=1 << 17), -3), (dict(n=1 << 24), -3),
    (dict(cu_q=ctypes.c_void_p(4098)), -4), (dict(out=ctypes.c_void_p(4104)), -4),
    (dict(os=I64x2(513, 128)), -4), (dict(qs=I64x2(-8, 128)), -5), (dict(os=I64x2(512, -8)), -5),
], ids=str)
def test_packed_entry_refuses(lib, change, code):
    assert packed(lib, **change) == code


def test_packed_entry_has_nothing_to_do(lib):
    assert packed(lib, tq=0) == 0
    assert packed(lib, n=0, rest=0) == 0


def test_cpu_tensors_are_refused():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        T.attention_packed(q, q, q, torch.tensor([0, 4], dtype=torch.int32))


I64x3 = _lib.I64x3


def shared(lib, **change):
    a = dict(q=ONE, pk=ONE, pv=ONE, k=ONE, v=ONE, out=ONE, lse=None, slopes=None, lengths=None, b=2, sq=1,
             p=9000, s=20, hq=4, hk=2, d=128, qs=I64x3(512, 512, 128), pks=I64x2(256, 128),
             pvs=I64x2(256, 128), ks=I64x3(5120, 256, 128), vs=I64x3(5120, 256, 128),
             os=I64x3(512, 512, 128), scale=1.0, dtype=2, parts=ONE, pb=1 << 30, ws=ONE, wsb=256, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return lib.trx_attn_fwd_shared(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(dtype=0), -2), (dict(hk=3), -3), (dict(b=-1), -3), (dict(p=-1), -3), (dict(s=-1), -3),
    (dict(d=96), -6), (dict(scale=0.0), -6), (dict(scale=1e-31), -6), (dict(scale=float("nan")), -6), (dict(q=None), -1),
    (dict(pk=None), -1), (dict(pv=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1),
    (dict(ws=None), -9), (dict(parts=None), -9), (dict(parts=ctypes.c_void_p(4104)), -9), (dict(pb=16), -9),
    (dict(b=1 << 17), -3), (dict(p=1 << 29), -3), (dict(s=1 << 29), -3), (dict(sq=1 << 30), -3),
    (dict(lengths=ctypes.c_void_p(4098)), -4), (dict(out=ctypes.c_void_p(4104)), -4),
    (dict(os=I64x3(512, 516, 128)), -4), (dict(qs=I64x3(-8, 512, 128)), -5), (dict(pks=I64x2(256, -8)), -5),
], ids=str)
def test_shared_entry_refuses(lib, change, code):
    assert shared(lib, **change) == code


# in parts; the sequences' own keys alone, by the kernel for few rows, which makes no tensor map of q; one pass
@pytest.mark.parametrize("way", [dict(), dict(p=0), dict(p=0, sq=16), dict(p=0, sq=17), dict(p=9, sq=200)], ids=str)
@pytest.mark.parametrize("change,code", [
    (dict(qs=I64x3(1 << 20, 512, 132)), -4), (dict(qs=I64x3((1 << 20) + 4, 512, 128)), -4),
    (dict(qs=I64x3(1 << 20, 512, 129)), -4), (dict(q=ctypes.c_void_p(4098)), -4), (dict(q=ctypes.c_void_p(4104)), -4),
    (dict(qs=I64x3(1 << 20, 512, 64)), -5), (dict(qs=I64x3(64, 512, 128)), -5), (dict(qs=I64x3(0, 512, 128)), -5),
], ids=str)
def test_shared_entry_refuses_queries_it_cannot_read(lib, way, change, code):
    assert shared(lib, **way, **change) == code


@pytest.mark.parametrize("way", [dict(p=0, sq=16), dict(p=0, sq=17), dict(p=9, sq=200)], ids=str)
def test_shared_entry_refuses_rows_of_queries_it_cannot_read(lib, way):
    assert shared(lib, qs=I64x3(1 << 20, 516, 128), **way) == -4
    assert shared(lib, qs=I64x3(1 << 20, 120, 128), **way) == -5


def test_shared_entry_has_nothing_to_do(lib):
    assert shared(lib, b=0) == 0
    assert shared(lib, sq=0) == 0


def test_shared_bytes(lib):
    """Space for the results of the prefix's splits: none without a prefix, none for one pass."""
    size = lib.trx_attn_shared_bytes
    assert size(64, 1, 0, 100, 32, 8, 128) == 0  # no prefix
    assert size(16, 320, 4096, 384, 32, 8, 128) == 0 and size(16, 8, 1024, 512, 32, 8, 128) == 0
    row = 64 * 32 * 129 * 4
    n = size(64, 1, 8192, 1024, 32, 8, 128)
    assert n >= row and n % row == 0
    assert size(4, 100, 30000, 300, 32, 8, 128) > 0  # many rows, but a long prefix
    for bad in ((0, 1, 5, 5, 4, 2, 64), (1, 1, -1, 5, 4, 2, 64), (1, 1, 5, -1, 4, 2, 64), (1, 1, 5, 5, 4, 3, 64),
                (1 << 20, 1, 5, 5, 4, 2, 64), (60000, 1 << 20, 5, 5, 4, 2, 64)):
        assert size(*bad) == 0


@pytest.mark.parametrize("b,sq,hq,rows", [(50_000, 3, 128, 2), (65_535, 5, 64, 4), (50_000, 12, 32, 8),
                                          (65_535, 20, 16, 16)])
def test_shared_bytes_of_more_rows_than_a_grid_holds(lib, b, sq, hq, rows):
    """`rows` of the batch are a block of the prefix's launch, which has room for 65535 of them: beyond that the
    call takes one pass, whatever a cost says."""
    size = lib.trx_attn_shared_bytes
    assert b * sq > 65535 * rows
    assert size(b, sq, 6000, 20, hq, 1, 128) == 0
    assert size(65535 * rows // sq, sq, 6000, 20, hq, 1, 128) > 0


def test_cpu_tensors_are_refused_behind_a_prefix():
    q, pk = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        T.attention_shared_prefix(q, pk, pk, q, q)
