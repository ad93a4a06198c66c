"""What the packed and shared-prefix attention refuse: at the C entries before any launch, and in the
tensor-level functions. Nothing here runs on a GPU."""
import ctypes

import pytest
import torch

import trinix_b200 as T
from trinix_b200 import _lib

I64x2 = _lib.I64x2
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
