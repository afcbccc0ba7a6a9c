"""Packed attention on the host: what the Python layer and the C entries refuse before any GPU is touched."""

import ctypes

import pytest
import torch

import open_vc_attn
from open_vc_attn import _lib


def test_python_layer_refuses_before_the_device():
    q = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="same CUDA device"):
        open_vc_attn.attention_packed(q, q, q, cu)
    with pytest.raises(ValueError, match="packed"):
        open_vc_attn.attention_packed(q[None], q[None], q[None], cu)
    with pytest.raises(ValueError, match="multiple"):
        open_vc_attn.attention_packed(q[:, :1], q, q, cu)


def test_c_entry_refuses_bad_arguments():
    import __graft_entry__

    __graft_entry__.build()
    lib, bad = _lib.load(), -1
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf) // 16 * 16 + 16
    good = (ctypes.c_int64 * 2)(256, 128)

    def call(q=p, k=p, v=p, qs=good, ks=good, vs=good, dtype=1, cq=p, ck=p, b=1, tq=4, tk=4, hq=2, hk=2, flags=0, scale=0.1, out=p, ws=p):
        return lib.ovc_attention_packed(q, qs, k, ks, v, vs, dtype, cq, ck, b, tq, tk, hq, hk, flags, scale, out, None, ws, None, None, None)

    for change in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cq=None), dict(ck=None), dict(qs=None), dict(q=p + 2),
                   dict(out=p + 8), dict(cq=p + 2), dict(dtype=2), dict(b=0), dict(tq=0), dict(tk=0), dict(hq=0), dict(hk=0), dict(hq=3),
                   dict(hq=129, hk=1), dict(flags=2), dict(flags=8), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                   dict(scale=float("inf")), dict(tq=(1 << 30) + 1), dict(hk=65536, hq=65536), dict(b=(1 << 20) + 1)):
        assert call(**change) == bad, change
    assert call(scale=3e38) == bad  # finite, but not times log2(e)
    for strides in ((0, 128), (256, 0), (-256, 128), (252, 128), (256, 130)):
        for name in ("qs", "ks", "vs"):
            assert call(**{name: (ctypes.c_int64 * 2)(*strides)}) == bad, strides
    # a launch that splits the keys needs its workspace
    assert lib.ovc_attention_packed_workspace(1, 1, 4096, 8, 8) > 0
    assert call(tq=1, tk=4096, hq=8, hk=8, ws=None) == bad
    assert call(tq=1, tk=4096, hq=8, hk=8, ws=p + 4) == bad


def test_workspace_sizes():
    lib = _lib.load()
    size = lib.ovc_attention_packed_workspace
    assert size(1, 73397, 73397, 14, 14) == 0          # rows enough for every SM
    assert size(1, 129, 129, 2, 2) == 0                # keys too few to share
    assert size(0, 1, 1, 1, 1) == size(1, 1, 1, 3, 2) == size(1, 0, 4096, 1, 1) == 0
    for b, tq, tk, hq, hk in ((16, 16, 200000, 32, 8), (4, 893, 59497, 28, 4), (1, 1, 1 << 30, 128, 1)):
        assert 0 < size(b, tq, tk, hq, hk) < 1 << 30


def test_the_version_counts_these_entries():
    import __graft_entry__

    __graft_entry__.build()
    assert _lib.load().ovc_version() >= 2
