"""Rotary positions on the host: argument checks of the Python layer and of the C entries, before any GPU is touched."""

import ctypes

import pytest
import torch

import open_vc_attn
from open_vc_attn import _lib


def test_plan_refusals():
    p = torch.zeros(4, 3, dtype=torch.int32)
    for bad in (None, [0], p.double(), p[0], p[None, None]):
        with pytest.raises(ValueError, match="positions must be an int32"):
            open_vc_attn.rotary_plan(bad)
    for axes in ((), (43, 42, 42), (0, 64, 64), (44, 44, 44)):
        with pytest.raises(ValueError, match="even channel counts"):
            open_vc_attn.rotary_plan(p, axes=axes)
    with pytest.raises(ValueError, match="2 are described"):
        open_vc_attn.rotary_plan(p, axes=(64, 64))
    with pytest.raises(ValueError, match="128 channels in all"):
        open_vc_attn.rotary_plan(p, axes=(40, 40, 40), interleaved=False)
    with pytest.raises(ValueError, match="axis or head"):
        open_vc_attn.rotary_plan(p, frequencies="both")
    for theta in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="theta"):
            open_vc_attn.rotary_plan(p, theta=theta)
    for eps in (-1e-6, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            open_vc_attn.rotary_plan(p, eps=eps)
    with pytest.raises(ValueError, match="CUDA device"):
        open_vc_attn.rotary_plan(p)


def test_calls_refuse_cpu_tensors_and_foreign_plans():
    q = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="same CUDA device"):
        open_vc_attn.rotary_qk(q, q, None)
    with pytest.raises(ValueError, match="Expected"):
        open_vc_attn.rotary_qk(q[..., :64], q, None)
    with pytest.raises(ValueError, match="same CUDA device"):
        open_vc_attn.attention(q, q, q, rotary=None)


def test_grid_positions():
    got = open_vc_attn.grid_positions(2, 2, 3, text=1, start=(5, 0, 1), device="cpu")
    assert got.dtype == torch.int32 and got.shape == (13, 3)
    assert got[0].tolist() == [0, 0, 0] and got[1].tolist() == [5, 0, 1] and got[-1].tolist() == [6, 1, 3]
    with pytest.raises(ValueError, match="at least one"):
        open_vc_attn.grid_positions(0, 2, 3, device="cpu")


def test_c_entries_refuse_bad_arguments():
    import __graft_entry__

    __graft_entry__.build()
    lib, bad = _lib.load(), -1
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf) // 16 * 16 + 16
    turns, axis = (ctypes.c_double * 64)(), (ctypes.c_uint8 * 64)()

    def plan(**change):
        fields = dict(positions=p, position_batch_stride=0, turns=ctypes.addressof(turns), pair_axis=ctypes.addressof(axis),
                      q_weight=None, k_weight=None, position_type=0, axes=1, half_split=0, eps=1e-6)
        return ctypes.byref(_lib.OvcRotary(**{**fields, **change}))

    strides = (ctypes.c_int64 * 3)(1024, 256, 128)

    def rotate(r=None, q=p, k=p, dtype=1, b=1, s=4, hq=2, hk=2, qs=strides, out=p):
        return lib.ovc_rotary_qk(q, qs, k, strides, dtype, b, s, hq, hk, plan() if r is None else r, out, p, None)

    assert lib.ovc_rotary_qk(None, None, None, None, 1, 1, 1, 1, 1, None, None, None, None) == bad
    assert rotate(q=None) == rotate(k=p + 2) == rotate(out=p + 8) == rotate(dtype=2) == rotate(b=0) == rotate(s=0) == bad
    assert rotate(hq=0) == rotate(hk=65536) == rotate(b=32767, s=1 << 30) == rotate(qs=(ctypes.c_int64 * 3)(1024, 256, 132)) == bad
    assert rotate(qs=(ctypes.c_int64 * 3)(1024, -256, 128)) == bad
    for change in (dict(positions=None), dict(positions=p + 2), dict(positions=p + 4, position_type=1), dict(position_type=3),
                   dict(axes=0), dict(axes=65), dict(eps=-1.0), dict(eps=float("nan")), dict(turns=None), dict(pair_axis=None),
                   dict(position_batch_stride=-1), dict(q_weight=p + 2)):
        assert rotate(plan(**change)) == bad, change
    axis[63] = 1  # an axis that the positions do not have
    assert rotate() == bad
    axis[63] = 0
    turns[3] = float("inf")
    assert rotate() == bad
    turns[3] = 0.0
    general = lib.ovc_prepare_rotary
    assert general(p, p, p, 1, 1, 128, 1, plan(), p + 4, p, p, p, p, p, p, None, None) == bad  # misaligned codes
    assert general(p, p, p, 1, 1, 128, 1, plan(), p, p, p + 4, p, p, p, p, None, None) == bad
    assert general(p, p, p, 7, 1, 128, 1, plan(), p, p, p, p, p, p, p, None, None) == bad
    assert general(p, p, p, 1, 1, 128, 1, plan(), p, p, p, p, None, p, p, None, None) == bad
    assert general(p, p, p + 2, 1, 1, 128, 1, plan(), p, p, p, p, p, p, p, None, None) == bad
    assert general(p, p, p, 1, 2, 128, 1, plan(), p, p, p, p, p, p, p, p, None) == bad  # bounds of a batch
    fused = lib.ovc_prepare_fused_rotary
    assert fused(p, p, None, 1, 128, 1, plan(), p, p, p, p, p, p, p, None, None) == bad
    assert fused(p, p, p, 1, 128, 1, None, p, p, p, p, p, p, p, None, None) == bad
    assert fused(p, p, p, 1, 128, 1, plan(), p, p, p + 8, p, p, p, p, None, None) == bad


def test_plan_refuses_frequencies_that_overflow():
    with pytest.raises(ValueError, match="theta"):
        _plan_on_meta(theta=5e-324)


def _plan_on_meta(**options):
    class Positions(torch.Tensor):  # passes for a CUDA tensor; the refusal comes before anything is read
        is_cuda = True

    return open_vc_attn.rotary_plan(torch.zeros(4, 1, dtype=torch.int32).as_subclass(Positions), axes=(128,), **options)


@pytest.mark.parametrize("bad", [2.0 ** 30, -(2.0 ** 30), 1e300])
def test_c_entries_refuse_frequencies_that_fractional_positions_cannot_take(bad):
    import __graft_entry__

    __graft_entry__.build()
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf) // 16 * 16 + 16
    turns, axis = (ctypes.c_double * 64)(), (ctypes.c_uint8 * 64)()
    turns[5] = bad
    plan = _lib.OvcRotary(positions=p, position_batch_stride=0, turns=ctypes.addressof(turns), pair_axis=ctypes.addressof(axis),
                          q_weight=None, k_weight=None, position_type=2, axes=1, half_split=0, eps=1e-6)
    strides = (ctypes.c_int64 * 3)(1024, 256, 128)
    assert lib.ovc_rotary_qk(p, strides, p, strides, 1, 1, 4, 2, 2, ctypes.byref(plan), p, p, None) == -1
    assert lib.ovc_prepare_rotary(p, p, p, 1, 1, 128, 1, ctypes.byref(plan), p, p, p, p, p, p, p, None, None) == -1


def test_plan_refuses_thetas_that_fractional_positions_cannot_take():
    with pytest.raises(ValueError, match="fractional"):
        _float_plan_on_meta(theta=1e-30)


def _float_plan_on_meta(**options):
    class Positions(torch.Tensor):
        is_cuda = True

    return open_vc_attn.rotary_plan(torch.zeros(4, 1).as_subclass(Positions), axes=(128,), **options)


@pytest.mark.parametrize("eps", [1e39, float("inf"), -1e-30])
def test_plan_refuses_an_eps_that_float32_cannot_hold(eps):
    with pytest.raises(ValueError, match="eps"):
        _float_plan_on_meta(eps=eps)
