"""Rotary positions with several axes, with the RMS norm of the query and key heads (host side of ovc_rotary_qk and of the
FP8 preparation that rotates, include/ovc.h).

Video and image transformers turn each pair of a head's channels by an angle that grows with the token's position along one
axis (frame, row or column); many normalise the head first.  Both happen right before attention, so here they are one pass
over Q and K (``rotary_qk``), or no pass at all: the FP8 preparation rotates the values it quantises
(``attention(..., rotary=plan)``).  The reference leaves the rotation to its callers.
"""

import ctypes
import math
from dataclasses import dataclass

import torch

from . import _lib

_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


@dataclass(frozen=True, eq=False)
class RotaryPlan:
    """What ``rotary_plan`` laid out; kept by the caller for as long as positions and weights stay the same."""

    positions: torch.Tensor
    axes: tuple
    interleaved: bool
    q_weight: torch.Tensor
    k_weight: torch.Tensor
    eps: float
    turns: tuple
    pair_axis: tuple
    arguments: object  # the C struct; points into the tensors above

    def check(self, q, k, name="rotary"):
        """Raise unless the plan fits Q and K ([S,H,128] or [B,S,H,128])."""
        if not isinstance(self, RotaryPlan):
            raise TypeError(f"{name} must be a plan made by rotary_plan")
        batch = q.shape[0] if q.ndim == 4 else 1
        s = q.shape[-3]
        if k.shape[-3] != s or (q.ndim == 4 and k.shape[0] != batch):
            raise ValueError("Rotary positions need Q and K of the same tokens")
        if self.positions.device != q.device:
            raise ValueError("Rotary positions must reside with Q and K")
        if tuple(self.positions.shape[:-1]) not in ((s,), (batch, s)):
            raise ValueError(f"Rotary positions are for {tuple(self.positions.shape[:-1])} tokens, Q and K have {(batch, s)}")


def rotary_plan(positions, *, axes=(44, 42, 42), theta=10000.0, interleaved=True, frequencies="axis", q_weight=None,
                k_weight=None, eps=1e-6):
    """Lay out a rotation for tokens at ``positions``.

    positions    [S, A], or [B, S, A] for a batch with positions of its own: CUDA, int32, int64 or float32 (fractional
                 positions are allowed).  ``grid_positions`` makes those of a clip.
    axes         channels of each of the A axes, in the order of the head's channels: even, 128 in all or fewer; channels
                 behind them stay as they are (interleaved pairs only).
    theta        pair i of an axis with d channels turns by theta^(-2 i / d) radians per position.  With
                 ``frequencies="head"`` i and d count over all axes together (sections of one set of frequencies).
    interleaved  a pair is two neighbouring channels; otherwise channels i and i + 64.
    q_weight, k_weight  [128] or None: RMS norm of each head of Q / K before the rotation, x * weight / sqrt(mean(x^2) + eps).
                 Weights are taken over as float32 at this point.

    Two host threads or streams may use one plan at once; it is not written after this call.
    """
    if not isinstance(positions, torch.Tensor) or positions.ndim not in (2, 3) or positions.dtype not in _POSITION_TYPES:
        raise ValueError("positions must be an int32, int64 or float32 tensor [S, axes] or [B, S, axes]")
    axes = tuple(int(d) for d in axes)
    total = sum(axes)
    if not axes or any(d < 2 or d % 2 for d in axes) or total > 128:
        raise ValueError("axes must be even channel counts, 128 in all at most")
    if positions.shape[-1] != len(axes):
        raise ValueError(f"positions have {positions.shape[-1]} axes, {len(axes)} are described")
    if not interleaved and total != 128:
        raise ValueError("pairs of channels i and i + 64 need axes of 128 channels in all")
    if frequencies not in ("axis", "head"):
        raise ValueError("frequencies must be axis or head")
    if not (math.isfinite(theta) and theta > 0.0):
        raise ValueError("theta must be positive and finite")
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError("eps must be finite and not negative")
    if not positions.is_cuda:
        raise ValueError("positions must reside on a CUDA device")
    if positions.requires_grad:
        raise ValueError("Forward inference only; detach inputs explicitly")
    weights = []
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            if tuple(w.shape) != (128,) or not w.is_floating_point() or w.device != positions.device:
                raise ValueError(f"{name} must be a floating-point tensor of 128 values with the positions")
            w = w.detach().float().contiguous()
        weights.append(w)
    pair_axis = [a for a, d in enumerate(axes) for _ in range(d // 2)]
    if frequencies == "axis":
        exponents = [2.0 * i / d for d in axes for i in range(d // 2)]
    else:
        exponents = [2.0 * i / total for i in range(total // 2)]
    turns = [float(theta) ** -e / (2.0 * math.pi) for e in exponents]
    rest = 64 - len(turns)
    turns, pair_axis = turns + [0.0] * rest, pair_axis + [0] * rest
    positions = positions.contiguous()
    host = ((ctypes.c_double * 64)(*turns), (ctypes.c_uint8 * 64)(*pair_axis))
    arguments = _lib.OvcRotary(
        positions.data_ptr(), positions.shape[-2] * positions.shape[-1] if positions.ndim == 3 else 0, ctypes.addressof(host[0]),
        ctypes.addressof(host[1]), *[None if w is None else w.data_ptr() for w in weights], _POSITION_TYPES[positions.dtype],
        len(axes), 0 if interleaved else 1, eps,
    )
    return RotaryPlan(positions, axes, bool(interleaved), *weights, float(eps), host[0], host[1], arguments)


def grid_positions(frames, height, width, *, text=0, start=(0, 0, 0), device="cuda"):
    """int32 [text + frames * height * width, 3]: (frame, row, column) of a clip's patches in raster order, counted from
    ``start``, behind ``text`` tokens at (0, 0, 0), which a rotation leaves as they are."""
    if min(frames, height, width) < 1 or text < 0:
        raise ValueError("a clip has at least one frame, row and column, and text must not be negative")
    at = [torch.arange(n, device=device, dtype=torch.int32) + int(o) for n, o in zip((frames, height, width), start)]
    clip = torch.stack(torch.meshgrid(*at, indexing="ij"), -1).reshape(-1, 3)
    return torch.cat([clip.new_zeros((text, 3)), clip]) if text else clip


def readable(t):
    """``t`` itself where its heads can be read in place by 16-byte accesses, else a dense copy."""
    strides = t.stride()
    if strides[-1] == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in strides[:-1]):
        return t
    return t.contiguous()


def rotary_qk(q, k, plan):
    """Rotated (and, with weights, normalised) Q and K, in new dense tensors of their types.

    q [S,Hq,128] or [B,S,Hq,128], k with the same tokens and any number of heads, float16 or bfloat16.  Slices of a fused
    projection are read in place.  float32 inside (angles in float64), rounded once.
    """
    if q.ndim not in (3, 4) or k.ndim != q.ndim or q.shape[-1] != 128 or k.shape[-1] != 128 or min(q.shape[-2], k.shape[-2]) < 1:
        raise ValueError("Expected [S,H,128] or [B,S,H,128] Q/K")
    if not q.is_cuda or k.device != q.device:
        raise ValueError("Q/K must reside on the same CUDA device")
    if q.requires_grad or k.requires_grad:
        raise ValueError("Forward inference only; detach inputs explicitly")
    if k.dtype != q.dtype:
        raise ValueError("Expected matching dtypes")
    code = _lib.dtype_code(q.dtype)
    RotaryPlan.check(plan, q, k, "plan")
    lib = _lib.load()
    with torch.cuda.device(q.device):
        q_out, k_out = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
        if q.numel() == 0:
            return q_out, k_out
        q, k = readable(q), readable(k)
        batch = q.shape[0] if q.ndim == 4 else 1
        strides = [(ctypes.c_int64 * 3)(*((0,) * (4 - t.ndim) + t.stride()[:-1])) for t in (q, k)]
        _lib.check(
            lib.ovc_rotary_qk(
                q.data_ptr(), strides[0], k.data_ptr(), strides[1], code, batch, q.shape[-3], q.shape[-2], k.shape[-2],
                ctypes.byref(plan.arguments), q_out.data_ptr(), k_out.data_ptr(), _lib.stream_pointer(q.device),
            ),
            "ovc_rotary_qk",
        )
    return q_out, k_out


def quantize_qk(q, k, plan):
    """fp8_quantize_per_block of rotated Q and K: (q codes, q descale, k codes, k descale), one launch."""
    batch = q.shape[0] if q.ndim == 4 else 1
    s, h = q.shape[-3:-1]
    blocks = (s + 127) // 128
    lib = _lib.load()
    q8, k8 = [torch.empty((batch, s, h, 128), dtype=torch.float8_e4m3fn, device=q.device) for _ in range(2)]
    qs, ks = [torch.empty((batch, h, blocks), dtype=torch.float32, device=q.device) for _ in range(2)]
    _lib.check(
        lib.ovc_quantize_qk_rotary(
            q.data_ptr(), k.data_ptr(), _lib.dtype_code(q.dtype), batch, s, h, ctypes.byref(plan.arguments), q8.data_ptr(),
            k8.data_ptr(), qs.data_ptr(), blocks, ks.data_ptr(), blocks, _lib.stream_pointer(q.device),
        ),
        "ovc_quantize_qk_rotary",
    )
    return q8, qs, k8, ks
