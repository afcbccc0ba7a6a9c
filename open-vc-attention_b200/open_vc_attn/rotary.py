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

_Three = ctypes.c_int64 * 3
_LARGEST_EPS = torch.finfo(torch.float32).max
_MOST_TURNS = 2.0 ** 30  # per float32 position: the kernels carry the whole turns in 32 bits
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


@dataclass(frozen=True, eq=False)
class RotaryPlan:
    """What ``rotary_plan`` laid out; kept by the caller for as long as positions and weights stay the same."""

    positions: torch.Tensor
    tokens: tuple
    axes: tuple
    interleaved: bool
    q_weight: torch.Tensor
    k_weight: torch.Tensor
    eps: float
    turns: object
    pair_axis: object
    arguments: object  # a pointer to the C struct, which points into the members above

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
        tokens = self.tokens
        if tokens != (s,) and tokens != (batch, s):
            raise ValueError(f"Rotary positions are for {tokens} tokens, Q and K have {(batch, s)}")


def rotary_plan(positions, *, axes=(44, 42, 42), theta=10000.0, interleaved=True, frequencies="axis", q_weight=None,
                k_weight=None, eps=1e-6):
    """Lay out a rotation for tokens at ``positions``.

    positions    [S, A], or [B, S, A] for a batch with positions of its own: CUDA, int32, int64 or float32 (fractional
                 positions are allowed).  ``grid_positions`` makes those of a clip.  Contiguous ones are referred to and read by
                 every call and replay, so that a captured step may count on in place; others are copied here.
    axes         channels of each of the A axes, in the order of the head's channels: even, 128 in all or fewer; channels
                 behind them are not turned (interleaved pairs only): without a norm they stay as they are, whatever they hold.
    theta        pair i of an axis with d channels turns by theta^(-2 i / d) radians per position (below 2^30 turns, where
                 positions are float32).  With ``frequencies="head"`` i and d count over all axes together (sections of one
                 set of frequencies).
    interleaved  a pair is two neighbouring channels; otherwise channels i and i + 64.
    q_weight, k_weight  [128] or None: RMS norm of each head of Q / K before the rotation, x * weight / sqrt(mean(x^2) + eps).
                 Weights are copied here, as float32.

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
    if not 0.0 <= eps <= _LARGEST_EPS:
        raise ValueError("eps must be finite, in float32 as well, and not negative")
    if not positions.is_cuda:
        raise ValueError("positions must reside on a CUDA device")
    if positions.requires_grad:
        raise ValueError("Forward inference only; detach inputs explicitly")
    weights = []
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            if tuple(w.shape) != (128,) or not w.is_floating_point() or w.device != positions.device:
                raise ValueError(f"{name} must be a floating-point tensor of 128 values with the positions")
            w = w.detach().to(torch.float32, copy=True, memory_format=torch.contiguous_format)
        weights.append(w)
    pair_axis = [a for a, d in enumerate(axes) for _ in range(d // 2)]
    if frequencies == "axis":
        exponents = [2.0 * i / d for d in axes for i in range(d // 2)]
    else:
        exponents = [2.0 * i / total for i in range(total // 2)]
    try:
        turns = [float(theta) ** -e / (2.0 * math.pi) for e in exponents]
    except OverflowError:
        raise ValueError("theta is too small: its frequencies overflow") from None
    if positions.dtype == torch.float32 and max(turns) >= _MOST_TURNS:
        raise ValueError("theta is too small for fractional positions: at most 2**30 turns per position")
    rest = 64 - len(turns)
    turns, pair_axis = turns + [0.0] * rest, pair_axis + [0] * rest
    positions = positions.contiguous()
    host = ((ctypes.c_double * 64)(*turns), (ctypes.c_uint8 * 64)(*pair_axis))
    arguments = _lib.OvcRotary(
        positions.data_ptr(), positions.shape[-2] * positions.shape[-1] if positions.ndim == 3 else 0, ctypes.addressof(host[0]),
        ctypes.addressof(host[1]), *[None if w is None else w.data_ptr() for w in weights], _POSITION_TYPES[positions.dtype],
        len(axes), 0 if interleaved else 1, eps,
    )
    return RotaryPlan(positions, tuple(positions.shape[:-1]), axes, bool(interleaved), *weights, float(eps), *host, ctypes.pointer(arguments))


def grid_positions(frames, height, width, *, text=0, start=(0, 0, 0), device="cuda"):
    """int32 [text + frames * height * width, 3]: (frame, row, column) of a clip's patches in raster order, counted from
    ``start``, behind ``text`` tokens at (0, 0, 0), which a rotation leaves as they are."""
    if min(frames, height, width) < 1 or text < 0:
        raise ValueError("a clip has at least one frame, row and column, and text must not be negative")
    at = [torch.arange(n, device=device, dtype=torch.int32) + int(o) for n, o in zip((frames, height, width), start)]
    clip = torch.stack(torch.meshgrid(*at, indexing="ij"), -1).reshape(-1, 3)
    return torch.cat([clip.new_zeros((text, 3)), clip]) if text else clip


def _strides(t):
    """Elements from one batch item, token and head of [S,H,128] or [B,S,H,128] to the next, as a C array; None where the heads
    cannot be read in place by 16-byte accesses."""
    shape = t.shape
    if t.is_contiguous():
        token = 128 * shape[-2]
        return None if t.data_ptr() % 16 else _Three(shape[-3] * token, token, 128)
    stride = t.stride()
    if stride[-1] != 1 or t.data_ptr() % 16:
        return None
    # the stride of a dimension of one entry is never used, and may be anything
    used = [0 if n == 1 else s for n, s in zip(shape[:-1], stride)]
    if any(s % 8 for s in used):
        return None
    return _Three(*used) if len(used) == 3 else _Three(0, *used)


def rotary_qk(q, k, plan):
    """Rotated (and, with weights, normalised) Q and K, in new dense tensors of their types.

    q [S,Hq,128] or [B,S,Hq,128], k with the same tokens and any number of heads, float16 or bfloat16.  Slices of a fused
    projection are read in place.  float32 inside (angles in 64-bit fixed point), rounded once.
    """
    if q.ndim not in (3, 4) or k.ndim != q.ndim or q.shape[-1] != 128 or k.shape[-1] != 128 or min(q.shape[-2], k.shape[-2]) < 1:
        raise ValueError("Expected [S,H,128] or [B,S,H,128] Q/K")
    device = q.device
    if not q.is_cuda or k.device != device:
        raise ValueError("Q/K must reside on the same CUDA device")
    if q.requires_grad or k.requires_grad:
        raise ValueError("Forward inference only; detach inputs explicitly")
    if k.dtype != q.dtype:
        raise ValueError("Expected matching dtypes")
    code = _lib.dtype_code(q.dtype)
    RotaryPlan.check(plan, q, k, "plan")
    lib = _lib.load()
    with _lib.on_device(device):
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        if q.numel() == 0:
            return q_out, k_out
        q_strides, k_strides = _strides(q), _strides(k)
        if q_strides is None:
            q = q.clone(memory_format=torch.contiguous_format)
            q_strides = _strides(q)
        if k_strides is None:
            k = k.clone(memory_format=torch.contiguous_format)
            k_strides = _strides(k)
        _lib.check(
            lib.ovc_rotary_qk(
                q.data_ptr(), q_strides, k.data_ptr(), k_strides, code, q.shape[0] if q.ndim == 4 else 1, q.shape[-3],
                q.shape[-2], k.shape[-2], plan.arguments, q_out.data_ptr(), k_out.data_ptr(), _lib.raw_stream(device.index),
            ),
            "ovc_rotary_qk",
        )
    return q_out, k_out


def prepare_rotary(q, k, v, plan, bounds=None):
    """fp8_quantize_per_block of rotated Q and K and fp8_quantize_per_head of V, dense inputs: codes of the inputs' shapes, and
    the descales of Q, K [B,H,blocks] and V [B,H].  ``bounds``: int32 [2] to be set to [0, S] (one sequence)."""
    s, h, _ = q.shape[-3:]
    batch = q.shape[0] if q.ndim == 4 else 1
    q8, k8, v8 = [torch.empty_like(t, dtype=torch.float8_e4m3fn) for t in (q, k, v)]
    qs = q.new_empty((batch, h, (s + 127) // 128), dtype=torch.float32)
    ks = torch.empty_like(qs)
    vs = q.new_empty((batch, h), dtype=torch.float32)
    amax = torch.empty_like(vs)
    _lib.check(
        _lib.load().ovc_prepare_rotary(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.dtype_code(q.dtype), batch, s, h, plan.arguments,
            q8.data_ptr(), k8.data_ptr(), v8.data_ptr(), qs.data_ptr(), ks.data_ptr(), vs.data_ptr(), amax.data_ptr(),
            None if bounds is None else bounds.data_ptr(), _lib.raw_stream(q.device.index),
        ),
        "ovc_prepare_rotary",
    )
    return q8, k8, v8, qs, ks, vs
