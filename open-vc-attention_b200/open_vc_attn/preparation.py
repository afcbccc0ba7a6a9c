"""Fused preparation of one long sequence for the packed attention path.

Host side of ovc_prepare_fused; mirrors prepare_fp8_fused of the reference
(src/open_vc_attn/preparation.py:83-162): same validation and messages, same result layout.
"""

import torch

from . import _lib
from .rotary import RotaryPlan


def prepare_fp8_fused(q, k, v, *, cu_seqlens=None, rotary=None):
    """Prepare contiguous [S,H,128] or [1,S,H,128] self-attention for B200.

    Requires S >= 32768.  Pass existing int32 CUDA [0,S] metadata to have it reused by identity;
    its values are the caller's contract.  Nothing here synchronises with the host.  With ``rotary`` (from
    ``rotary_plan``) Q and K are normalised and rotated in the launch that quantises them.
    """
    from .api import PreparedFP8, validate_qkv

    validate_qkv(q, k, v)
    if (q.ndim == 4 and q.shape[0] != 1) or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("Fused preparation requires single-sequence [S,H,128] self-attention")
    if q.shape[-3] < 32768 or any(not t.is_contiguous() for t in (q, k, v)):
        raise ValueError("Fused preparation requires contiguous Q/K/V and S >= 32768")
    if _lib.capability(q.device) != (10, 0):
        raise ValueError("Fused preparation is currently validated for B200 only")
    if rotary is not None:
        RotaryPlan.check(rotary, q, k)
    shape = tuple(q.shape)
    q, k, v = [t if t.ndim == 3 else t[0] for t in (q, k, v)]
    if cu_seqlens is not None and (
        cu_seqlens.shape != (2,)
        or cu_seqlens.dtype != torch.int32
        or cu_seqlens.device != q.device
        or not cu_seqlens.is_contiguous()
    ):
        raise ValueError("cu_seqlens must be contiguous int32 [0,S] on the QKV device")
    return _prepare_packed(q, k, v, shape, cu_seqlens, rotary)


def _prepare_packed(q, k, v, shape, cu_seqlens=None, rotary=None):
    """The three launches, without the length/device policy checks (any S >= 1)."""
    from .api import PreparedFP8

    s, h, d = q.shape
    lib = _lib.load()
    with _lib.on_device(q.device):
        bounds = None  # int32 [2] that the quantiser sets to [0, S] on the way
        if cu_seqlens is None and rotary is not None:
            cu_seqlens = bounds = q.new_empty(2, dtype=torch.int32)
        elif cu_seqlens is None:
            cu_seqlens = torch.arange(0, s + 1, s, device=q.device, dtype=torch.int32)
        blocks = (s + 127) // 128
        q_blocks = (blocks + 1) // 2 * 2
        padded = blocks * 128
        q8 = torch.empty_like(q, dtype=torch.float8_e4m3fn)
        k8 = torch.empty_like(q8)
        qs = q.new_empty((1, h, q_blocks), dtype=torch.float32)
        ks = q.new_empty((1, h, blocks), dtype=torch.float32)
        packed = q8.new_empty((h, d, padded))
        amax = q.new_empty((1, h), dtype=torch.float32)
        vs = torch.empty_like(amax)
        outputs = [t.data_ptr() for t in (q8, k8, packed, qs, ks, vs, amax)]
        stream = _lib.raw_stream(q.device.index)
        inputs = (q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.dtype_code(q.dtype), s, h)
        if rotary is None:
            _lib.check(lib.ovc_prepare_fused(*inputs, *outputs, stream), "ovc_prepare_fused")
        else:
            outputs.append(None if bounds is None else bounds.data_ptr())
            _lib.check(lib.ovc_prepare_fused_rotary(*inputs, rotary.arguments, *outputs, stream), "ovc_prepare_fused_rotary")
        result = packed[..., :s].movedim(-1, 0)
        layout = dict(cu_seqlens_q=cu_seqlens, cu_seqlens_k=cu_seqlens, max_seqlen_q=s, max_seqlen_k=s)
        return PreparedFP8(q8, k8, result, qs, ks, vs, layout, shape, v_prepacked=True)
