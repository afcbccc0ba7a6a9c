"""Attention over packed sequences in 16 bits (host side of ovc_attention_packed, include/ovc.h).

``attention`` quantises to FP8 for one long sequence (or a batch of equal ones) with as many key heads as query heads.  This is
its counterpart for what surrounds a video transformer: text encoders and autoregressive parts, whose sequences differ in
length, share key heads between query heads, mask the future or add one token at a time, and are too short or too sensitive
for FP8.  The reference's kernel interface names these options (cute/interface.py:110-179); its public functions use none.
"""

import ctypes
import math

import torch

from . import _lib
from .forward import _raise_if_flagged, _status


_Two = ctypes.c_int64 * 2
# softmax_scale, and its product with log2(e), as normal float32 numbers
_SMALLEST_SCALE, _LARGEST_SCALE = 2.0 ** -126, 2.0 ** 127


def _span(t):
    begin = t.data_ptr()
    return begin, begin + 2 * (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1)


def _overlap(a, b):
    """Whether the 16-bit tensors reach into each other's memory; one that lies in gaps of the other counts, too."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _in_place(t):
    """Elements from one token and one head of [T,H,128] to the next, as a C array; None where the rows cannot be read in
    place."""
    tokens, heads, _ = t.shape
    if t.data_ptr() % 16:
        return None
    if t.is_contiguous():
        return _Two(128 * heads, 128)
    token, head, channel = t.stride()
    # the stride of a single token or head is never used, and may be anything
    if tokens == 1:
        token = 128 * heads
    if heads == 1:
        head = 128
    if channel != 1 or token <= 0 or head <= 0 or token % 8 or head % 8:
        return None
    return _Two(token, head)


def _dense(t):
    t = t.clone(memory_format=torch.contiguous_format)
    return t, _in_place(t)


def _check_bounds(name, cu, device):
    if not isinstance(cu, torch.Tensor) or cu.dtype != torch.int32 or cu.ndim != 1 or cu.shape[0] < 2 or not cu.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of at least two bounds")
    if cu.device != device:
        raise ValueError(f"{name} must reside with Q/K/V")


def attention_packed(q, k, v, cu_seqlens_q, cu_seqlens_k=None, *, causal=False, softmax_scale=None, return_lse=False, out=None):
    """softmax(Q K^T * scale) V of each of several sequences packed behind each other, in float16 or bfloat16.

    q             [Tq,Hq,128]; k, v [Tk,Hk,128], Hq a multiple of Hk (at most 128 query heads to a key head): query head h
                  reads key head h // (Hq // Hk).  Slices of a fused projection are read in place.
    cu_seqlens_q  int32 CUDA [B+1], 0 first, not decreasing: sequence b is rows cu_seqlens_q[b] to cu_seqlens_q[b+1].  Its
                  values stay on the device; bounds outside the tensors or out of order give wrong rows, nothing worse.
    cu_seqlens_k  the same for K and V; None: that of Q.  Lengths may be zero.
    causal        token t of lq sees the keys below t + 1 + lk - lq (the last token sees every key).
    softmax_scale 1 / sqrt(128) by default.
    out           written and returned if given ([Tq,Hq,128] contiguous, Q's type, no memory of Q, K or V): rows behind the
                  last sequence stay as they were.  Without it those rows of the new tensor are zero.

    Returns out, or (out, lse) with lse [Hq,Tq] float32, the logarithm of the sum of exponentials of the scaled scores.  A
    row that sees no key is zero, whatever V holds, its lse -inf, and so is the lse of rows behind the last sequence.  Keys of
    other sequences, of the padding and of the masked future never contribute, whatever they hold; values that are not finite
    within a row's own sequence may reach rows that see some keys, but not those.  Scores, sums and the accumulator are
    float32; probabilities are rounded to the inputs' type for the second product.

    Stream ordered, no synchronisation, capturable (after a call outside of a capture, since the first one on a device allocates
    a status word).  As for ``attention``, a launch whose bounded waits expire leaves NaN and is
    reported by a later call or by ``forward.check_status``.
    """
    if q.ndim != 3 or k.ndim != 3:
        raise ValueError("Expected packed [T,H,128] Q/K/V")
    tq, hq, dim_q = q.shape
    tk, hk, dim_k = k.shape
    if dim_q != 128 or dim_k != 128:
        raise ValueError("Expected packed [T,H,128] Q/K/V")
    if k.shape != v.shape:
        raise ValueError("K and V shapes must match")
    if hk < 1 or hq < hk or hq % hk or hq // hk > 128:
        raise ValueError("Query heads must be a multiple of the key heads, 128 to each at most")
    device = q.device
    if not q.is_cuda or k.device != device or v.device != device:
        raise ValueError("Q/K/V must reside on the same CUDA device")
    if q.requires_grad or k.requires_grad or v.requires_grad:
        raise ValueError("Forward inference only; detach inputs explicitly")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("Expected matching float16 or bfloat16 Q/K/V")
    if max(tq, tk) > 1 << 30:
        raise ValueError("At most 2**30 packed rows")
    _check_bounds("cu_seqlens_q", cu_seqlens_q, device)
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    elif cu_seqlens_k is not cu_seqlens_q:
        _check_bounds("cu_seqlens_k", cu_seqlens_k, device)
    if cu_seqlens_k.shape != cu_seqlens_q.shape:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must describe the same number of sequences")
    if softmax_scale is None:
        softmax_scale = 128 ** -0.5
    if not _SMALLEST_SCALE <= softmax_scale <= _LARGEST_SCALE:
        raise ValueError("softmax_scale must be positive and finite, in float32 and times log2(e) as well")
    flags = _lib.OVC_ATTN_CAUSAL if causal else 0
    if out is None:
        flags |= _lib.OVC_ATTN_ZERO_TAIL
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != device or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor of Q's shape, type and device")
    elif out.requires_grad:
        raise ValueError("Forward inference only; detach inputs explicitly")
    elif any(_overlap(out, t) for t in (q, k, v)):
        raise ValueError("out must not share memory with Q/K/V")
    lib = _lib.load()
    _raise_if_flagged(device)
    with _lib.on_device(device):
        lse = None
        if return_lse:  # (the kernel sets what lies behind the last sequence together with the rows of out only)
            lse = q.new_empty((hq, tq), dtype=torch.float32) if out is None else q.new_full((hq, tq), -math.inf, dtype=torch.float32)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if tq == 0:
            return (out, lse) if return_lse else out
        if tk == 0:
            # Every row of every sequence sees no key.
            ends = torch.arange(tq, device=device) < cu_seqlens_q[-1]
            if flags & _lib.OVC_ATTN_ZERO_TAIL:
                out.zero_()
            else:
                out.masked_fill_(ends[:, None, None], 0)
            return (out, lse.fill_(-math.inf)) if return_lse else out
        q_strides, k_strides, v_strides = _in_place(q), _in_place(k), _in_place(v)
        if q_strides is None:
            q, q_strides = _dense(q)
        if k_strides is None:
            k, k_strides = _dense(k)
        if v_strides is None:
            v, v_strides = _dense(v)
        sizes = (cu_seqlens_q.shape[0] - 1, tq, tk, hq, hk)
        size = lib.ovc_attention_packed_workspace(*sizes)
        workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        words, mirror = _status(device)
        _lib.check(
            lib.ovc_attention_packed(
                q.data_ptr(), q_strides, k.data_ptr(), k_strides, v.data_ptr(), v_strides,
                _lib.OVC_BF16 if q.dtype == torch.bfloat16 else _lib.OVC_F16, cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(),
                *sizes, flags, softmax_scale, out.data_ptr(), None if lse is None else lse.data_ptr(),
                None if workspace is None else workspace.data_ptr(), words.data_ptr() + 4, mirror.data_ptr(),
                _lib.raw_stream(device.index),
            ),
            "ovc_attention_packed",
        )
    return (out, lse) if return_lse else out
