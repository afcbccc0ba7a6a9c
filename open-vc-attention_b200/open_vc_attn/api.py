"""Public inference API: same names, arguments and errors as src/open_vc_attn/api.py of the reference.

The interface (signatures, dataclass fields, validation rules and messages) derives from open-vc-attention
0.3.0, BSD 3-Clause, Copyright (c) 2022 the respective contributors; see NOTICE at the repository root.
"""

from dataclasses import dataclass

import torch

from . import _lib
from ._dispatch import DEFAULT_MID_WINDOW_BLOCKS, DEFAULT_VERSION, require_version
from .rotary import RotaryPlan, prepare_rotary


def raw_forward(q, k, v, *, version=DEFAULT_VERSION, **kwargs):
    """Advanced kernel interface: FP8 inputs plus the kernel's own keyword contract.

    Forward only: gradients are rejected.  Returns (output, optional LSE).
    """
    if any(t.requires_grad for t in (q, k, v)):
        raise ValueError("open_vc_attn is an inference API; detach inputs explicitly")
    require_version(version)
    from .forward import flash_attn_fwd

    with torch.cuda.device(q.device):
        return flash_attn_fwd(q, k, v, **kwargs)[:2]


def validate_qkv(q, k, v, *, floating=True):
    if q.ndim not in (3, 4) or k.ndim != q.ndim or v.ndim != q.ndim:
        raise ValueError("Expected [S,H,128] or [B,S,H,128] Q/K/V")
    for t in (q, k, v):
        if t.shape[-1] != 128 or t.numel() < 1:
            raise ValueError("The convenience API requires nonempty D=128 inputs")
    if k.shape != v.shape or q.shape[-2:] != k.shape[-2:]:
        raise ValueError("The convenience API requires MHA and matching K/V shapes")
    if q.ndim == 4 and q.shape[0] != k.shape[0]:
        raise ValueError("Q/K/V batch sizes must match")
    device = q.device
    if not q.is_cuda or k.device != device or v.device != device:
        raise ValueError("Q/K/V must reside on the same CUDA device")
    if q.requires_grad or k.requires_grad or v.requires_grad:
        raise ValueError("Forward inference only; detach inputs explicitly")
    allowed = (torch.float16, torch.bfloat16) if floating else (torch.float8_e4m3fn,)
    if q.dtype not in allowed or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"Expected matching dtypes from {allowed}")
    # The reference also admits SM103 (api.py:43-44); libovc.so holds sm_100a code only.
    if _lib.capability(device) != (10, 0):
        raise ValueError("This release validates Blackwell SM100 (B200) only")


def _layout(q, k, v, bounds=None):
    """``bounds``: int32 [2] that the preparation will set to [0, S], where Q and K have the same tokens."""
    original_shape = tuple(q.shape)
    if q.ndim == 3 or q.shape[0] == 1:
        q, k, v = [(t if t.ndim == 3 else t[0]).contiguous() for t in (q, k, v)]
        sq, sk = q.shape[0], k.shape[0]
        # [0, S], built on the device (one launch) so that the call stays capturable in a CUDA graph.
        cu_q = torch.arange(0, sq + 1, sq, device=q.device, dtype=torch.int32) if bounds is None else bounds
        kwargs = {
            "cu_seqlens_q": cu_q,
            "cu_seqlens_k": cu_q if sk == sq else torch.arange(0, sk + 1, sk, device=q.device, dtype=torch.int32),
            "max_seqlen_q": sq,
            "max_seqlen_k": sk,
        }
    else:
        q, k, v = [t.contiguous() for t in (q, k, v)]
        kwargs = {}
    return q, k, v, kwargs, original_shape


@dataclass(frozen=True)
class PreparedFP8:
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    q_descale: torch.Tensor
    k_descale: torch.Tensor
    v_descale: torch.Tensor
    layout: dict
    output_shape: tuple
    v_prepacked: bool = False


def _packed_dsl_available():
    """The packed path is compiled ahead of time here, so it is always available."""
    return True


def _fused_preparation_eligible(q, k, v, *, version, mode, causal, return_lse):
    """Which calls take the fused, packed preparation (src/open_vc_attn/api.py:86-99)."""
    return (
        version == DEFAULT_VERSION
        and mode == "expcast"
        and not causal
        and not return_lse
        and (q.ndim == 3 or (q.ndim == 4 and q.shape[0] == 1))
        and q.shape == k.shape == v.shape
        and q.shape[-3] >= 32768
        and all(t.is_contiguous() for t in (q, k, v))
        and _lib.capability(q.device) == (10, 0)
        and _packed_dsl_available()
    )


def prepare_fp8(q, k, v, *, rotary=None):
    """Q/K: per 128 tokens per head; V: per sequence per head; E4M3 max 448.

    The returned tensors retain descales in FP32.  Preparation is stream ordered.
    ``rotary`` (from ``rotary_plan``): Q and K are normalised and rotated on the way, without a rounding to 16 bits.
    """
    validate_qkv(q, k, v)
    if rotary is not None:
        RotaryPlan.check(rotary, q, k)
        with _lib.on_device(q.device):
            bounds = q.new_empty(2, dtype=torch.int32) if q.ndim == 3 or q.shape[0] == 1 else None
            q, k, v, layout, shape = _layout(q, k, v, bounds)
            return PreparedFP8(*prepare_rotary(q, k, v, rotary, bounds), layout, shape)
    from .quantization import fp8_quantize_per_block, fp8_quantize_per_head

    with _lib.on_device(q.device):
        q, k, v, layout, shape = _layout(q, k, v)
        q8, qs = fp8_quantize_per_block(q, block_l=128)
        k8, ks = fp8_quantize_per_block(k, block_l=128)
        v8, vs = fp8_quantize_per_head(v)
        if q.ndim == 3:
            q8, k8, v8 = q8[0], k8[0], v8[0]
        return PreparedFP8(q8, k8, v8, qs, ks, vs, layout, shape)


def prepare_fp8_fused(q, k, v, *, cu_seqlens=None, rotary=None):
    """Three-kernel B200 preparation; returns V already in the packed layout.

    Dense single-sequence self-attention only, S >= 32768, D=128.  Optional contiguous int32 CUDA
    metadata must contain [0, S]; the caller owns its values.  ``rotary`` as for ``prepare_fp8``.
    """
    from .preparation import prepare_fp8_fused as implementation

    return implementation(q, k, v, cu_seqlens=cu_seqlens, rotary=rotary)


def attention_fp8(
    prepared,
    *,
    version=DEFAULT_VERSION,
    causal=False,
    softmax_scale=None,
    mid_window_blocks=DEFAULT_MID_WINDOW_BLOCKS,
    return_lse=False,
):
    """Run prepared FP8 ExpCast attention, using a four-block mid-window scan by default.

    ``mid_window_blocks=None`` restores the plain right-to-left scan.  Generic prepared inputs have
    V packed inside this call; fused prepared inputs already contain packed V.
    """
    if version != DEFAULT_VERSION:
        raise ValueError(f"Prepared FP8 attention requires version={DEFAULT_VERSION!r}")
    flags = {"expcast": True}
    if getattr(prepared, "v_prepacked", False):
        if causal or return_lse:
            raise ValueError("Prepacked V requires dense Open-VC ExpCast without LSE")
        flags["v_prepacked"] = True
    out, lse = raw_forward(
        prepared.q,
        prepared.k,
        prepared.v,
        version=version,
        q_descale=prepared.q_descale,
        k_descale=prepared.k_descale,
        v_descale=prepared.v_descale,
        **prepared.layout,
        **flags,
        causal=causal,
        softmax_scale=softmax_scale,
        mid_window_blocks=None if causal else mid_window_blocks,
        return_lse=return_lse,
    )
    out = out.reshape(prepared.output_shape)
    return (out, lse) if return_lse else out


def attention(
    q,
    k,
    v,
    *,
    version=DEFAULT_VERSION,
    mode="expcast",
    causal=False,
    softmax_scale=None,
    mid_window_blocks=DEFAULT_MID_WINDOW_BLOCKS,
    return_lse=False,
    preparation="auto",
    rotary=None,
):
    """BF16/FP16 in, BF16 attention out, FP8 quantisation included.

    A 3-D tensor is one sequence; 4-D tensors are independent batch items.  ``preparation='auto'``
    fuses preparation for eligible long single-sequence calls, ``'unfused'`` keeps the general
    preparation and ``'fused'`` requires the packed contract.  ``mode="bf16"`` belongs to the
    reference's second backend, which this build does not contain: it raises.
    ``rotary`` (from ``rotary_plan``): Q and K are given as projected; the preparation normalises and rotates them.
    """
    validate_qkv(q, k, v)
    if rotary is not None:
        RotaryPlan.check(rotary, q, k)
    if mode not in ("bf16", "expcast"):
        raise ValueError("mode must be bf16 or expcast")
    if (mode == "bf16") != (version == "reference"):
        raise ValueError('mode="bf16" requires version="reference"; ExpCast requires Open-VC')
    require_version(version)
    if preparation not in ("auto", "unfused", "fused"):
        raise ValueError("preparation must be auto, unfused, or fused")
    fuse = preparation != "unfused" and _fused_preparation_eligible(
        q, k, v, version=version, mode=mode, causal=causal, return_lse=return_lse
    )
    if preparation == "fused" and not fuse:
        raise ValueError(
            "Fused preparation requires contiguous B200 single-sequence self-attention, "
            "S >= 32768, DSL 4.6.2, dense Open-VC ExpCast and no LSE"
        )
    return attention_fp8(
        prepare_fp8_fused(q, k, v, rotary=rotary) if fuse else prepare_fp8(q, k, v, rotary=rotary),
        version=version,
        causal=causal,
        softmax_scale=softmax_scale,
        mid_window_blocks=mid_window_blocks,
        return_lse=return_lse,
    )
