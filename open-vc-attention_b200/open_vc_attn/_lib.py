"""ctypes binding of libovc.so (declared in include/ovc.h).

The library is the product: when it is missing or a call fails this module raises; there is no
PyTorch or CPU fallback.
"""

import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIBRARY_PATH = os.path.join(os.path.dirname(_HERE), "lib", "libovc.so")

OVC_F16, OVC_BF16 = 0, 1
OVC_ATTN_CAUSAL, OVC_ATTN_V_UNPACKED = 1, 2  # flags of ovc_attention_ex
OVC_ATTN_ZERO_TAIL = 4  # and, with OVC_ATTN_CAUSAL, of ovc_attention_packed
STATUS_WAIT_EXPIRED = 1

_p, _i, _l, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


class OvcRotary(ctypes.Structure):
    """struct ovc_rotary of include/ovc.h."""

    _fields_ = [
        ("positions", _p), ("position_batch_stride", _l), ("turns", _p), ("pair_axis", _p), ("q_weight", _p), ("k_weight", _p),
        ("position_type", _i), ("axes", _i), ("half_split", _i), ("eps", _f),
    ]


SIGNATURES = {
    "ovc_version": (_i, []),
    "ovc_error_string": (ctypes.c_char_p, [_i]),
    "ovc_last_cuda_error": (_i, []),
    "ovc_quantize_per_block": (_i, [_p, _i, _l, _l, _l, _p, _p, _l, _p]),
    "ovc_head_amax": (_i, [_p, _i, _l, _l, _l, _p, _p]),
    "ovc_quantize_per_head": (_i, [_p, _i, _l, _l, _l, _p, _p, _p, _p]),
    "ovc_prepare_fused": (_i, [_p, _p, _p, _i, _l, _l, _p, _p, _p, _p, _p, _p, _p, _p]),
    "ovc_prepare_fused_static": (_i, [_p, _p, _p, _i, _l, _l, _p, _p, _p, _p, _p, _p, _p]),
    "ovc_pack_v": (_i, [_p, _l, _l, _l, _p, _p]),
    "ovc_div_full": (_i, [_p, _p, _p, _l, _p]),
    "ovc_repair_score": (_i, [_p, _i, _l, _l, _p, _p, _p, _p]),
    "ovc_repair_rows": (_i, [_p, _p, _p, _i, _p, _p, _p, _p, _l, _l, _l, _l, _l, _p]),
    "ovc_attention": (_i, [_p, _p, _p, _p, _l, _p, _p, _p, _l, _p, _l, _l, _l, _l, _f, _i, _p, _p]),
    "ovc_bench_conversion": (_i, [_p, _l, _l, _p]),
    "ovc_selftest_wait": (_i, [_p, _l, _p, _p]),
    "ovc_copy_head_slice": (_i, [_p, _l, _l, _p, _l, _l, _l, _l, _l, _i, _p]),
    "ovc_attention_ex": (_i, [_p, _p, _p, _p, _l, _p, _p, _p, _l, _p, _p, _i, _l, _l, _l, _l, _f, _i, _p, _p]),
    "ovc_attention_packed": (_i, [_p, _p, _p, _p, _p, _p, _i, _p, _p, _l, _l, _l, _l, _l, _i, _f, _p, _p, _p, _p, _p, _p]),
    "ovc_attention_packed_workspace": (_l, [_l, _l, _l, _l, _l]),
    "ovc_rotary_qk": (_i, [_p, _p, _p, _p, _i, _l, _l, _l, _l, _p, _p, _p, _p]),
    "ovc_prepare_rotary": (_i, [_p, _p, _p, _i, _l, _l, _l, _p, _p, _p, _p, _p, _p, _p, _p, _p, _p]),
    "ovc_prepare_fused_rotary": (_i, [_p, _p, _p, _i, _l, _l, _p, _p, _p, _p, _p, _p, _p, _p, _p, _p]),
    "ovc_vs_assign": (_i, [_p, _p, _p, _l, _l, _l, _p]),
    "ovc_vs_accumulate": (_i, [_p, _p, _p, _p, _l, _l, _l, _p]),
    "ovc_vs_update_centers": (_i, [_p, _p, _p, _l, _l, _p]),
    "ovc_vs_block_stats": (_i, [_p, _p, _p, _p, _l, _l, _p]),
    "ovc_vs_block_write": (_i, [_p, _p, _p, _p, _p, _p, _p, _p, _p, _l, _l, _p]),
    "ovc_cast_e4m3": (_i, [_p, _i, _p, _l, _p]),
    "ovc_attention_vsmooth_workspace": (_l, [_l, _l]),
    "ovc_attention_vsmooth": (_i, [_p, _p, _p, _p, _p, _p, _p, _p, _l, _l, _l, _f, _i, _p, _p]),
}

_lib = None


def load():
    """Load libovc.so once and declare every entry point's signature."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIBRARY_PATH):
            raise RuntimeError(
                f"{LIBRARY_PATH} is missing: build it with `python open-vc-attention_b200/build.py` "
                "(needs nvcc); open_vc_attn has no fallback path"
            )
        lib = ctypes.CDLL(LIBRARY_PATH)
        for name, (restype, argtypes) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = restype, argtypes
        _lib = lib
    return _lib


def check(code, what):
    if code != 0:
        lib = load()
        text = lib.ovc_error_string(code).decode()
        raise RuntimeError(f"{what} failed: {text} (code {code}, cuda error {lib.ovc_last_cuda_error()})")


def dtype_code(dtype):
    import torch

    if dtype == torch.float16:
        return OVC_F16
    if dtype == torch.bfloat16:
        return OVC_BF16
    raise ValueError(f"Expected float16 or bfloat16, got {dtype}")


def stream_pointer(device):
    import torch

    return torch.cuda.current_stream(device).cuda_stream


def raw_stream(index):
    """The current stream of device ``index`` as stream_pointer gives it, without making a Stream object (2 us less a call)."""
    import torch

    return torch._C._cuda_getCurrentRawStream(index)


_capabilities = {}


def capability(device):
    """torch.cuda.get_device_capability, asked for once per device."""
    have = _capabilities.get(device.index)
    if have is None:
        import torch

        have = _capabilities[device.index] = torch.cuda.get_device_capability(device)
    return have


class on_device:
    """Makes ``device`` current for a with block; costs nothing where it is current already."""

    __slots__ = ("guard",)

    def __init__(self, device):
        import torch

        self.guard = None if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exception):
        if self.guard is not None:
            self.guard.__exit__(*exception)
