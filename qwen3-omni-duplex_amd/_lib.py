"""ctypes binding of libi4moe.so, the C ABI declared in include/i4moe.h.

Only plain pointers, sizes and a hipStream_t cross the boundary.  torch is used
by the callers for device memory and the current stream; nothing here falls
back to a CPU or torch implementation: if the library is missing or was built
for another ABI version, every entry point raises.
"""
from __future__ import annotations

import ctypes
from ctypes import POINTER, c_char_p, c_int, c_int32, c_int64, c_size_t, c_void_p
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "libi4moe.so"
ABI_VERSION = 9
ERR_WORKSPACE = -7  # I4_ERR_WORKSPACE
ERR_HANDOFF = -10  # I4_ERR_HANDOFF: the one code a kernel stores in a status word

# element types and layouts (include/i4moe.h)
F32, F16, BF16 = 0, 1, 2
LAYOUT_CT, LAYOUT_AWQ, LAYOUT_TILE = 0, 1, 2
LAYOUTS = {"ct": LAYOUT_CT, "awq": LAYOUT_AWQ, "tile": LAYOUT_TILE}

_DT = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


class QWeightC(ctypes.Structure):
    """struct i4_qweight"""

    _fields_ = [
        ("packed", c_void_p),
        ("scale", c_void_p),
        ("zeros", c_void_p),
        ("packed_estride", c_int64),
        ("scale_estride", c_int64),
        ("zeros_estride", c_int64),
        ("layout", c_int32),
        ("group", c_int32),
        ("scale_dtype", c_int32),
        ("E", c_int32),
        ("N", c_int32),
        ("K", c_int32),
    ]


class MoeWeightsC(ctypes.Structure):
    """struct i4_moe_weights"""

    _fields_ = [("gate_up", QWeightC), ("down", QWeightC), ("router_w", c_void_p),
                ("norm_w", c_void_p), ("norm_eps", ctypes.c_float),
                ("gate_up_tile", QWeightC), ("down_tile", QWeightC)]


class DWeightC(ctypes.Structure):
    """struct i4_dweight"""

    _fields_ = [("data", c_void_p), ("scale", c_void_p), ("E", c_int32), ("N", c_int32),
                ("K", c_int32)]


class DmoeWeightsC(ctypes.Structure):
    """struct i4_dmoe_weights"""

    _fields_ = [("gate_up", DWeightC), ("down", DWeightC), ("router_w", c_void_p),
                ("shared_gate_up", DWeightC), ("shared_down", DWeightC),
                ("shared_gate_w", c_void_p)]


class ThinkerLayerC(ctypes.Structure):
    """struct i4_thinker_layer"""

    _fields_ = [("in_norm_w", c_void_p), ("q_norm_w", c_void_p), ("k_norm_w", c_void_p),
                ("k_cache", c_void_p), ("v_cache", c_void_p), ("eps", ctypes.c_float),
                ("qkv", QWeightC), ("o", QWeightC), ("moe", MoeWeightsC)]


class KVCacheC(ctypes.Structure):
    """struct i4_kvcache"""

    _fields_ = [("k", c_void_p), ("v", c_void_p), ("batch_stride", c_int64),
                ("head_stride", c_int64), ("row_stride", c_int64), ("batch", c_int32),
                ("n_kv_heads", c_int32), ("max_len", c_int32), ("head_dim", c_int32),
                ("dtype", c_int32)]


class KV8CacheC(ctypes.Structure):
    """struct i4_kv8cache"""

    _fields_ = [("k", c_void_p), ("v", c_void_p), ("k_scale", c_void_p), ("v_scale", c_void_p),
                ("k_tail", c_void_p), ("v_tail", c_void_p), ("batch", c_int32),
                ("n_kv_heads", c_int32), ("blocks", c_int32), ("head_dim", c_int32),
                ("dtype", c_int32), ("format", c_int32)]


# The structs of the paged entries come as their bytes (struct.pack: 0.2 us; a Structure's
# instance and its conversion: 0.8), of a handle's as its address.

class RotaryC(ctypes.Structure):
    """struct i4_rotary"""

    _fields_ = [("inv_freq", c_void_p), ("axes", c_void_p), ("factor", ctypes.c_float),
                ("pairs", c_int32), ("layout", c_int32)]


class TurnC(ctypes.Structure):
    """struct i4_turn"""

    _fields_ = [("pos", c_void_p), ("axis_stride", c_int64), ("batch_stride", c_int64),
                ("axes", c_int32)]


class HeadsC(ctypes.Structure):
    """struct i4_heads"""

    _fields_ = [("x", c_void_p), ("y", c_void_p), ("xb", c_int64), ("xt", c_int64),
                ("xh", c_int64), ("yb", c_int64), ("yt", c_int64), ("yh", c_int64),
                ("heads", c_int32)]


class PagedCacheC(ctypes.Structure):
    """struct i4_pagedcache"""

    _fields_ = [("k", c_void_p), ("v", c_void_p), ("table", c_void_p), ("page_stride", c_int64),
                ("head_stride", c_int64), ("table_stride", c_int64), ("batch", c_int32),
                ("n_kv_heads", c_int32), ("pages", c_int32), ("page", c_int32),
                ("table_len", c_int32), ("head_dim", c_int32), ("dtype", c_int32)]


# name -> (restype, argtypes); every function declared in include/i4moe.h
SIGNATURES = {
    "i4_abi_version": (c_int, []),
    "i4_strerror": (c_char_p, [c_int]),
    "i4_dq_gemv": (c_int, [c_void_p, c_int, c_int64, POINTER(QWeightC), c_void_p, c_int,
                           c_void_p, c_int, c_void_p, c_size_t, c_void_p]),
    "i4_dq_gemv_workspace_bytes": (c_size_t, [POINTER(QWeightC), c_int]),
    "i4_dq_gemv_bounded": (c_int, [c_void_p, c_int, c_int64, POINTER(QWeightC), c_void_p, c_int,
                                   c_void_p, c_int, c_void_p, c_size_t, c_int, c_int, c_void_p]),
    "i4_linear": (c_int, [c_void_p, c_int, c_int, POINTER(QWeightC), c_void_p, c_void_p, c_int,
                          c_void_p, c_size_t, c_void_p]),
    "i4_linear_workspace_bytes": (c_size_t, [POINTER(QWeightC), c_int]),
    "i4_linear_awq_mfma": (c_int, [POINTER(QWeightC), c_int]),
    "i4_unpack": (c_int, [POINTER(QWeightC), c_void_p, c_void_p]),
    "i4_dequant": (c_int, [POINTER(QWeightC), c_void_p, c_int, c_void_p]),
    "i4_repack_awq_to_ct": (c_int, [POINTER(QWeightC), c_void_p, c_void_p, c_void_p, c_int, c_int,
                                    c_void_p]),
    "i4_repack_tile": (c_int, [POINTER(QWeightC), c_void_p, c_void_p, c_void_p, c_int, c_int,
                               c_void_p]),
    "i4_router_logits": (c_int, [c_void_p, c_int, c_int, c_int, c_void_p, c_int, c_void_p,
                                 ctypes.c_float, c_void_p, c_void_p, c_void_p]),
    "i4_route_topk": (c_int, [c_void_p, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p,
                              c_void_p, c_int, c_void_p]),
    "i4_moe_forward": (c_int, [c_void_p, c_int, c_int, POINTER(MoeWeightsC), c_int, c_int,
                               c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                               c_size_t, c_void_p]),
    "i4_moe_workspace_bytes": (c_size_t, [c_int, c_int, c_int, c_int, c_int]),
    "i4_moe_forward_status": (c_int, [c_void_p, c_int, c_int, POINTER(MoeWeightsC), c_int,
                                      c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                      c_void_p, c_size_t, c_void_p, c_void_p]),
    "i4_moe_forward_bounded": (c_int, [c_void_p, c_int, c_int, POINTER(MoeWeightsC), c_int,
                                       c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_size_t,
                                       c_int, c_int, c_void_p]),
    "i4_moe_status_offset": (c_size_t, [c_int, c_int, c_int, c_int, c_int]),
    "i4_moe_forward_noalloc": (c_int, [c_void_p, c_int, c_int, POINTER(MoeWeightsC), c_int, c_int,
                                       c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                       c_void_p, c_void_p]),
    "i4_moe_down_wait": (c_int, [c_void_p, c_int, POINTER(QWeightC), c_void_p, c_int, c_int, c_int,
                                 c_void_p, c_void_p, c_void_p, c_int, c_void_p]),
    "i4_moe_gate_up": (c_int, [c_void_p, c_int, POINTER(QWeightC), c_void_p, c_int, c_void_p,
                               c_void_p]),
    "i4_moe_route_gate_up": (c_int, [c_void_p, c_int, POINTER(QWeightC), c_void_p, c_int, c_int,
                                     c_int, c_void_p, c_void_p, c_void_p, c_void_p]),
    "i4_moe_down_combine": (c_int, [c_void_p, c_int, POINTER(QWeightC), c_void_p, c_void_p, c_int,
                                    c_void_p, c_void_p, c_void_p]),
    "i4_moe_stack_forward": (c_int, [c_void_p, c_int, c_int, POINTER(MoeWeightsC), c_int, c_int,
                                     c_int, c_void_p, c_void_p, c_size_t, c_void_p]),
    "i4_moe_stack_workspace_bytes": (c_size_t, [c_int, c_int, c_int, c_int, c_int]),
    "i4_moe_route_sum": (c_int, [c_void_p, c_int, c_void_p, POINTER(MoeWeightsC), c_int, c_void_p,
                                 c_int, c_void_p, c_size_t, c_void_p]),
    "i4_moe_experts_x": (c_int, [c_void_p, c_int, POINTER(MoeWeightsC), c_int, c_int, c_void_p,
                                 c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "i4_moe_sum": (c_int, [c_void_p, c_int, c_void_p, POINTER(MoeWeightsC), c_int, c_void_p,
                           c_void_p, c_size_t, c_void_p]),
    "i4_rmsnorm_linear": (c_int, [c_void_p, c_int, c_int, c_void_p, ctypes.c_float,
                                  POINTER(QWeightC), c_void_p, c_void_p, c_int, c_void_p]),
    "i4_rmsnorm": (c_int, [c_void_p, c_int, c_int, c_int, c_void_p, ctypes.c_float, c_void_p,
                           c_void_p]),
    "i4_attn_decode": (c_int, [c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p,
                               ctypes.c_float, c_void_p, c_int, c_void_p, c_void_p, c_int,
                               c_void_p, c_void_p, c_size_t, c_void_p]),
    "i4_attn_decode_at": (c_int, [c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p,
                                  ctypes.c_float, c_void_p, c_void_p, c_void_p, c_void_p, c_int,
                                  c_void_p, c_void_p, c_size_t, c_void_p]),
    "i4_attn_decode_workspace_bytes": (c_size_t, [c_int, c_int, c_int]),
    "i4_attn_decode_o": (c_int, [c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p,
                                 ctypes.c_float, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                 c_int, POINTER(QWeightC), c_void_p, c_void_p, c_void_p,
                                 c_size_t, c_void_p]),
    "i4_attn_decode_o_workspace_bytes": (c_size_t, [c_int, c_int, c_int]),
    "i4_attn_decode_o_status_offset": (c_size_t, [c_int, c_int, c_int]),
    "i4_attn_decode_qkv_o": (c_int, [c_void_p, c_int, c_void_p, ctypes.c_float,
                                     POINTER(QWeightC), c_int, c_int, c_int, c_void_p, c_void_p,
                                     c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_int,
                                     POINTER(QWeightC), c_void_p, c_void_p, c_size_t, c_void_p]),
    "i4_attn_decode_qkv_o_workspace_bytes": (c_size_t, [c_int, c_int, c_int, c_int]),
    "i4_thinker_layer_decode": (c_int, [c_void_p, c_int, c_void_p, ctypes.c_float,
                                        POINTER(QWeightC), c_int, c_int, c_int, c_void_p,
                                        c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                        c_int, POINTER(QWeightC), POINTER(MoeWeightsC), c_int,
                                        c_int, c_void_p, c_void_p, c_size_t, c_void_p]),
    "i4_thinker_layer_workspace_bytes": (c_size_t, [c_int, c_int, c_int, c_int, c_int, c_int,
                                                    c_int, c_int]),
    "i4_thinker_decode_step": (c_int, [c_void_p, c_int, POINTER(ThinkerLayerC), c_int, c_int,
                                       c_int, c_int, c_void_p, c_void_p, c_int, c_int, c_int,
                                       c_int, c_void_p, c_void_p, c_size_t, c_void_p]),
    "i4_thinker_decode_step_workspace_bytes": (c_size_t, [c_int, c_int, c_int, c_int, c_int,
                                                          c_int, c_int, c_int]),
    "i4_rope_append": (c_int, [c_void_p, c_int, c_int, c_int64, c_int64, c_int, c_void_p,
                               c_void_p, ctypes.c_float, c_void_p, c_void_p, c_int, c_int,
                               c_void_p, c_void_p, POINTER(KVCacheC), c_void_p]),
    "i4_attn_window": (c_int, [c_void_p, c_int, c_int, c_int64, c_int64, c_int64, c_int,
                               POINTER(KVCacheC), c_void_p, c_int, c_void_p, c_int, c_int,
                               ctypes.c_float, c_void_p, c_void_p, c_size_t, c_void_p, c_void_p]),
    "i4_attn_window_workspace_bytes": (c_size_t, [c_int, c_int, c_int, c_int, c_int, c_int,
                                                  c_int]),
    "i4_kv8_append": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int64, c_int64, c_int64,
                              POINTER(KV8CacheC), c_void_p, c_int, c_void_p, c_void_p]),
    "i4_kv8_values": (c_int, [POINTER(KV8CacheC), c_void_p, c_void_p, c_void_p]),
    "i4_attn_kv8": (c_int, [c_void_p, c_int, c_int, c_int64, c_int64, c_int64, c_int,
                            POINTER(KV8CacheC), c_void_p, c_int, c_void_p, c_int, c_int,
                            ctypes.c_float, c_void_p, c_void_p, c_size_t, c_void_p, c_void_p]),
    "i4_rope": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_int,
                        c_void_p, c_void_p, c_int, c_void_p]),
    "i4_paged_append": (c_int, [c_void_p, c_int, c_int, c_int64, c_int64, c_int, c_void_p,
                                c_void_p, ctypes.c_float, c_void_p, c_void_p, c_int, c_void_p,
                                c_void_p, c_int, c_void_p, c_void_p, c_void_p]),
    "i4_attn_paged": (c_int, [c_void_p, c_int, c_int, c_int64, c_int64, c_int64, c_int,
                              c_void_p, c_void_p, c_int, c_void_p, c_int, c_int,
                              c_int, ctypes.c_float, c_void_p, c_void_p, c_size_t, c_void_p, c_void_p]),
    "i4_attn_paged_call_bytes": (c_size_t, [c_int, c_int, c_int, c_int, c_int, c_int, c_int,
                                            c_int]),
    "i4_attn_paged_workspace_bytes": (c_size_t, [c_int, c_int, c_int, c_int, c_int, c_int,
                                                 c_int]),
    "i4_dmoe_forward": (c_int, [c_void_p, c_int, c_int, POINTER(DmoeWeightsC), c_int, c_int,
                                c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                c_size_t, c_void_p]),
    "i4_dmoe_workspace_bytes": (c_size_t, [c_int, c_int, c_int, c_int, c_int]),
    "i4_dmoe_workspace_bytes_h": (c_size_t, [c_int, c_int, c_int, c_int, c_int, c_int]),
    "i4_dmoe_status_offset": (c_size_t, [c_int, c_int, c_int, c_int, c_int]),
    "i4_dmoe_down_wait": (c_int, [c_void_p, c_int, POINTER(DmoeWeightsC), c_int, c_int,
                                  c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_int,
                                  c_void_p]),
}

_lib = None


def lib() -> ctypes.CDLL:
    """Load libi4moe.so once and declare every signature."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is not built: run __graft_entry__.build() (hipcc, gfx950) first")
        lb = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lb, name)
            fn.restype = res
            fn.argtypes = args
        ver = lb.i4_abi_version()
        if ver != ABI_VERSION:
            raise RuntimeError(f"libi4moe ABI {ver}, package expects {ABI_VERSION}")
        _lib = lb
    return _lib


def check(rc: int) -> None:
    if rc != 0:
        raise RuntimeError(lib().i4_strerror(rc).decode())


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DT[dt]
    except KeyError:
        raise RuntimeError(f"unsupported dtype {dt}") from None


def half_code(dt: torch.dtype) -> int:
    if dt not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"activations must be float16 or bfloat16, got {dt}")
    return _DT[dt]


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# The raw handle of the current stream, without the Stream object that torch.cuda makes
# around it (0.2 against 2.1 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream(device: torch.device) -> int:
    if _raw_stream is None or device.index is None:
        return torch.cuda.current_stream(device).cuda_stream
    return _raw_stream(device.index)


class Handle:
    """An object that holds addresses for the kernels: its attributes are set once, so that no
    tensor can be taken from behind its address.  (Properties over other slots would do too, and
    cost each call their reads.)"""

    __slots__ = ()

    def __setattr__(self, name: str, value) -> None:
        if hasattr(self, name):
            raise AttributeError(f"{type(self).__name__}.{name} cannot be replaced: make another "
                                 f"{type(self).__name__}")
        object.__setattr__(self, name, value)

    def __delattr__(self, name: str) -> None:
        raise AttributeError(f"{type(self).__name__}.{name} cannot be taken away")


def require_device(*ts: torch.Tensor | None) -> torch.device:
    dev, index = None, -2
    for t in ts:
        if t is None:
            continue
        i = t.get_device()  # -1: not on a device
        if i != index:
            if t.device.type != "cuda":
                raise RuntimeError("libi4moe operates on HIP device tensors only "
                                   f"(got a tensor on {t.device})")
            if dev is not None:
                raise RuntimeError("all tensors must be on the same device")
            dev, index = t.device, i
    if dev is None:
        raise RuntimeError("no device tensor given")
    return dev
