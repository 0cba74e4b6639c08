"""ane_amd -- MI355X (gfx950) implementation of ane's quantized compute path.

Python mirror of the reference's C++ entry points for this path:

* ``Op`` -- the opcode numbering of the reference's ``enum class ane::Op``
  (include/ane/ane.hpp:47-177) plus ``dense_fused_i8`` (README.md:84-97).
* ``encode`` / ``dispatch`` -- ``ane::dispatch`` (include/ane/ane.hpp:206-220):
  ``[op:u8]`` followed by each argument's little-endian bytes, handed to the
  C entry point ``stream_exec`` of ``libane_amd.so``.
* thin wrappers over the kernel-level C ABI (``include/ane_hip.h``) that take
  torch tensors for device memory and the current torch stream.

The native library is required: importing works without it (so the CPU test
suite can inspect the package), but every call raises if it is missing.
"""
from __future__ import annotations

import ctypes
import enum
import os
import struct
from pathlib import Path
from typing import Any, Iterable

PKG_DIR = Path(__file__).resolve().parent
LIB_PATH = PKG_DIR / "libane_amd.so"


class Op(enum.IntEnum):
    """Opcode numbers served by this build (reference include/ane/ane.hpp:47-177)."""

    dense_i8 = 0x18
    quantize_fp32_i8 = 0x19
    dequantize_i8_fp32 = 0x1A
    pack_b_i8 = 0x1B
    quantize_fp32_i8_channelwise = 0x1C
    dense_u8s8 = 0x1E
    rms_norm_fp32 = 0x51
    silu_fp32 = 0x54
    rope_fp32 = 0x55
    softmax_fp32 = 0x56
    q8_0_gemv = 0x57
    q4_0_gemv = 0x58
    cblas_igemm = 0x61
    cblas_ugemm = 0x62
    cblas_usgemm = 0x63
    q4_k_gemv = 0x75
    q2_k_gemv = 0x76
    q3_k_gemv = 0x77
    q5_k_gemv = 0x78
    q6_k_gemv = 0x79
    get_rows_q8_0 = 0x7C
    get_rows_q4_0 = 0x7D
    dense_fused_i8 = 0x80


# R-mode GEMV formats besides Q8_0: name -> (bytes, values) per (super-)block
QFORMATS = {"q4_0": (18, 32), "q4_k": (144, 256), "q2_k": (84, 256), "q3_k": (110, 256),
            "q5_k": (176, 256), "q6_k": (210, 256)}


class AneError(RuntimeError):
    """A call into libane_amd.so returned a non-zero ane_status."""

    def __init__(self, status: int, message: str):
        super().__init__(f"ane status {status}: {message}")
        self.status = status


STATUS = {
    0: "ANE_OK",
    1: "ANE_ERR_INVALID_ARG",
    2: "ANE_ERR_BAD_POINTER",
    3: "ANE_ERR_BUFFER_TOO_SMALL",
    4: "ANE_ERR_UNKNOWN_OPCODE",
    5: "ANE_ERR_TRUNCATED",
    6: "ANE_ERR_HIP",
    7: "ANE_ERR_NO_DEVICE",
    8: "ANE_ERR_WORKSPACE",
    9: "ANE_ERR_GRID_WAIT",
}

# Symbols include/ane_hip.h, include/ggml-ane-hip.h and include/ane_decode.h
# declare; the library must export every one.
EXPORTS = (
    "stream_exec",
    "ane_last_error",
    "ane_last_error_message",
    "ane_set_stream",
    "ane_set_host_staging",
    "ane_stream_exec_async",
    "ane_hip_quantize_workspace_size",
    "ane_hip_quantize_fp32_i8",
    "ane_hip_dequantize_i8_fp32",
    "ane_hip_quantize_channelwise",
    "ane_hip_packed_b_size",
    "ane_hip_pack_b_i8",
    "ane_hip_dense_i8",
    "ane_hip_dense_fused_i8_workspace_size",
    "ane_hip_dense_fused_i8",
    "ane_hip_dense_fused_i8_quantize",
    "ane_hip_dense_fused_i8_gemm",
    "ane_hip_dense_fused_i8_status",
    "ane_hip_grid_wait_status",
    "ane_hip_set_grid_wait_limit",
    "ane_hip_gemm_s8_i32",
    "ane_hip_q8_0_gemv",
    "ane_hip_cblas_igemm_workspace_size",
    "ane_hip_cblas_igemm",
    "ane_hip_q4_0_gemv",
    "ane_hip_q4_k_gemv",
    "ane_hip_q2_k_gemv",
    "ane_hip_q3_k_gemv",
    "ane_hip_q5_k_gemv",
    "ane_hip_q6_k_gemv",
    "ane_hip_get_rows_q8_0",
    "ane_hip_get_rows_q4_0",
    "ane_hip_q8_0_mul_mat_workspace_size",
    "ane_hip_q8_0_mul_mat_workspace_size_n",
    "ane_hip_q8_0_mul_mat",
    "ane_hip_q8_0_mul_mat_noalloc_max_bytes",
    "ane_hip_q8_0_mul_mat_noalloc",
    "ane_hip_device_check",
    "ane_hip_version",
    # include/ggml-ane-hip.h
    "ane_ggml_backend_name",
    "ane_ggml_device_name",
    "ane_ggml_backend_init",
    "ane_ggml_backend_free",
    "ane_ggml_backend_set_q8_mode",
    "ane_ggml_supports_op",
    "ane_ggml_compute_forward",
    "ane_ggml_graph_compute",
    # include/ane_decode.h
    "ane_decode_workspace_size",
    "ane_decode_token",
    "ane_hip_q8_0_matvec_fused",
    "ane_hip_rope_kv_append",
    "ane_hip_attention_workspace_size",
    "ane_hip_attention_decode",
    "ane_hip_silu_mul",
    "ane_hip_q8_0_matvec_silu",
    "ane_hip_attention_decode_rope",
    "ane_hip_q8_0_matvec_q8",
    "ane_hip_q8_0_gate_up_silu_quant",
    "ane_hip_silu_mul_quant",
    "ane_hip_rms_norm",
    "ane_hip_add_fp32",
    "ane_hip_rms_norm_fp32",
    "ane_hip_silu_fp32",
    "ane_hip_rope_fp32",
    "ane_hip_softmax_fp32",
    "ane_decode_ggml_workspace_size",
    "ane_decode_token_ggml",
    "ane_ggml_backend_get_stream",
    "ane_ggml_backend_set_stream",
    "ane_hip_paged_rope_append",
    "ane_hip_attention_prompt_workspace_size",
    "ane_hip_attention_prompt",
    "ane_hip_attention_shared_workspace_size",
    "ane_hip_attention_shared",
    "ane_hip_pages_workspace_size",
    "ane_hip_pages_reserve",
    "ane_hip_pages_fork",
    "ane_hip_pages_free",
    "ane_hip_pages_copy",
    "ane_hip_pages_compact",
    "ane_hip_paged_norm_rope_append",
    "ane_hip_attention_rule_workspace_size",
    "ane_hip_attention_rule",
    "ane_hip_quantize_tokens",
    "ane_hip_dense_i8_scaled",
    "ane_hip_linear_i8_workspace_size",
    "ane_hip_linear_i8",
)

_lib: ctypes.CDLL | None = None

_c = ctypes
_P = _c.c_void_p
_SIGS: dict[str, tuple[Any, list[Any]]] = {
    "stream_exec": (None, [_P, _c.c_size_t]),
    "ane_last_error": (_c.c_int, []),
    "ane_last_error_message": (_c.c_char_p, []),
    "ane_set_stream": (None, [_P]),
    "ane_set_host_staging": (None, [_c.c_int]),
    "ane_stream_exec_async": (_c.c_int, [_P, _c.c_size_t, _P]),
    "ane_hip_quantize_workspace_size": (_c.c_size_t, [_c.c_uint64]),
    "ane_hip_quantize_fp32_i8": (_c.c_int, [_c.c_uint64, _c.c_int, _P, _P, _P, _P, _c.c_size_t, _P]),
    "ane_hip_dequantize_i8_fp32": (_c.c_int, [_c.c_uint64, _c.c_float, _P, _P, _P]),
    "ane_hip_quantize_channelwise": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _P, _P, _P]),
    "ane_hip_packed_b_size": (_c.c_size_t, [_c.c_uint32, _c.c_uint32]),
    "ane_hip_pack_b_i8": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _P, _P]),
    "ane_hip_dense_i8": (
        _c.c_int,
        [_c.c_uint32, _c.c_uint32, _c.c_uint32, _c.c_float, _c.c_float, _c.c_uint8, _P, _P, _P, _P,
         _c.c_int, _P],
    ),
    "ane_hip_dense_fused_i8_workspace_size": (_c.c_size_t, [_c.c_int32, _c.c_int32, _c.c_int32]),
    "ane_hip_dense_fused_i8": (
        _c.c_int,
        [_c.c_int32, _c.c_int32, _c.c_int32, _c.c_float, _c.c_int, _P, _P, _P, _P, _P, _c.c_size_t, _P],
    ),
    "ane_hip_dense_fused_i8_quantize": (
        _c.c_int, [_c.c_int32, _c.c_int32, _c.c_int32, _P, _P, _P, _P, _c.c_size_t, _P]),
    "ane_hip_dense_fused_i8_gemm": (
        _c.c_int, [_c.c_int32, _c.c_int32, _c.c_int32, _c.c_float, _c.c_int, _P, _P, _c.c_size_t, _P]),
    "ane_hip_dense_fused_i8_status": (_c.c_int, [_P, _P]),
    "ane_hip_grid_wait_status": (_c.c_int, [_P]),
    "ane_hip_set_grid_wait_limit": (None, [_c.c_uint64]),
    "ane_hip_gemm_s8_i32": (
        _c.c_int,
        [_c.c_uint32, _c.c_uint32, _c.c_uint32, _P, _c.c_uint32, _P, _c.c_uint32, _P, _P],
    ),
    "ane_hip_q8_0_gemv": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _P, _P, _P]),
    "ane_hip_cblas_igemm_workspace_size": (_c.c_size_t, [_c.c_uint32, _c.c_uint32, _c.c_uint32]),
    "ane_hip_cblas_igemm": (
        _c.c_int,
        [_c.c_int, _c.c_int, _c.c_uint8, _c.c_uint32, _c.c_uint32, _c.c_uint32, _c.c_uint32, _c.c_uint32,
         _c.c_uint32, _c.c_float, _c.c_float, _P, _P, _P, _P, _c.c_size_t, _P],
    ),
    **{f"ane_hip_{f}_gemv": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _P, _P, _P]) for f in QFORMATS},
    "ane_hip_get_rows_q8_0": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _c.c_uint64, _P, _P, _P]),
    "ane_hip_get_rows_q4_0": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _c.c_uint64, _P, _P, _P]),
    "ane_hip_q8_0_mul_mat_workspace_size": (_c.c_size_t, [_c.c_uint32, _c.c_uint32]),
    "ane_hip_q8_0_mul_mat_workspace_size_n": (_c.c_size_t, [_c.c_uint32, _c.c_uint32, _c.c_uint32]),
    "ane_hip_q8_0_mul_mat": (
        _c.c_int,
        [_c.c_uint32, _c.c_uint32, _c.c_uint32, _P, _P, _P, _P, _c.c_size_t, _P],
    ),
    "ane_hip_q8_0_mul_mat_noalloc_max_bytes": (_c.c_size_t, []),
    "ane_hip_q8_0_mul_mat_noalloc": (_c.c_int, [_c.c_uint32, _c.c_uint32, _c.c_uint32, _P, _P, _P, _P]),
    "ane_hip_device_check": (_c.c_int, []),
    "ane_hip_version": (_c.c_char_p, []),
    "ane_ggml_backend_name": (_c.c_char_p, []),
    "ane_ggml_device_name": (_c.c_char_p, []),
    "ane_ggml_backend_init": (_P, [_P]),
    "ane_ggml_backend_free": (None, [_P]),
    "ane_ggml_backend_set_q8_mode": (None, [_P, _c.c_int]),
    "ane_ggml_supports_op": (_c.c_int, [_P]),
    "ane_ggml_compute_forward": (_c.c_int, [_P, _P]),
    "ane_ggml_graph_compute": (_c.c_int, [_P, _P, _c.c_int]),
    "ane_decode_workspace_size": (_c.c_size_t, [_P]),
    "ane_decode_token": (_c.c_int, [_P, _P, _P, _c.c_uint32, _P, _P, _c.c_size_t, _P]),
    "ane_hip_q8_0_matvec_fused": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _P, _c.c_float, _P, _P, _P, _P]),
    "ane_hip_rope_kv_append": (_c.c_int, [_P, _P, _P, _c.c_uint32, _P, _P, _P]),
    "ane_hip_attention_workspace_size": (_c.c_size_t, [_P]),
    "ane_hip_attention_decode": (_c.c_int, [_P, _P, _P, _P, _c.c_uint32, _P, _P, _c.c_size_t, _P]),
    "ane_hip_silu_mul": (_c.c_int, [_c.c_uint32, _P, _P, _P]),
    "ane_hip_q8_0_matvec_silu": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _P, _P, _P, _P]),
    "ane_hip_attention_decode_rope": (_c.c_int, [_P, _P, _P, _c.c_uint32, _P, _P, _P, _P, _P, _c.c_size_t, _P]),
    "ane_hip_q8_0_matvec_q8": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _P, _P, _P, _P]),
    "ane_hip_q8_0_gate_up_silu_quant": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _P, _c.c_float, _P, _P, _P]),
    "ane_hip_silu_mul_quant": (_c.c_int, [_c.c_uint32, _P, _P, _P]),
    "ane_hip_rms_norm": (_c.c_int, [_c.c_uint32, _P, _P, _c.c_float, _P, _P]),
    "ane_hip_add_fp32": (_c.c_int, [_c.c_uint32, _P, _P, _P, _P]),
    "ane_hip_rms_norm_fp32": (_c.c_int, [_c.c_uint32, _c.c_uint32, _c.c_float, _P, _P, _P, _P]),
    "ane_hip_silu_fp32": (_c.c_int, [_c.c_uint64, _P, _P, _P]),
    "ane_hip_rope_fp32": (_c.c_int, [_c.c_uint32, _c.c_uint32, _c.c_uint32, _c.c_float, _P, _P, _P]),
    "ane_hip_softmax_fp32": (_c.c_int, [_c.c_uint32, _c.c_uint32, _P, _P, _P]),
    "ane_decode_ggml_workspace_size": (_c.c_size_t, [_P]),
    "ane_decode_token_ggml": (_c.c_int, [_P, _P, _P, _c.c_float, _c.c_uint32, _P, _P, _c.c_size_t, _P, _c.c_int]),
    "ane_ggml_backend_get_stream": (_P, [_P]),
    "ane_ggml_backend_set_stream": (None, [_P, _P]),
    "ane_hip_paged_rope_append": (
        _c.c_int, [_P, _c.c_uint32, _P, _c.c_uint32, _P, _c.c_uint32, _c.c_int, _P, _c.c_uint64, _P, _P, _c.c_uint64,
                   _P, _c.c_uint32, _c.c_int, _P, _c.c_uint64, _P]),
    "ane_hip_attention_prompt_workspace_size": (_c.c_size_t, [_P, _c.c_uint32, _c.c_uint32, _c.c_uint32]),
    "ane_hip_attention_prompt": (
        _c.c_int, [_P, _c.c_uint32, _P, _c.c_uint32, _P, _c.c_uint32, _c.c_uint32, _c.c_int, _P, _c.c_uint64,
                   _c.c_float, _P, _c.c_uint64, _P, _c.c_size_t, _P]),
    "ane_hip_attention_shared_workspace_size": (
        _c.c_size_t, [_P, _c.c_uint32, _c.c_uint32, _c.c_uint32, _c.c_uint32]),
    "ane_hip_attention_shared": (
        _c.c_int, [_P, _c.c_uint32, _P, _c.c_uint32, _c.c_uint32, _P, _P, _c.c_uint32, _c.c_uint32, _c.c_int, _P,
                   _c.c_uint64, _c.c_float, _P, _c.c_uint64, _P, _c.c_size_t, _P]),
    "ane_hip_pages_workspace_size": (_c.c_size_t, [_P]),
    "ane_hip_pages_reserve": (_c.c_int, [_P, _c.c_uint32, _P, _P, _P, _P, _c.c_size_t, _P]),
    "ane_hip_pages_fork": (_c.c_int, [_P, _c.c_uint32, _P, _P, _P, _P, _c.c_size_t, _P]),
    "ane_hip_pages_free": (_c.c_int, [_P, _c.c_uint32, _P, _P]),
    "ane_hip_pages_copy": (_c.c_int, [_P, _c.c_uint32, _P, _P, _P]),
    "ane_hip_pages_compact": (_c.c_int, [_P, _P, _P, _P, _P, _c.c_size_t, _P]),
    "ane_hip_paged_norm_rope_append": (
        _c.c_int, [_P, _c.c_uint32, _P, _c.c_uint32, _P, _c.c_uint32, _c.c_int, _P, _c.c_uint64, _P, _P, _c.c_uint64,
                   _P, _P, _P, _c.c_float, _c.c_int, _P, _c.c_uint64, _P]),
    "ane_hip_attention_rule_workspace_size": (_c.c_size_t, [_P, _c.c_uint32, _c.c_uint32, _c.c_uint32, _P]),
    "ane_hip_attention_rule": (
        _c.c_int, [_P, _c.c_uint32, _P, _c.c_uint32, _P, _c.c_uint32, _c.c_uint32, _P, _c.c_int, _P, _c.c_uint64,
                   _c.c_float, _P, _c.c_uint64, _P, _c.c_size_t, _P]),
    "ane_hip_quantize_tokens": (
        _c.c_int, [_c.c_uint32, _c.c_uint32, _c.c_int, _P, _c.c_uint64, _P, _c.c_float, _P, _c.c_uint64, _P, _P]),
    "ane_hip_dense_i8_scaled": (
        _c.c_int, [_c.c_uint32, _c.c_uint32, _c.c_uint32, _P, _c.c_uint64, _P, _P, _c.c_uint64, _P, _P, _P, _c.c_uint64,
                   _c.c_int, _P, _c.c_uint64, _P]),
    "ane_hip_linear_i8_workspace_size": (_c.c_size_t, [_c.c_uint32, _c.c_uint32, _c.c_uint32]),
    "ane_hip_linear_i8": (
        _c.c_int, [_c.c_uint32, _c.c_uint32, _c.c_uint32, _c.c_int, _P, _c.c_uint64, _P, _c.c_float, _P, _c.c_uint64, _P,
                   _P, _P, _c.c_uint64, _c.c_int, _P, _c.c_uint64, _P, _c.c_size_t, _P]),
}


def lib() -> ctypes.CDLL:
    """Load libane_amd.so (built by ``python -m ane_amd.build``); raise if absent."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -m ane_amd.build` "
                "(there is no CPU fallback for this library)"
            )
        handle = ctypes.CDLL(str(LIB_PATH), mode=os.RTLD_NOW | ctypes.RTLD_GLOBAL)
        for name, (res, args) in _SIGS.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


# ---------------------------------------------------------------- encoding
class _Arg:
    __slots__ = ("fmt", "value", "keep")

    def __init__(self, fmt: str, value: Any, keep: Any = None):
        self.fmt = fmt
        self.value = value
        self.keep = keep


class Record(bytes):
    """An encoded record that also holds the tensors its pointers refer to,
    so a temporary operand cannot be freed (and its memory reused) between
    encoding and execution."""

    keep: tuple = ()


def u8(v: int) -> _Arg:
    return _Arg("<B", int(v))


def boolean(v: bool) -> _Arg:
    return _Arg("<B", 1 if v else 0)


def u32(v: int) -> _Arg:
    return _Arg("<I", int(v))


def i32(v: int) -> _Arg:
    return _Arg("<i", int(v))


def f32(v: float) -> _Arg:
    return _Arg("<f", float(v))


def ptr(v: Any) -> _Arg:
    """Any pointer operand: a torch tensor (its data_ptr) or an integer address."""
    if hasattr(v, "data_ptr"):
        return _Arg("<Q", int(v.data_ptr()), keep=v)
    return _Arg("<Q", int(v or 0))


def encode(op: int, *args: _Arg) -> Record:
    """Byte record of ane::dispatch(op, args...) (include/ane/ane.hpp:206-220)."""
    out = bytearray([int(op) & 0xFF])
    keep = []
    for a in args:
        if not isinstance(a, _Arg):
            raise TypeError("dispatch arguments must be typed: u32/i32/f32/u8/boolean/ptr")
        out += struct.pack(a.fmt, a.value)
        if a.keep is not None:
            keep.append(a.keep)
    rec = Record(bytes(out))
    rec.keep = tuple(keep)
    return rec


def _ceil(x: int, m: int) -> int:
    return (x + m - 1) // m * m


def _need(t: Any, nbytes: int, what: str) -> None:
    """Raise AneError(ANE_ERR_BUFFER_TOO_SMALL) if tensor ``t`` holds fewer
    than ``nbytes`` bytes from its first element to the end of its storage.

    stream_exec checks every operand against its HIP allocation, but torch's
    caching allocator carves tensors out of larger allocations, so a short
    tensor would pass that check and the kernel would touch its neighbours.
    Raw integer addresses are left to stream_exec's check."""
    if nbytes <= 0 or not hasattr(t, "untyped_storage"):
        return
    have = t.untyped_storage().nbytes() - t.storage_offset() * t.element_size()
    if have < nbytes:
        raise AneError(3, f"{what} needs {nbytes} bytes, the tensor holds {have}")


# Typed records with the reference's argument order (Appendix of the opcode
# table: bytecode_interpreter.s parse sites cited in ane_amd/csrc/stream_exec.cpp).
# Tensor operands are checked against the extents the opcode reads and writes.
def rec_dense_i8(M, N, K, sa, sb, relu, A, Bp, bias, C, unsigned_a=False) -> bytes:
    op = Op.dense_u8s8 if unsigned_a else Op.dense_i8
    if N:
        Mp, Kp = max(16, _ceil(M, 16)), _ceil(K, 64)
        _need(A, Mp * Kp, "dense A")
        _need(Bp, _ceil(N, 16) // 16 * (Kp // 4) * 64, "dense B_packed")
        _need(bias, 4 * N, "dense bias")
        _need(C, 4 * Mp * N, "dense C")
    return encode(op, u32(M), u32(N), u32(K), f32(sa), f32(sb), boolean(relu), ptr(A), ptr(Bp),
                  ptr(bias), ptr(C))


def rec_quantize(count, src, dst, scale_out) -> bytes:
    n = max(16, _ceil(count, 16))
    _need(src, 4 * n, "quantize_fp32_i8 src")
    _need(dst, n, "quantize_fp32_i8 dst")
    _need(scale_out, 4, "quantize_fp32_i8 scale_out")
    return encode(Op.quantize_fp32_i8, u32(count), ptr(src), ptr(dst), ptr(scale_out))


def rec_dequantize(count, scale, src, dst) -> bytes:
    n = _ceil(count, 16)
    _need(src, n, "dequantize_i8_fp32 src")
    _need(dst, 4 * n, "dequantize_i8_fp32 dst")
    return encode(Op.dequantize_i8_fp32, u32(count), f32(scale), ptr(src), ptr(dst))


def rec_pack_b(K, N, src, dst) -> bytes:
    _need(src, K * N, "pack_b_i8 src")
    _need(dst, _ceil(N, 16) // 16 * (_ceil(K, 4) // 4) * 64, "pack_b_i8 dst")
    return encode(Op.pack_b_i8, u32(K), u32(N), ptr(src), ptr(dst))


def rec_channelwise(rows, cols, src, dst, scales) -> bytes:
    if rows:
        cpad = max(16, _ceil(cols, 16))
        _need(src, 4 * rows * cpad, "channelwise src")
        _need(dst, rows * cpad, "channelwise dst")
        _need(scales, 4 * rows, "channelwise scales")
    return encode(Op.quantize_fp32_i8_channelwise, u32(rows), u32(cols), ptr(src), ptr(dst), ptr(scales))


def rec_q8_0_gemv(M, K, x, W, y) -> bytes:
    if M:
        nb = K >> 5
        _need(x, 4 * 32 * nb, "q8_0_gemv x")
        _need(W, M * nb * 34, "q8_0_gemv W")
        _need(y, 4 * M, "q8_0_gemv y")
    return encode(Op.q8_0_gemv, u32(M), u32(K), ptr(x), ptr(W), ptr(y))


def rec_q_gemv(fmt, M, K, x, W, y) -> bytes:
    """Record of one of the QFORMATS GEMVs (same layout as q8_0_gemv)."""
    if M:
        bb, vals = QFORMATS[fmt]
        nsb = K // vals
        _need(x, 4 * vals * nsb, f"{fmt}_gemv x")
        _need(W, M * nsb * bb, f"{fmt}_gemv W")
        _need(y, 4 * M, f"{fmt}_gemv y")
    return encode(Op[f"{fmt}_gemv"], u32(M), u32(K), ptr(x), ptr(W), ptr(y))


def rec_get_rows(fmt, n_rows, dim, table, indices, out) -> bytes:
    """get_rows_q8_0 / get_rows_q4_0 record: [n_rows:u32][dim:u32][table][indices][out]."""
    if n_rows and dim >= 32:
        _need(indices, 4 * n_rows, f"get_rows_{fmt} indices")
        _need(out, 4 * n_rows * (dim >> 5) * 32, f"get_rows_{fmt} out")
    return encode(Op[f"get_rows_{fmt}"], u32(n_rows), u32(dim), ptr(table), ptr(indices), ptr(out))


IGEMM_VARIANTS = {"igemm": 0, "ugemm": 1, "usgemm": 2}


def _igemm_extents(flags, M, N, K, lda, ldb, ldc):
    """Bytes of A, B and C the integer GEMM handler's arithmetic touches."""
    Ke = K // 64 * 64
    a = b = 0
    if Ke and M and N:
        if flags & 1:
            g = (M - 1) - (M - 1) % 16
            mx = ((M - 1) % 16) * lda + g
            if M > 16:
                mx = max(mx, 15 * lda + g - 16)
            a = mx + Ke
        else:
            a = (M - 1) * lda + Ke
        b = (N - 1) * ldb + Ke if flags & 2 else (Ke - 1) * ldb + N
    c = 4 * ((M - 1) * ldc + N) if M and N else 0
    return a, b, c


def rec_cblas_igemm(kind, flags, M, N, K, lda, ldb, ldc, alpha, beta, A, B, C) -> bytes:
    """cblas_igemm / cblas_ugemm / cblas_usgemm (kind "igemm", "ugemm",
    "usgemm"): [op][flags:u8][M N K lda ldb ldc:u32][alpha beta:f32][A][B][C]
    (bytecode_interpreter.s:8355-8369)."""
    a, b, c = _igemm_extents(flags, M, N, K, lda, ldb, ldc)
    _need(A, a, f"cblas_{kind} A")
    _need(B, b, f"cblas_{kind} B")
    _need(C, c, f"cblas_{kind} C")
    return encode(Op.cblas_igemm + IGEMM_VARIANTS[kind], u8(flags), u32(M), u32(N), u32(K), u32(lda), u32(ldb),
                  u32(ldc), f32(alpha), f32(beta), ptr(A), ptr(B), ptr(C))


def rec_rms_norm(dim, eps, x, w, out) -> bytes:
    """rms_norm_fp32 (0x51): [dim:u32][eps:f32][in][weight][out] (bytecode_interpreter.s:6509-6514)."""
    for t, nm in ((x, "in"), (w, "weight"), (out, "out")):
        _need(t, 4 * dim, f"rms_norm_fp32 {nm}")
    return encode(Op.rms_norm_fp32, u32(dim), f32(eps), ptr(x), ptr(w), ptr(out))


def rec_silu(count, x, out) -> bytes:
    """silu_fp32 (0x54): [count:u32][in][out] (:6618-6621)."""
    _need(x, 4 * count, "silu_fp32 in")
    _need(out, 4 * count, "silu_fp32 out")
    return encode(Op.silu_fp32, u32(count), ptr(x), ptr(out))


def rec_rope(dim, pos, theta, x, out) -> bytes:
    """rope_fp32 (0x55): [dim:u32][pos:u32][theta:f32][in][out] (:6715-6720)."""
    _need(x, 4 * (dim // 2 * 2), "rope_fp32 in")
    _need(out, 4 * (dim // 2 * 2), "rope_fp32 out")
    return encode(Op.rope_fp32, u32(dim), u32(pos), f32(theta), ptr(x), ptr(out))


def rec_softmax(dim, x, out) -> bytes:
    """softmax_fp32 (0x56): [dim:u32][in][out] (:6914-6917)."""
    _need(x, 4 * dim, "softmax_fp32 in")
    _need(out, 4 * dim, "softmax_fp32 out")
    return encode(Op.softmax_fp32, u32(dim), ptr(x), ptr(out))


def rec_dense_fused_i8(M, N, K, scale, relu, A, B, C) -> bytes:
    if M > 0 and N > 0:
        _need(A, 4 * M * K, "dense_fused_i8 A")
        _need(B, 4 * K * N, "dense_fused_i8 B")
        _need(C, 4 * M * N, "dense_fused_i8 C")
    return encode(Op.dense_fused_i8, i32(M), i32(N), i32(K), f32(scale), boolean(relu), ptr(A), ptr(B),
                  ptr(C))


# ---------------------------------------------------------------- execution
def _stream_handle(stream: Any = None) -> int:
    if stream is None:
        import torch

        stream = torch.cuda.current_stream()
    if hasattr(stream, "cuda_stream"):
        return int(stream.cuda_stream)
    return int(stream or 0)


def stream_exec(data: bytes | Iterable[bytes], stream: Any = None) -> None:
    """Run encoded records through the C entry point ``stream_exec`` on
    ``stream`` (default: torch's current stream) and raise AneError on failure."""
    records = [data] if isinstance(data, (bytes, bytearray)) else list(data)
    data = b"".join(records)  # `records` keeps every operand alive until the call returns
    L = lib()
    L.ane_set_stream(_stream_handle(stream))
    buf = ctypes.create_string_buffer(bytes(data), len(data))
    L.stream_exec(buf, len(data))
    st = L.ane_last_error()
    del records
    if st != 0:
        raise AneError(st, L.ane_last_error_message().decode(errors="replace"))


def dispatch(op: int, *args: _Arg, stream: Any = None) -> None:
    """``ane::dispatch(op, args...)`` with explicitly typed arguments."""
    stream_exec(encode(op, *args), stream=stream)


def check(status: int, what: str = "") -> None:
    if status != 0:
        raise AneError(status, f"{what}: {STATUS.get(status, '?')}")


def _p(t: Any) -> int:
    if t is None:
        return 0
    return int(t.data_ptr()) if hasattr(t, "data_ptr") else int(t)


def _scratch(nbytes: int, device, stream: Any = None, zero: bool = False):
    """A temporary device workspace for a call launched on ``stream``.

    It is allocated on that stream (torch's caching allocator keys blocks by
    the stream they were allocated on), so when the tensor is dropped right
    after the asynchronous call the block is only reused by work ordered
    after the kernels on that same stream."""
    import torch

    if stream is None:
        s = torch.cuda.current_stream(device)
    elif isinstance(stream, torch.cuda.Stream):
        s = stream
    else:
        s = torch.cuda.ExternalStream(_stream_handle(stream), device=device)
    with torch.cuda.stream(s):
        return (torch.zeros if zero else torch.empty)(max(int(nbytes), 1), dtype=torch.uint8, device=device)


# Kernel-level wrappers (device tensors, current torch stream unless given).
def quantize_fp32_i8(src, dst, scale_out, count=None, pad16=True, workspace=None, stream=None):
    n = src.numel() if count is None else count
    L = lib()
    wsb = L.ane_hip_quantize_workspace_size(n)
    ws = workspace if workspace is not None else _scratch(wsb, src.device, stream)
    check(L.ane_hip_quantize_fp32_i8(n, 1 if pad16 else 0, _p(src), _p(dst), _p(scale_out), _p(ws), wsb,
                                     _stream_handle(stream)), "quantize_fp32_i8")


def _capturing(stream: Any = None) -> bool:
    """True when ``stream`` (default: torch's current stream) is capturing a graph."""
    import torch

    if stream is None:
        return torch.cuda.is_current_stream_capturing()
    if not isinstance(stream, torch.cuda.Stream):
        h = _stream_handle(stream)
        if h == 0:
            return False  # the null stream never captures
        stream = torch.cuda.ExternalStream(h)
    s = stream
    with torch.cuda.stream(s):
        return torch.cuda.is_current_stream_capturing()


def dense_fused_i8_status(workspace, stream=None) -> None:
    """Raise AneError(ANE_ERR_GRID_WAIT) if the last quantize call made with
    ``workspace`` ran a grid-wide wait that gave up or was completed by
    another launch's arrivals (its outputs are then not valid).
    Synchronizes the stream; not allowed while it is capturing."""
    check(lib().ane_hip_dense_fused_i8_status(_p(workspace), _stream_handle(stream)), "dense_fused_i8")


def _want_check(check_arg, stream) -> bool:
    return (not _capturing(stream)) if check_arg is None else bool(check_arg)


def dense_fused_i8(M, N, K, scale, relu, A, B, C, scales_out=None, workspace=None, stream=None, check_wait=None):
    """Op::dense_fused_i8 on the kernel ABI.  check_wait: None (default)
    checks the quantizer's wait record after the call (dense_fused_i8_status,
    which synchronizes the stream) unless the stream is capturing; False
    leaves that to the caller; True always checks."""
    L = lib()
    wsb = L.ane_hip_dense_fused_i8_workspace_size(M, N, K)
    ws = workspace if workspace is not None else _scratch(wsb, A.device, stream)
    check(L.ane_hip_dense_fused_i8(M, N, K, scale, 1 if relu else 0, _p(A), _p(B), _p(C), _p(scales_out),
                                   _p(ws), wsb, _stream_handle(stream)), "dense_fused_i8")
    if M > 0 and N > 0 and _want_check(check_wait, stream):
        dense_fused_i8_status(ws, stream)


def dense_fused_i8_quantize(M, N, K, A, B, workspace, scales_out=None, stream=None, check_wait=None):
    """The quantize phase of dense_fused_i8; check_wait as for dense_fused_i8."""
    check(lib().ane_hip_dense_fused_i8_quantize(M, N, K, _p(A), _p(B), _p(scales_out), _p(workspace),
                                                workspace.numel(), _stream_handle(stream)),
          "dense_fused_i8_quantize")
    if M > 0 and N > 0 and _want_check(check_wait, stream):
        dense_fused_i8_status(workspace, stream)


def dense_fused_i8_gemm(M, N, K, scale, relu, C, workspace, stream=None):
    check(lib().ane_hip_dense_fused_i8_gemm(M, N, K, scale, 1 if relu else 0, _p(C), _p(workspace),
                                            workspace.numel(), _stream_handle(stream)),
          "dense_fused_i8_gemm")


def dense_fused_i8_workspace_size(M, N, K) -> int:
    return int(lib().ane_hip_dense_fused_i8_workspace_size(M, N, K))


def gemm_s8_i32(A, Bt, acc, M, N, K, lda=None, ldb=None, stream=None):
    check(lib().ane_hip_gemm_s8_i32(M, N, K, _p(A), lda or K, _p(Bt), ldb or K, _p(acc),
                                    _stream_handle(stream)), "gemm_s8_i32")


def cblas_igemm(kind, flags, M, N, K, lda, ldb, ldc, alpha, beta, A, B, C, blas=False, workspace=None,
                stream=None):
    """The integer GEMMs on the kernel-level ABI; blas=False reproduces the
    handler (what stream_exec runs), blas=True the BLAS form."""
    L = lib()
    wsb = L.ane_hip_cblas_igemm_workspace_size(M, N, K)
    ws = workspace if workspace is not None else _scratch(wsb, C.device, stream)
    check(L.ane_hip_cblas_igemm(IGEMM_VARIANTS[kind], 1 if blas else 0, flags, M, N, K, lda, ldb, ldc, alpha, beta,
                                _p(A), _p(B), _p(C), _p(ws), wsb, _stream_handle(stream)), f"cblas_{kind}")


def q8_0_gemv(M, K, x, W, y, stream=None):
    check(lib().ane_hip_q8_0_gemv(M, K, _p(x), _p(W), _p(y), _stream_handle(stream)), "q8_0_gemv")


def q_gemv(fmt, M, K, x, W, y, stream=None):
    """y = W x for W in one of QFORMATS (the reference's R-mode arithmetic)."""
    if fmt not in QFORMATS:
        raise ValueError(f"unknown format {fmt!r}")
    check(getattr(lib(), f"ane_hip_{fmt}_gemv")(M, K, _p(x), _p(W), _p(y), _stream_handle(stream)),
          f"{fmt}_gemv")


def get_rows(fmt, n_rows, dim, table, table_rows, indices, out, stream=None):
    """out[r] = dequantized table row indices[r] (fmt "q8_0" or "q4_0")."""
    if fmt not in ("q8_0", "q4_0"):
        raise ValueError(f"unknown format {fmt!r}")
    check(getattr(lib(), f"ane_hip_get_rows_{fmt}")(n_rows, dim, _p(table), table_rows, _p(indices), _p(out),
                                                     _stream_handle(stream)), f"get_rows_{fmt}")


def q8_0_mul_mat_workspace_size(K, T, N=None) -> int:
    """Workspace bytes for q8_0_mul_mat: with N, enough for every route of
    an N-row matrix (ane_hip_q8_0_mul_mat_workspace_size_n); without, the
    minimum (some routes are then not taken; results are the same)."""
    if N is None:
        return int(lib().ane_hip_q8_0_mul_mat_workspace_size(K, T))
    return int(lib().ane_hip_q8_0_mul_mat_workspace_size_n(N, K, T))


def q8_0_mul_mat(N, K, T, x, W, y, workspace=None, stream=None):
    L = lib()
    if workspace is None:
        wsb = L.ane_hip_q8_0_mul_mat_workspace_size_n(N, K, T)
        ws = _scratch(wsb, W.device, stream)
    else:
        ws = workspace
        wsb = (workspace.numel() * workspace.element_size() if hasattr(workspace, "numel")
               else L.ane_hip_q8_0_mul_mat_workspace_size(K, T))
    check(L.ane_hip_q8_0_mul_mat(N, K, T, _p(x), _p(W), _p(y), _p(ws), wsb, _stream_handle(stream)),
          "q8_0_mul_mat")


def q8_0_mul_mat_noalloc(N, K, T, x, W, y, stream=None):
    """q8_0_mul_mat with its workspace in the library's static device array
    (no allocation; calls overlapping on one device race)."""
    check(lib().ane_hip_q8_0_mul_mat_noalloc(N, K, T, _p(x), _p(W), _p(y), _stream_handle(stream)),
          "q8_0_mul_mat_noalloc")


def pack_b_i8(K, N, src, dst, stream=None):
    check(lib().ane_hip_pack_b_i8(K, N, _p(src), _p(dst), _stream_handle(stream)), "pack_b_i8")


def packed_b_size(K, N) -> int:
    return int(lib().ane_hip_packed_b_size(K, N))


def dense_i8(M, N, K, sa, sb, relu, A, Bp, bias, C, unsigned_a=False, stream=None):
    check(lib().ane_hip_dense_i8(M, N, K, sa, sb, 1 if relu else 0, _p(A), _p(Bp), _p(bias), _p(C),
                                 1 if unsigned_a else 0, _stream_handle(stream)), "dense_i8")


def require_gpu() -> None:
    """Raise unless libane_amd.so is loadable and a gfx950 device is present."""
    st = lib().ane_hip_device_check()
    if st != 0:
        raise AneError(st, "no usable gfx950 device")


# ---------------------------------------------------------------- ggml hook
class GgmlType:
    """ggml_type values the hook distinguishes (include/ggml-ane-hip.h)."""
    F32 = 0
    F16 = 1
    Q4_0 = 2
    Q8_0 = 8
    I32 = 26


class GgmlOp:
    """enum ane_ggml_op (include/ggml-ane-hip.h)."""
    NONE = 0
    MUL_MAT = 1
    OTHER = 2
    ADD = 3
    MUL = 4
    SCALE = 5
    RMS_NORM = 6
    SOFT_MAX = 7
    SILU = 8
    ROPE = 9
    CPY = 10


class GgmlTensor(ctypes.Structure):
    """Mirror of struct ane_ggml_tensor (ggml's ne/nb/type/op/src/data)."""


GgmlTensor._fields_ = [
    ("type", ctypes.c_int32),
    ("ne", ctypes.c_int64 * 4),
    ("nb", ctypes.c_size_t * 4),
    ("op", ctypes.c_int32),
    ("src", ctypes.POINTER(GgmlTensor) * 10),
    ("data", ctypes.c_void_p),
    ("op_params", ctypes.c_int32 * 16),
]

_TYPE_SIZE = {GgmlType.F32: (1, 4), GgmlType.F16: (1, 2), GgmlType.Q4_0: (32, 18), GgmlType.Q8_0: (32, 34),
              GgmlType.I32: (1, 4)}


def ggml_op_params(*values) -> list:
    """op_params words from ints and floats (floats stored as their fp32
    bits, as ggml's memcpy into op_params does)."""
    import struct

    out = []
    for v in values:
        out.append(struct.unpack("<i", struct.pack("<f", v))[0] if isinstance(v, float) else int(v))
    return out


def ggml_tensor(type_, ne, data=None, nb=None, op=GgmlOp.NONE, src=(), op_params=()) -> GgmlTensor:
    """A node with ggml's default (contiguous) strides unless nb is given;
    op_params: int32 words (ggml_op_params packs floats)."""
    ne = list(ne) + [1] * (4 - len(ne))
    t = GgmlTensor()
    t.type = type_
    t.op = op
    for i in range(4):
        t.ne[i] = ne[i]
    if nb is None:
        blk, size = _TYPE_SIZE[type_]
        nb = [size, size * (ne[0] // blk)]
        nb.append(nb[1] * ne[1])
        nb.append(nb[2] * ne[2])
    for i in range(4):
        t.nb[i] = nb[i]
    for i, s_ in enumerate(src):
        if s_ is not None:
            t.src[i] = ctypes.pointer(s_)
    for i, w in enumerate(op_params):
        t.op_params[i] = w
    t.data = _p(data) or None
    return t


class GgmlBackend:
    """The backend instance of include/ggml-ane-hip.h (device workspace, stream)."""

    def __init__(self, stream=None, q8_mode: int = 0):
        self.L = lib()
        self.h = self.L.ane_ggml_backend_init(_stream_handle(stream))
        if not self.h:
            raise AneError(6, "ane_ggml_backend_init failed")
        self.L.ane_ggml_backend_set_q8_mode(self.h, q8_mode)

    @property
    def stream(self) -> int:
        return int(self.L.ane_ggml_backend_get_stream(self.h) or 0)

    def set_stream(self, stream) -> None:
        self.L.ane_ggml_backend_set_stream(self.h, _stream_handle(stream))

    def supports(self, node: GgmlTensor) -> bool:
        return bool(self.L.ane_ggml_supports_op(ctypes.byref(node)))

    def compute(self, node: GgmlTensor) -> None:
        check(self.L.ane_ggml_compute_forward(self.h, ctypes.byref(node)), "ane_ggml_compute_forward")

    def graph_compute(self, nodes) -> None:
        arr = (ctypes.POINTER(GgmlTensor) * len(nodes))(*[ctypes.pointer(n) for n in nodes])
        check(self.L.ane_ggml_graph_compute(self.h, arr, len(nodes)), "ane_ggml_graph_compute")

    def close(self) -> None:
        if self.h:
            self.L.ane_ggml_backend_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---------------------------------------------------------------- decode step
class DecodeConfig(ctypes.Structure):
    """Mirror of struct ane_decode_config (include/ane_decode.h)."""

    _fields_ = [(n, ctypes.c_uint32) for n in ("n_layers", "hidden", "ffn", "n_heads", "n_kv_heads",
                                                "head_dim", "ctx")] + [("eps", ctypes.c_float)]


class DecodeLayer(ctypes.Structure):
    """Mirror of struct ane_decode_layer (device pointers)."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("w_qkv", "w_o", "w_gate_up", "w_down", "attn_norm",
                                                "ffn_norm", "k_cache", "v_cache")]


def rope_table(ctx: int, head_dim: int = 128, base: float = 500000.0):
    """(cos, sin) of pos * base^(-2i/head_dim), fp32 [ctx][head_dim/2][2],
    computed in float64 and rounded once."""
    import numpy as np

    i = np.arange(head_dim // 2, dtype=np.float64)
    theta = np.power(base, -2.0 * i / head_dim)
    ang = np.arange(ctx, dtype=np.float64)[:, None] * theta[None, :]
    return np.stack([np.cos(ang), np.sin(ang)], axis=-1).astype(np.float32)


def q8_0_matvec_fused(N, K, x, W, y, norm_w=None, eps=0.0, residual=None, stream=None):
    check(lib().ane_hip_q8_0_matvec_fused(N, K, _p(x), _p(norm_w), eps, _p(W), _p(residual), _p(y),
                                          _stream_handle(stream)), "q8_0_matvec_fused")


def rope_kv_append(cfg, qkv, table, pos, k_cache, v_cache, stream=None):
    check(lib().ane_hip_rope_kv_append(ctypes.byref(cfg), _p(qkv), _p(table), pos, _p(k_cache), _p(v_cache),
                                       _stream_handle(stream)), "rope_kv_append")


def attention_decode(cfg, q, k_cache, v_cache, length, out, workspace=None, stream=None):
    L = lib()
    wsb = L.ane_hip_attention_workspace_size(ctypes.byref(cfg))
    ws = workspace if workspace is not None else _scratch(wsb, q.device, stream, zero=True)
    check(L.ane_hip_attention_decode(ctypes.byref(cfg), _p(q), _p(k_cache), _p(v_cache), length, _p(out), _p(ws),
                                     wsb, _stream_handle(stream)), "attention_decode")


def q8_0_matvec_silu(N, K, gu, W, y, residual=None, stream=None):
    check(lib().ane_hip_q8_0_matvec_silu(N, K, _p(gu), _p(W), _p(residual), _p(y), _stream_handle(stream)),
          "q8_0_matvec_silu")


def attention_decode_rope(cfg, qkv, table, pos, k_cache, v_cache, out, workspace=None, stream=None, out_q8=None):
    L = lib()
    wsb = L.ane_hip_attention_workspace_size(ctypes.byref(cfg))
    ws = workspace if workspace is not None else _scratch(wsb, qkv.device, stream, zero=True)
    check(L.ane_hip_attention_decode_rope(ctypes.byref(cfg), _p(qkv), _p(table), pos, _p(k_cache), _p(v_cache),
                                          _p(out), _p(out_q8), _p(ws), wsb, _stream_handle(stream)),
          "attention_decode_rope")


def silu_mul(n, gu, h, stream=None):
    check(lib().ane_hip_silu_mul(n, _p(gu), _p(h), _stream_handle(stream)), "silu_mul")


def q8_act_bytes(n):
    """Bytes of the Q8 activation form of n values: qx [n/32][32] int8, then dx [n/32] fp32."""
    return n // 32 * 36


def silu_mul_quant(n, gu, xq, stream=None):
    check(lib().ane_hip_silu_mul_quant(n, _p(gu), _p(xq), _stream_handle(stream)), "silu_mul_quant")


def q8_0_gate_up_silu_quant(F, K, x, norm_w, W, xq, eps=1e-5, stream=None):
    """xq = q8(silu(gate) * up) of the gate|up product (rows interleaved in 32-row groups)."""
    check(lib().ane_hip_q8_0_gate_up_silu_quant(F, K, _p(x), _p(norm_w), float(eps), _p(W), _p(xq),
                                                 _stream_handle(stream)), "q8_0_gate_up_silu_quant")


def interleave_gate_up(W_gate, W_up):
    """Rows of the decode step's w_gate_up: gate and up in alternating 32-row groups."""
    import numpy as np

    F = W_gate.shape[0]
    assert W_up.shape == W_gate.shape and F % 32 == 0
    return np.stack([W_gate.reshape(F // 32, 32, -1), W_up.reshape(F // 32, 32, -1)], axis=1).reshape(2 * F, -1)


def q8_0_matvec_q8(N, K, xq, W, y, residual=None, stream=None):
    check(lib().ane_hip_q8_0_matvec_q8(N, K, _p(xq), _p(W), _p(residual), _p(y), _stream_handle(stream)),
          "q8_0_matvec_q8")


def decode_workspace(cfg, device="cuda"):
    """A device workspace for decode_token."""
    import torch

    return torch.zeros(lib().ane_decode_workspace_size(ctypes.byref(cfg)), dtype=torch.uint8, device=device)


ARITH_BUILD = 0
ARITH_REFERENCE = 1


def rms_norm(K, x, w, eps, out, stream=None):
    """The build's RMSNorm (the fused products' arithmetic), one row."""
    check(lib().ane_hip_rms_norm(K, _p(x), _p(w), float(eps), _p(out), _stream_handle(stream)), "rms_norm")


def rms_norm_fp32(rows, dim, eps, x, w, out, stream=None):
    check(lib().ane_hip_rms_norm_fp32(rows, dim, float(eps), _p(x), _p(w), _p(out), _stream_handle(stream)),
          "rms_norm_fp32")


def silu_fp32(count, x, out, stream=None):
    check(lib().ane_hip_silu_fp32(count, _p(x), _p(out), _stream_handle(stream)), "silu_fp32")


def rope_fp32(rows, dim, pos, theta, x, out, stream=None):
    check(lib().ane_hip_rope_fp32(rows, dim, pos, float(theta), _p(x), _p(out), _stream_handle(stream)),
          "rope_fp32")


def softmax_fp32(rows, dim, x, out, stream=None):
    check(lib().ane_hip_softmax_fp32(rows, dim, _p(x), _p(out), _stream_handle(stream)), "softmax_fp32")


def decode_ggml_workspace(cfg, device="cuda"):
    import torch

    return torch.zeros(lib().ane_decode_ggml_workspace_size(ctypes.byref(cfg)), dtype=torch.uint8, device=device)


def decode_token_ggml(cfg, layers, table, pos, x, workspace, backend, arith=ARITH_BUILD, theta=500000.0):
    """One token through the ggml backend (GgmlBackend): MUL_MAT nodes for the
    products, the steps around them in the build's or the reference's arithmetic."""
    check(lib().ane_decode_token_ggml(ctypes.byref(cfg), layers, _p(table), float(theta), pos, _p(x),
                                      _p(workspace), workspace.numel(), backend.h, arith), "decode_token_ggml")


def decode_token(cfg, layers, table, pos, x, workspace, stream=None):
    """layers: a ctypes array of DecodeLayer (host memory)."""
    L = lib()
    check(L.ane_decode_token(ctypes.byref(cfg), layers, _p(table), pos, _p(x), _p(workspace),
                             workspace.numel(), _stream_handle(stream)), "decode_token")


# ---------------------------------------------------------------- paged cache, batches
NO_PAGE = -1  # ANE_NO_PAGE in the int32 tensors of page numbers


class PagedCache(ctypes.Structure):
    """Mirror of struct ane_paged_cache (include/ane_decode.h), over device
    tensors that it keeps alive: k_pages, v_pages fp16 [layers][pages][kv heads]
    [page size][head dim], page_table int32 [sequences][max pages] (NO_PAGE in
    unused entries), kv_len int32 [sequences], page_refs int32 [pages].  Calls
    go to these tensors: write into them, a new one needs a new PagedCache."""

    _fields_ = [(n, ctypes.c_uint32) for n in ("n_layers", "n_heads", "n_kv_heads", "head_dim", "page_size", "n_pages",
                                                "n_seqs", "max_pages")] + [
        (n, ctypes.c_void_p) for n in ("k_ptr", "v_ptr", "table_ptr", "len_ptr", "refs_ptr")]

    def __init__(self, n_heads, k_pages, v_pages, page_table, kv_len, page_refs=None):
        import torch

        if k_pages.dim() != 5 or k_pages.shape != v_pages.shape or page_table.dim() != 2:
            raise ValueError("k_pages and v_pages are [layers][pages][kv heads][page size][head dim], page_table "
                             "[sequences][max pages]")
        ints = [page_table, kv_len] + ([] if page_refs is None else [page_refs])
        if any(t.dtype != torch.float16 for t in (k_pages, v_pages)) or any(t.dtype != torch.int32 for t in ints):
            raise ValueError("pages are float16; page_table, kv_len and page_refs int32")
        if not all(t.is_contiguous() and t.device == k_pages.device for t in (k_pages, v_pages, *ints)):
            raise ValueError("the cache's tensors are contiguous and on one device")
        n_layers, n_pages, n_kv, page_size, head_dim = k_pages.shape
        if kv_len.numel() != page_table.shape[0] or (page_refs is not None and page_refs.numel() != n_pages):
            raise ValueError("kv_len has an entry for each sequence, page_refs one for each page")
        self.k_pages, self.v_pages, self.page_table = k_pages, v_pages, page_table
        self.kv_len, self.page_refs = kv_len, page_refs
        super().__init__(n_layers, n_heads, n_kv, head_dim, page_size, n_pages, page_table.shape[0],
                         page_table.shape[1], _p(k_pages), _p(v_pages), _p(page_table), _p(kv_len), _p(page_refs))
        # what every call asks for, as plain attributes (a field or a tensor's
        # property costs several times as much to read)
        self._at = ctypes.addressof(self)
        self._q, self._kv = (n_heads, head_dim), (n_kv, head_dim)
        self._scale = head_dim ** -0.5
        self._device = k_pages.get_device()  # -1: not on a GPU, and no call takes it
        self._types = {torch.float32: 0, torch.float16: 1}
        self._int32 = torch.int32
        self._cuda, self._current = torch.cuda, torch._C._cuda_getDevice
        self._raw_stream = torch._C._cuda_getCurrentRawStream
        self._pages_need = None

    @classmethod
    def empty(cls, n_layers, n_heads, n_kv_heads, head_dim, page_size, n_pages, n_seqs, max_pages, device="cuda"):
        """A cache whose pages are all free."""
        import torch

        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.float16, device=device) for _ in range(2))
        table = torch.full((n_seqs, max_pages), NO_PAGE, dtype=torch.int32, device=device)
        kv_len, refs = (torch.zeros(m, dtype=torch.int32, device=device) for m in (n_seqs, n_pages))
        return cls(n_heads, k, v, table, kv_len, refs)


def _rows(t, width, cache, what):
    """(pointer, type, tokens, row stride) of activations [tokens][heads][head_dim] whose heads are contiguous."""
    heads, dim = width
    tokens, h, d = t.shape if t.dim() == 3 else (0, 0, 0)
    if h != heads or d != dim:
        raise ValueError(f"{what} is [tokens][{heads}][{dim}]")
    ty = cache._types.get(t.dtype)
    if ty is None:
        raise ValueError(f"{what} is float32 or float16")
    if t.get_device() != cache._device:
        raise ValueError(f"{what} is on the cache's device")
    s0, s1, s2 = t.stride()
    if (s2 != 1 or (s1 != dim and heads > 1)) and tokens:
        raise ValueError(f"the heads of a token of {what} are contiguous")
    return t.data_ptr(), ty, tokens, s0 if tokens > 1 else heads * dim


def _ints(t, n, cache, what):
    """The pointer of a device array of at least n int32, or None."""
    if t is None:
        return None
    if t.dtype != cache._int32 or not t.is_contiguous() or t.numel() < n or t.get_device() != cache._device:
        raise ValueError(f"{what} is a contiguous int32 tensor of {n} entries on the cache's device")
    return t.data_ptr()


def _launch(fn, cache, what, stream, args):
    """fn(*args, stream) on the cache's device and, unless given, its current stream."""
    if cache._device < 0:
        raise ValueError("the cache is not in GPU memory")
    if cache._device == cache._current():
        st = fn(*args, cache._raw_stream(cache._device) if stream is None else _stream_handle(stream))
    else:
        with cache._cuda.device(cache._device):
            st = fn(*args, cache._raw_stream(cache._device) if stream is None else _stream_handle(stream))
    if st:
        check(st, what)


def _batch(q_start, seqs, rows, cache):
    """(n, q_start pointer, seqs pointer) of a packed batch of `rows` tokens."""
    n = rows if q_start is None else q_start.numel() - 1
    if n < 0:
        raise ValueError("q_start has an entry more than the batch has rows")
    return n, _ints(q_start, n + 1, cache, "q_start"), _ints(seqs, n, cache, "seqs")


def _work(cache, workspace, need, stream):
    """(workspace, pointer, bytes): the caller's, or a temporary one of need() bytes (the tensor has to
    live until the call is queued)."""
    if cache._device < 0:
        raise ValueError("the cache is not in GPU memory")
    if workspace is None:
        workspace = _scratch(need(), cache.k_pages.device, stream)
    elif workspace.get_device() != cache._device or not workspace.is_contiguous():
        raise ValueError("the workspace is contiguous, on the cache's device")
    return workspace, workspace.data_ptr(), workspace.nbytes


def paged_rope_append(cache, layer, q_start, q, k, v, table, q_out, seqs=None, stream=None):
    """RoPE of q and k and the append of k and v to the pages of one layer:
    q, k, v [tokens][heads][head_dim] (views of one qkv tensor will do), the new
    tokens of batch row i in rows q_start[i] .. q_start[i+1]-1 (None: one each);
    q_out takes the rotated q; q and q_out None: k and v only; table None: no
    rotation."""
    kp, ty, tokens, ks = _rows(k, cache._kv, cache, "k")
    vp, tv, nv, vs = _rows(v, cache._kv, cache, "v")
    if (ty, tokens, ks) != (tv, nv, vs):
        raise ValueError("k and v have the same shape, strides and type")
    n, qs, sq = _batch(q_start, seqs, tokens, cache)
    qp = op = None
    q0 = o0 = to = 0
    if q is not None and q_out is not None:
        qp, tq, nq, q0 = _rows(q, cache._q, cache, "q")
        op, to, no, o0 = _rows(q_out, cache._q, cache, "q_out")
        if tq != ty or nq != tokens or no < tokens:
            raise ValueError("q has the tokens and type of k, q_out room for them")
    elif q is not None or q_out is not None:
        raise ValueError("q and q_out go together")
    tp, positions = None, 0
    if table is not None:
        positions = table.shape[0]
        if (cache._types.get(table.dtype) != 0 or not table.is_contiguous()
                or table.numel() != positions * cache._q[1] or table.get_device() != cache._device):
            raise ValueError("table is a contiguous float32 [positions][head_dim/2][2] on the cache's device")
        tp = table.data_ptr()
    _launch(lib().ane_hip_paged_rope_append, cache, "paged_rope_append", stream,
            (cache._at, layer, sq, n, qs, tokens, ty, qp, q0, kp, vp, ks, tp, positions, to, op, o0))


def rope_freqs(rot_dim, base=10000.0, factor=1.0, scaling=None, context=8192, low=1.0, high=4.0):
    """(radians a position of each of the rot_dim/2 pairs in float64, the factor of cos and sin) for Rope: base^(-2i /
    rot_dim), for a context `factor` times the one of `context` positions the model was trained on scaled by

    None       not at all;
    "linear"   all of them divided by factor;
    "base"     base raised so that the slowest pair is divided by factor and the fastest kept;
    "turns"    divided by factor below `low` turns within the old context, kept from `high` turns on, blended by the
               number of turns in between;
    "index"    the same borders (usually low=1, high=32), blended by the pair's index, and cos and sin times
               0.1 ln(factor) + 1."""
    import numpy as np

    if rot_dim <= 0 or rot_dim % 2 or base <= 0 or factor <= 0 or context <= 0:
        raise ValueError("rot_dim is even, base, factor and context are positive")
    if scaling not in (None, "linear", "base", "turns", "index"):
        raise ValueError(f"unknown scaling {scaling!r}")
    i = np.arange(rot_dim // 2, dtype=np.float64)
    if scaling == "base" and rot_dim > 2:
        base = base * factor ** (rot_dim / (rot_dim - 2))
    f = np.power(float(base), -2.0 * i / rot_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling in ("turns", "index"):
        if not 0 < low < high:
            raise ValueError("0 < low < high")
        if scaling == "turns":
            keep = (context * f / (2 * np.pi) - low) / (high - low)
        else:
            at = [rot_dim * np.log(context / (2 * np.pi * t)) / (2 * np.log(base)) for t in (high, low)]
            first, last = max(np.floor(at[0]), 0), min(np.ceil(at[1]), rot_dim - 1)
            keep = 1.0 - (i - first) / max(last - first, 1e-3)
        keep = np.clip(keep, 0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    return f, (0.1 * np.log(factor) + 1.0 if scaling == "index" and factor > 1 else 1.0)


class Rope(ctypes.Structure):
    """Mirror of struct ane_rope (include/ane_decode.h) over a float64 device tensor of radians a position, which it
    keeps alive (rope_freqs makes the values); half: pairs (i, i + n) of a head's first 2 n values, else (2i, 2i + 1);
    factor multiplies cosines and sines."""

    _fields_ = [("rot_dim", ctypes.c_uint32), ("halves", ctypes.c_uint32), ("freqs_ptr", ctypes.c_void_p),
                ("factor", ctypes.c_double)]

    def __init__(self, freqs, half=False, factor=1.0):
        import torch

        if freqs.dtype != torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous():
            raise ValueError("freqs is a contiguous float64 tensor of a value a pair")
        self.freqs = freqs
        super().__init__(2 * freqs.numel(), int(bool(half)), _p(freqs), factor)
        self._at, self._device = ctypes.addressof(self), freqs.get_device()


def paged_norm_rope_append(cache, layer, q_start, q, k, v, rope, q_out, q_norm=None, k_norm=None, eps=1e-6, seqs=None,
                           stream=None):
    """RMSNorm of each q and k head (float32 weights [head_dim]; None: none), the rotation of `rope` (a Rope; None: none)
    and the append of k and v to the pages of one layer; the rest as paged_rope_append."""
    kp, ty, tokens, ks = _rows(k, cache._kv, cache, "k")
    vp, tv, nv, vs = _rows(v, cache._kv, cache, "v")
    if (ty, tokens, ks) != (tv, nv, vs):
        raise ValueError("k and v have the same shape, strides and type")
    n, qs, sq = _batch(q_start, seqs, tokens, cache)
    qp = op = None
    q0 = o0 = to = 0
    if q is not None and q_out is not None:
        qp, tq, nq, q0 = _rows(q, cache._q, cache, "q")
        op, to, no, o0 = _rows(q_out, cache._q, cache, "q_out")
        if tq != ty or nq != tokens or no < tokens:
            raise ValueError("q has the tokens and type of k, q_out room for them")
    elif q is not None or q_out is not None:
        raise ValueError("q and q_out go together")
    if rope is not None and rope._device != cache._device:
        raise ValueError("the rope's frequencies are on the cache's device")
    _launch(lib().ane_hip_paged_norm_rope_append, cache, "paged_norm_rope_append", stream,
            (cache._at, layer, sq, n, qs, tokens, ty, qp, q0, kp, vp, ks, None if rope is None else rope._at,
             _vector(q_norm, cache._q[1], cache._device, "q_norm"), _vector(k_norm, cache._q[1], cache._device, "k_norm"),
             eps, to, op, o0))


def _attention_rows(cache, q, out):
    qp, ty, tokens, q0 = _rows(q, cache._q, cache, "q")
    op, to, no, o0 = _rows(out, cache._q, cache, "out")
    if (ty, tokens) != (to, no):
        raise ValueError("out has the shape and type of q")
    return ty, tokens, qp, q0, op, o0


class AttentionRule(ctypes.Structure):
    """Mirror of struct ane_attention_rule (include/ane_decode.h), over device tensors that it keeps alive: scores capped
    at softcap by a tanh (0: not), lowered by slopes (float32 [heads]) times the distance, keys window and more positions
    back not seen (0: all), none before first (int32 [tokens]: where each new token's document begins; a token with a
    negative entry sees nothing), all below prefix (int32 [rows of the batch], none where it is 0 or negative) seen from
    both sides.  A call reads the tensors when it runs."""

    _fields_ = [("softcap", ctypes.c_float), ("window", ctypes.c_uint32), ("slopes_ptr", ctypes.c_void_p),
                ("first_ptr", ctypes.c_void_p), ("prefix_ptr", ctypes.c_void_p)]

    def __init__(self, softcap=0.0, slopes=None, window=0, first=None, prefix=None):
        import torch

        given = [t for t in (slopes, first, prefix) if t is not None]
        if slopes is not None and slopes.dtype != torch.float32:
            raise ValueError("slopes is a float32 tensor of a value a head")
        if any(t.dtype != torch.int32 for t in (first, prefix) if t is not None):
            raise ValueError("first and prefix are int32 tensors")
        if not all(t.dim() == 1 and t.is_contiguous() and t.get_device() == given[0].get_device() for t in given):
            raise ValueError("the rule's tensors are contiguous vectors on one device")
        if not 0 <= window < 1 << 32:
            raise ValueError("window is a number of positions")
        self.slopes, self.first, self.prefix = slopes, first, prefix
        super().__init__(softcap, window, _p(slopes) or None, _p(first) or None, _p(prefix) or None)
        self._at, self._device = ctypes.addressof(self), given[0].get_device() if given else None
        self._need = [None if t is None else t.numel() for t in (slopes, first, prefix)]


def _rule(rule, cache, tokens, n):
    """The rule's address, its tensors long enough for the call."""
    heads, first, prefix = rule._need
    if heads is not None and heads != cache._q[0]:
        raise ValueError("slopes has a value for each head")
    if (first is not None and first < tokens) or (prefix is not None and prefix < n):
        raise ValueError("first has an entry for each token, prefix one for each row of the batch")
    if rule._device is not None and rule._device != cache._device:
        raise ValueError("the rule's tensors are on the cache's device")
    return rule._at


def attention_prompt_workspace_size(cache, n, n_tokens, max_len=None, rule=None) -> int:
    if rule is not None:
        return int(lib().ane_hip_attention_rule_workspace_size(cache._at, n, n_tokens, max_len or 0, rule._at))
    return int(lib().ane_hip_attention_prompt_workspace_size(cache._at, n, n_tokens, max_len or 0))


def attention_prompt_workspace(cache, n, n_tokens, max_len=None, rule=None):
    """A workspace for attention_prompt calls of these very sizes, for callers that keep one (a smaller batch may need a
    larger one: the largest of theirs does for several)."""
    return _scratch(attention_prompt_workspace_size(cache, n, n_tokens, max_len, rule), cache.k_pages.device)


def attention_prompt(cache, layer, q_start, q, out, max_len=None, scale=None, seqs=None, workspace=None, stream=None,
                     rule=None):
    """Causal attention of packed prompts over the pages of one layer: q and out
    [tokens][heads][head_dim] float32 or float16, the new tokens of batch row i
    (its sequence's last positions, already appended) in rows q_start[i] ..
    q_start[i+1]-1 (q_start None: one each).  max_len bounds the sequences'
    lengths; scale None: 1/sqrt(head_dim); rule: an AttentionRule, for scores
    that are capped or lowered with the distance and for other masks."""
    ty, tokens, qp, q0, op, o0 = _attention_rows(cache, q, out)
    n, qs, sq = _batch(q_start, seqs, tokens, cache)
    workspace, wp, size = _work(cache, workspace,
                                lambda: attention_prompt_workspace_size(cache, n, tokens, max_len, rule), stream)
    scale = cache._scale if scale is None else scale
    if rule is not None:
        _launch(lib().ane_hip_attention_rule, cache, "attention_prompt", stream,
                (cache._at, layer, sq, n, qs, tokens, max_len or 0, _rule(rule, cache, tokens, n), ty, qp, q0, scale, op, o0,
                 wp, size))
        return
    _launch(lib().ane_hip_attention_prompt, cache, "attention_prompt", stream,
            (cache._at, layer, sq, n, qs, tokens, max_len or 0, ty, qp, q0, scale, op, o0, wp, size))


def attention_shared_workspace_size(cache, n, n_groups=0, max_prefix=None, max_len=None) -> int:
    return int(lib().ane_hip_attention_shared_workspace_size(cache._at, n, n_groups, max_prefix or 0, max_len or 0))


def attention_shared_workspace(cache, n, n_groups=0, max_prefix=None, max_len=None):
    """A workspace for attention_shared calls of these very sizes, for callers that keep one (a smaller batch may need a
    larger one: the largest of theirs does for several)."""
    return _scratch(attention_shared_workspace_size(cache, n, n_groups, max_prefix, max_len), cache.k_pages.device)


def attention_shared(cache, layer, q, out, max_len=None, group_start=None, prefix_len=None, max_prefix=None, scale=None,
                     seqs=None, workspace=None, stream=None):
    """One token of each batch row over the pages of one layer: q and out [rows]
    [heads][head_dim].  Rows group_start[g] .. group_start[g+1]-1 share their
    first prefix_len[g] positions, which are read once for the group;
    group_start None: no row shares anything."""
    ty, n, qp, q0, op, o0 = _attention_rows(cache, q, out)
    sq = _ints(seqs, n, cache, "seqs")
    if (group_start is None) != (prefix_len is None):
        raise ValueError("group_start and prefix_len go together")
    groups = 0 if group_start is None else group_start.numel() - 1
    gs, pl = _ints(group_start, groups + 1, cache, "group_start"), _ints(prefix_len, groups, cache, "prefix_len")
    workspace, wp, size = _work(
        cache, workspace, lambda: attention_shared_workspace_size(cache, n, groups, max_prefix, max_len), stream)
    _launch(lib().ane_hip_attention_shared, cache, "attention_shared", stream,
            (cache._at, layer, sq, n, groups, gs, pl, max_prefix or 0, max_len or 0, ty, qp, q0,
             cache._scale if scale is None else scale, op, o0, wp, size))


def _pages_need(cache) -> int:
    if cache._pages_need is None:
        cache._pages_need = int(lib().ane_hip_pages_workspace_size(cache._at))
    return cache._pages_need


def pages_workspace(cache):
    """A workspace for the page calls on this cache."""
    return _scratch(_pages_need(cache), cache.k_pages.device)


def pages_reserve(cache, seqs, new_len, served=None, workspace=None, stream=None):
    """Sequences seqs[i] grow to new_len[i] positions (int32 device tensors);
    served[i]: 1 where the pool had the pages."""
    n = seqs.numel()
    a, b, c = (_ints(t, n, cache, w) for t, w in ((seqs, "seqs"), (new_len, "new_len"), (served, "served")))
    workspace, wp, size = _work(cache, workspace, lambda: _pages_need(cache), stream)
    _launch(lib().ane_hip_pages_reserve, cache, "pages_reserve", stream, (cache._at, n, a, b, c, wp, size))


def pages_fork(cache, src, dst, served=None, workspace=None, stream=None):
    """Empty sequences dst[i] become copies of src[i] that share their whole pages."""
    n = src.numel()
    a, b, c = (_ints(t, n, cache, w) for t, w in ((src, "src"), (dst, "dst"), (served, "served")))
    workspace, wp, size = _work(cache, workspace, lambda: _pages_need(cache), stream)
    _launch(lib().ane_hip_pages_fork, cache, "pages_fork", stream, (cache._at, n, a, b, c, wp, size))


def pages_free(cache, seqs, stream=None):
    """The sequences become empty and give their pages up."""
    n = seqs.numel()
    _launch(lib().ane_hip_pages_free, cache, "pages_free", stream, (cache._at, n, _ints(seqs, n, cache, "seqs")))


def pages_copy(cache, src, dst, stream=None):
    """Pages dst[i] become copies of pages src[i] in every layer."""
    n = src.numel()
    _launch(lib().ane_hip_pages_copy, cache, "pages_copy", stream,
            (cache._at, n, _ints(src, n, cache, "src"), _ints(dst, n, cache, "dst")))


def pages_compact(cache, table_out=None, refs_out=None, n_live=None, workspace=None, stream=None):
    """The live pages move to the front of the pool; the new table and counts go
    to table_out and refs_out (None: the cache's own), the number of live pages
    to n_live."""
    t = _ints(table_out, cache.page_table.numel(), cache, "table_out")
    r, l = _ints(refs_out, cache.k_pages.shape[1], cache, "refs_out"), _ints(n_live, 1, cache, "n_live")
    workspace, wp, size = _work(cache, workspace, lambda: _pages_need(cache), stream)
    _launch(lib().ane_hip_pages_compact, cache, "pages_compact", stream, (cache._at, t, r, l, wp, size))


# ---------------------------------------------------------------- int8 linear layers of a batch
class _Torch:
    """What every call below asks torch for, looked up once (an import statement costs as much as a tensor's check)."""

    def __init__(self):
        import torch

        self.types = {torch.float32: 0, torch.float16: 1}
        self.float32, self.int8, self.device = torch.float32, torch.int8, torch.cuda.device
        self.current, self.raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


_TORCH: _Torch | None = None


def _torch() -> _Torch:
    global _TORCH
    if _TORCH is None:
        _TORCH = _Torch()
    return _TORCH


def _tokens(t, dev, what):
    """(pointer, type, tokens, values, row stride) of activations [tokens][values] whose values are contiguous."""
    ty = (_TORCH or _torch()).types.get(t.dtype)
    if ty is None or t.dim() != 2:
        raise ValueError(f"{what} is a float32 or float16 tensor [tokens][values]")
    (n, k), (s0, s1) = t.shape, t.stride()
    if t.get_device() != dev:
        raise ValueError(f"{what} is on the device of the others")
    if s1 != 1 and k > 1:
        raise ValueError(f"the values of a token of {what} are contiguous")
    if n > 1:
        if s0 < k:
            raise ValueError(f"the tokens of {what} do not overlap")
        return t.data_ptr(), ty, n, k, s0
    return t.data_ptr(), ty, n, k, k


def _vector(t, n, dev, what):
    """The pointer of n contiguous float32, or None."""
    if t is None:
        return None
    if t.dtype != (_TORCH or _torch()).float32 or t.numel() != n or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{what} is a contiguous float32 tensor of {n} values on the device of the others")
    return t.data_ptr()


def _int8_rows(t, k, dev, what):
    """(pointer, rows, row stride) of int8 rows of k values that can be read up to k rounded up to 16."""
    if t.dtype != (_TORCH or _torch()).int8 or t.dim() != 2 or t.get_device() != dev:
        raise ValueError(f"{what} is an int8 tensor [rows][{k}] on the device of the others")
    (n, width), (s0, s1) = t.shape, t.stride()
    if width != k or (s1 != 1 and k > 1):
        raise ValueError(f"{what} is an int8 tensor [rows][{k}], its rows contiguous")
    kp, p = (k + 15) // 16 * 16, t.data_ptr()
    if n <= 1:
        s0 = kp
    if (p | s0) & 15 or s0 < kp:
        raise ValueError(f"the rows of {what} start on 16 bytes (a view [:, :k] of rows of {kp} bytes will do)")
    if kp != k and n and t.storage_offset() + (n - 1) * s0 + kp > t.untyped_storage().nbytes():
        raise ValueError(f"the last row of {what} can be read up to {kp} bytes")
    return p, n, s0


def _on(dev, fn, what, stream, args):
    """fn(*args, stream) on device dev and, unless given, its current stream."""
    if dev < 0:
        raise ValueError("the tensors are not in GPU memory")
    t = _TORCH or _torch()
    if dev == t.current():
        st = fn(*args, t.raw_stream(dev) if stream is None else _stream_handle(stream))
    else:
        with t.device(dev):
            st = fn(*args, t.raw_stream(dev) if stream is None else _stream_handle(stream))
    if st:
        check(st, what)


def quantize_tokens(x, q, scales, norm_w=None, eps=1e-5, stream=None):
    """q, scales of activations x [tokens][values], each token on its own, after an RMSNorm where norm_w is given.
    q is int8 [tokens][values], its rows starting on 16 bytes; values past the last up to the next 16 are zeroed."""
    dev = x.get_device()
    xp, ty, n, k, xs = _tokens(x, dev, "x")
    qp, rows, qs = _int8_rows(q, k, dev, "q")
    if rows != n:
        raise ValueError("q has the shape of x")
    sp, wp = _vector(scales, n, dev, "scales"), _vector(norm_w, k, dev, "norm_w")
    _on(dev, lib().ane_hip_quantize_tokens, "quantize_tokens", stream, (n, k, ty, xp, xs, wp, eps, qp, qs, sp))


def _product(n, k, dev, w, w_scales, out, bias, residual):
    wp, rows, ws = _int8_rows(w, k, dev, "w")
    op, ty, no, width, os_ = _tokens(out, dev, "out")
    if no != n or width != rows:
        raise ValueError("out is [tokens][rows of w]")
    rp, rs = None, 0
    if residual is not None:
        rp, tr, nr, wr, rs = _tokens(residual, dev, "residual")
        if (tr, nr, wr) != (ty, no, width):
            raise ValueError("residual has the shape and type of out")
    return rows, wp, ws, _vector(w_scales, rows, dev, "w_scales"), _vector(bias, rows, dev, "bias"), rp, rs, ty, op, os_


def dense_i8_scaled(q, q_scales, w, w_scales, out, bias=None, residual=None, stream=None):
    """out [tokens][rows of w] = the product of int8 tokens q and int8 weights w, times the scales of token and row,
    plus bias [rows of w] and residual (out's shape and type; may be out).  Rows of q hold zeros from their last value
    up to the next 16 (quantize_tokens writes them)."""
    dev = q.get_device()
    k = q.shape[-1]
    qp, n, qs = _int8_rows(q, k, dev, "q")
    rows, wp, ws, cp, bp, rp, rs, ty, op, os_ = _product(n, k, dev, w, w_scales, out, bias, residual)
    _on(dev, lib().ane_hip_dense_i8_scaled, "dense_i8_scaled", stream,
        (n, rows, k, qp, qs, _vector(q_scales, n, dev, "q_scales"), wp, ws, cp, bp, rp, rs, ty, op, os_))


def linear_i8_workspace_size(T, N, K) -> int:
    return int(lib().ane_hip_linear_i8_workspace_size(T, N, K))


def linear_i8_workspace(T, N, K, device="cuda"):
    """A workspace for linear_i8 calls of up to T tokens through weights [N][K], for callers that keep one."""
    return _scratch(linear_i8_workspace_size(T, N, K), device)


def linear_i8(x, w, w_scales, out, norm_w=None, eps=1e-5, bias=None, residual=None, workspace=None, stream=None):
    """out [tokens][rows of w]: activations x [tokens][values] quantized a token at a time (after an RMSNorm where
    norm_w is given), times int8 weights w [rows][values] with a scale a row, plus bias and residual (may be out; out may
    be x)."""
    dev = x.get_device()
    xp, ty, n, k, xs = _tokens(x, dev, "x")
    rows, wp, ws, cp, bp, rp, rs, to, op, os_ = _product(n, k, dev, w, w_scales, out, bias, residual)
    np_ = _vector(norm_w, k, dev, "norm_w")
    if workspace is None:
        if dev < 0:
            raise ValueError("the tensors are not in GPU memory")
        workspace = _scratch(linear_i8_workspace_size(n, rows, k), x.device, stream)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("the workspace is contiguous, on the device of the others")
    _on(dev, lib().ane_hip_linear_i8, "linear_i8", stream,
        (n, rows, k, ty, xp, xs, np_, eps, wp, ws, cp, bp, rp, rs, to, op, os_, workspace.data_ptr(), workspace.nbytes))
