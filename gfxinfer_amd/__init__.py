"""gfxinfer_amd: MI355X (gfx950) speculative-verify hot path.

Python view of the C ABI declared in include/gfxinfer_amd.h.  The compute lives
in libgfxinfer_amd.so (hand-written HIP for gfx950); this module only loads it,
declares the signatures and offers thin wrappers that mirror the reference
launchers (src/kernels/lowbit_gemv.hip, src/kernels/qwen_ops.hip) with the same
argument meaning and error behaviour: a non-zero status raises GfxinferError
carrying the reference ErrorCode value and message.

There is no fallback: if the library is missing, importing the wrappers fails.
"""
from __future__ import annotations

import ctypes
import functools
import os
import re
import subprocess
from array import array

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
# GFXINFER_AMD_LIBRARY selects another build of the same library (the host-sanitizer
# build of `make -C gfxinfer_amd sanitize`); the default is the in-tree build.
LIBRARY = os.environ.get("GFXINFER_AMD_LIBRARY") or os.path.join(HERE, "libgfxinfer_amd.so")
HEADERS = [os.path.join(ROOT, "include", "gfxinfer_amd.h"),
           os.path.join(ROOT, "include", "gfxinfer_runtime.h")]

# include/gfxinfer/status.h:11-20
OK, INVALID_ARGUMENT, IO_ERROR, CORRUPT_ARTIFACT, UNSUPPORTED, HIP_ERROR, OUT_OF_MEMORY, INTERNAL = range(8)
# include/gfxinfer/artifact.h:26-33
W2G128, W3G128, W4G128 = 1, 2, 3
TYPE_F16, TYPE_F32, TYPE_BF16 = 0, 1, 2  # GFXI_F16, GFXI_F32, GFXI_BF16
ERROR_NAMES = {0: "ok", 1: "invalid_argument", 2: "io_error", 3: "corrupt_artifact",
               4: "unsupported", 5: "hip_error", 6: "out_of_memory", 7: "internal"}


class GfxinferError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"{ERROR_NAMES.get(code, code)}: {message}")
        self.code = code
        self.message = message


def build(jobs: int = 8) -> None:
    """Compile libgfxinfer_amd.so for gfx950 in-tree."""
    subprocess.run(["make", "-s", "-C", HERE, f"-j{jobs}"], check=True)


_lib: ctypes.CDLL | None = None

P = ctypes.c_void_p
SZ = ctypes.c_size_t
U32 = ctypes.c_uint32
I32 = ctypes.c_int32
F32 = ctypes.c_float

# name -> (restype, argtypes).  Every function of include/gfxinfer_amd.h.
SIGNATURES: dict[str, tuple] = {
    "gfxinfer_last_error": (ctypes.c_char_p, []),
    "gfxinfer_require_gfx950_device": (I32, [I32]),
    "gfxinfer_packed_row_bytes": (SZ, [I32, SZ]),
    "gfxinfer_tile_group128_for_gfx950": (I32, [I32, P, P, SZ, SZ, P, P]),
    "gfxinfer_untile_group128_for_gfx950": (I32, [I32, P, P, SZ, SZ, P, P]),
    "gfxinfer_launch_quantize_group128_gfx950": (I32, [I32, P, SZ, SZ, P, P, P, P]),
    "gfxinfer_launch_quantize_activation_i4": (I32, [P, P, P, SZ, U32, P]),
    "gfxinfer_launch_quantize_activation_i8": (I32, [P, P, P, SZ, U32, P]),
    "gfxinfer_launch_gfx950_i4_gemm": (I32, [I32, P, P, P, P, P, SZ, SZ, U32, I32, P]),
    "gfxinfer_launch_gfx950_i4_gemm_split": (I32, [I32, P, P, P, P, P, SZ, SZ, U32, U32, P]),
    "gfxinfer_gemm_split_count": (U32, [SZ, SZ, U32]),
    "gfxinfer_launch_gfx950_i4_gemm_half": (I32, [I32, P, P, P, P, P, SZ, SZ, U32, I32, P]),
    "gfxinfer_launch_gfx950_i4_gemm_fused": (I32, [I32, P, SZ, P, P, SZ, U32, I32, P]),
    "gfxinfer_launch_gfx950_i8_gemm": (I32, [I32, P, P, P, P, P, SZ, SZ, U32, P]),
    "gfxinfer_gemm_argmax_workspace_bytes": (SZ, [SZ, U32]),
    "gfxinfer_launch_gfx950_i4_gemm_argmax": (I32, [I32, P, P, P, P, P, SZ, SZ, U32, SZ, P, P, SZ, P, P]),
    "gfxinfer_launch_gfx950_i4_gemm_argmax_no_alloc": (I32, [I32, P, P, P, P, P, SZ, SZ, U32, SZ, P, P, P]),
    "gfxinfer_debug_gemm_partials": (I32, [I32, P, I32, P, SZ, SZ, U32, P, P]),
    "gfxinfer_debug_gemm_family": (I32, [I32, I32, P, P, P, P, P, I32, P, P, U32, SZ, SZ, U32, U32, P]),
    "gfxinfer_debug_gemm_direct_shape": (I32, [I32, SZ, SZ, U32, U32]),
    "gfxinfer_debug_gemm_prefill_workspace_bytes": (SZ, [SZ, U32]),
    "gfxinfer_debug_gemm_prefill": (I32, [I32, P, P, P, P, P, I32, SZ, SZ, U32, U32, P, SZ, P]),
    "gfxinfer_debug_stream_read": (I32, [P, SZ, P, U32, P]),
    "gfxinfer_debug_stream_read_oneshot": (I32, [P, SZ, P, U32, P]),
    "gfxinfer_launch_lowbit_row_gather_tiled": (I32, [I32, P, P, P, SZ, SZ, SZ, P]),
    "gfxinfer_launch_lowbit_row_gather_tiled_indirect": (I32, [I32, P, P, P, P, SZ, SZ, P]),
    "gfxinfer_launch_lowbit_row_gather_tiled_batch": (I32, [I32, P, P, P, P, P, P, U32, SZ, SZ, P]),
    "gfxinfer_launch_rms_norm": (I32, [P, P, P, SZ, F32, I32, P]),
    "gfxinfer_launch_rms_norm_batch": (I32, [P, P, P, SZ, U32, F32, I32, P]),
    "gfxinfer_launch_residual_add_rms_norm_batch": (I32, [P, P, P, P, P, SZ, U32, F32, I32, P]),
    "gfxinfer_launch_rms_norm_quantize_i4": (I32, [P, P, P, P, P, SZ, U32, F32, I32, P]),
    "gfxinfer_launch_residual_add_rms_norm_quantize_i4": (I32, [P, P, P, P, P, P, P, SZ, U32, F32, I32, P]),
    "gfxinfer_launch_residual_add_rms_norm_quantize_i4_planes": (I32, [P, P, U32, P, P, P, P, P, SZ, U32, F32, I32, P]),
    "gfxinfer_launch_dual_rms_norm_concat": (I32, [P, P, P, P, P, SZ, F32, I32, P]),
    "gfxinfer_launch_mtp_input_quantize_i4": (I32, [I32, P, P, SZ, U32, P, P, P, P, P, P, P, SZ, F32, I32, P]),
    "gfxinfer_launch_mtp_input_quantize_i4_from_keys": (I32, [I32, P, P, SZ, P, SZ, P, P, P, P, P, P, P, P, SZ, F32, I32, P]),
    "gfxinfer_launch_dual_rms_norm_concat_batch": (I32, [P, P, P, P, P, SZ, U32, F32, I32, P]),
    "gfxinfer_launch_silu_multiply": (I32, [P, P, P, SZ, P]),
    "gfxinfer_launch_silu_multiply_quantize_i4": (I32, [P, P, P, P, SZ, U32, P]),
    "gfxinfer_launch_float_to_half": (I32, [P, P, SZ, P]),
    "gfxinfer_launch_gdn_conv_update_block": (I32, [P, P, P, P, P, P, SZ, U32, P]),
    "gfxinfer_launch_gdn_recurrent_decode_block": (I32, [P, P, P, P, P, P, P, P, P, P, P, P, P, U32, U32, U32, U32, P, P]),
    "gfxinfer_launch_gdn_recurrent_window": (I32, [P, P, P, P, P, P, P, P, P, P, P, U32, U32, U32, U32, P]),
    "gfxinfer_launch_gdn_output_quantize_i4": (I32, [P, P, P, P, P, P, U32, U32, U32, P]),
    "gfxinfer_launch_gdn_conv_window": (I32, [P, P, P, P, P, P, P, P, P, P, P, P, P, P, P, U32, U32, U32, U32, P]),
    "gfxinfer_launch_gdn_restore_prefix_all": (I32, [P, P, P, P, P, P, SZ, U32, U32, U32, U32, U32, U32, P]),
    "gfxinfer_launch_qk_rms_norm_rope_block": (I32, [P, P, P, SZ, SZ, P, P, P, SZ, SZ, SZ, SZ, ctypes.c_uint64, U32, F32, P]),
    "gfxinfer_launch_qk_rms_norm_rope_block_indirect_position": (I32, [P, P, P, SZ, SZ, P, P, P, SZ, SZ, SZ, SZ, P, U32, F32, P]),
    "gfxinfer_launch_qk_rms_norm_rope_kv_append_block": (I32, [P, P, P, SZ, SZ, P, P, P, SZ, SZ, SZ, SZ, P, P, P, SZ, ctypes.c_uint64, U32, F32, P]),
    "gfxinfer_launch_qk_rms_norm_rope_kv_append_block_indirect_position": (I32, [P, P, P, SZ, SZ, P, P, P, SZ, SZ, SZ, SZ, P, P, P, SZ, P, U32, F32, P]),
    "gfxinfer_launch_kv_append_block": (I32, [P, P, P, P, SZ, SZ, U32, SZ, P]),
    "gfxinfer_launch_kv_append_block_indirect_position": (I32, [P, P, P, P, P, SZ, U32, SZ, P]),
    "gfxinfer_launch_argmax_batch": (I32, [P, P, SZ, SZ, U32, P]),
    "gfxinfer_launch_argmax_mapped": (I32, [P, P, P, SZ, P]),
    "gfxinfer_attention_workspace_bytes": (SZ, [U32, U32, U32, SZ]),
    "gfxinfer_launch_gated_attention_decode_block": (I32, [P, P, P, P, P, SZ, SZ, U32, U32, U32, U32, P, SZ, P]),
    "gfxinfer_launch_gated_attention_decode_block_indirect_position": (I32, [P, P, P, P, P, P, SZ, U32, U32, U32, U32, P, SZ, P]),
    "gfxinfer_launch_gated_attention_decode_block_quantize_i4": (I32, [P, P, P, P, P, P, P, SZ, SZ, U32, U32, U32, U32, P, SZ, P]),
    "gfxinfer_launch_gated_attention_decode_block_quantize_i4_indirect_position": (I32, [P, P, P, P, P, P, P, P, SZ, U32, U32, U32, U32, P, SZ, P]),
    "gfxinfer_launch_qk_rms_norm_rope_kv_append_attention_quantize_i4": (I32, [P, P, SZ, P, P, SZ, P, SZ, F32, P, P, P, P, P, P, P, SZ, SZ, U32, U32, U32, U32, P, SZ, P]),
    "gfxinfer_launch_qk_rms_norm_rope_kv_append_attention_quantize_i4_indirect_position": (I32, [P, P, SZ, P, P, SZ, P, SZ, F32, P, P, P, P, P, P, P, P, SZ, U32, U32, U32, U32, P, SZ, P]),
    "gfxinfer_rope_table_bytes": (SZ, [SZ, SZ]),
    "gfxinfer_launch_rope_table": (I32, [P, SZ, SZ, F32, P]),
    "gfxinfer_fused_rope_attention_supported": (I32, [U32, U32, U32, U32]),
    "gfxinfer_launch_gdn_conv_update": (I32, [P, P, P, P, SZ, P]),
    "gfxinfer_launch_gdn_recurrent_decode": (I32, [P, P, P, P, P, P, P, P, P, U32, U32, U32, P, P]),
    "gfxinfer_launch_gdn_restore_prefix": (I32, [P, P, P, P, P, P, SZ, U32, U32, U32, U32, P]),
    "gfxinfer_launch_kv_append": (I32, [P, P, P, P, SZ, SZ, SZ, P]),
    "gfxinfer_launch_gated_attention_decode": (I32, [P, P, P, P, P, SZ, SZ, U32, U32, U32, P, SZ, P]),
    "gfxinfer_qwen38_scratch_bytes": (SZ, [U32, SZ]),
    "gfxinfer_qwen38_bind_scratch": (I32, [P, P, SZ, U32, SZ]),
    "gfxinfer_qwen38_unbind_scratch": (I32, [P]),
    "gfxinfer_qwen38_launch_gated_attention_decode": (I32, [P, P, P, P, P, SZ, SZ, P]),
    "gfxinfer_qwen38_launch_gated_attention_decode_block": (I32, [P, P, P, P, P, SZ, SZ, U32, P]),
    "gfxinfer_qwen38_launch_gated_attention_decode_block_indirect_position": (I32, [P, P, P, P, P, P, SZ, U32, P]),
    "gfxinfer_qwen38_launch_gdn_recurrent_decode_block": (I32, [P] * 13 + [U32, P]),
    "gfxinfer_qwen38_launch_gdn_recurrent_decode": (I32, [P] * 10),
    "gfxinfer_launch_argmax": (I32, [P, P, SZ, P]),
    "gfxinfer_kv_pages_workspace_bytes": (SZ, [P]),
    "gfxinfer_launch_kv_pages_reset": (I32, [P, P]),
    "gfxinfer_launch_kv_pages_fork": (I32, [P, U32, P, U32, P]),
    "gfxinfer_launch_kv_pages_reserve": (I32, [P, P, U32, U32, P, P, SZ, P]),
    "gfxinfer_launch_kv_pages_append": (I32, [P, U32, P, P, P, U32, U32, P]),
    "gfxinfer_launch_kv_pages_advance": (I32, [P, P, U32, U32, P, P]),
    "gfxinfer_launch_kv_pages_free": (I32, [P, P, P, U32, P]),
    "gfxinfer_launch_kv_pages_copy": (I32, [P, P, P, U32, P]),
    "gfxinfer_launch_kv_pages_compact": (I32, [P, P, P, SZ, P]),
    "gfxinfer_kv_pages_attention_workspace_bytes": (SZ, [P, U32, U32, U32, SZ]),
    "gfxinfer_launch_kv_pages_gated_attention": (I32, [P, U32, P, P, P, P, U32, U32, U32, SZ, P, SZ, P]),
    "gfxinfer_kv_pages_chunk_attention_workspace_bytes": (SZ, [P, P, U32, U32]),
    "gfxinfer_launch_kv_pages_chunk_attention": (I32, [P, U32, P, P, P, P, P, P, U32, U32, P, SZ, P]),
    "gfxinfer_launch_kv_weights_begin": (I32, [P, P, P, P, U32, P]),
    "gfxinfer_kv_weights_workspace_bytes": (SZ, [P, P, U32, U32]),
    "gfxinfer_launch_kv_weights_add": (I32, [P, P, U32, P, P, P, P, U32, U32, P, SZ, P]),
    "gfxinfer_kv_pages_evict_workspace_bytes": (SZ, [P, U32, U32]),
    "gfxinfer_launch_kv_pages_evict": (I32, [P, P, P, U32, U32, U32, U32, P, P, SZ, P]),
    "gfxinfer_launch_quantize_rows_i8": (I32, [P, I32, SZ, SZ, SZ, P, P, P]),
    "gfxinfer_w8a8_gemm_workspace_bytes": (SZ, [SZ, SZ, SZ]),
    "gfxinfer_launch_w8a8_gemm": (I32, [P, P, P, P, P, I32, SZ, SZ, SZ, P, SZ, P]),
    "gfxinfer_logit_rules_workspace_bytes": (SZ, [SZ, U32]),
    "gfxinfer_launch_logit_rules": (I32, [P, SZ, SZ, U32, P, P, SZ, P, P, SZ, P]),
    # include/gfxinfer_runtime.h
    "gfxinfer_model_spec_qwen38_27b": (None, [P]),
    "gfxinfer_model_spec_qwen38_reference": (None, [P]),
    "gfxinfer_model_spec_tensor_count": (SZ, [P]),
    "gfxinfer_model_spec_tensor": (I32, [P, SZ, P]),
    "gfxinfer_model_create_synthetic": (I32, [P, ctypes.c_uint64, I32, P]),
    "gfxinfer_model_destroy": (None, [P]),
    "gfxinfer_model_stream": (P, [P]),
    "gfxinfer_model_weight_bytes": (SZ, [P]),
    "gfxinfer_model_find_tensor": (I32, [P, ctypes.c_char_p, P]),
    "gfxinfer_model_copy_tensor": (I32, [P, ctypes.c_char_p, I32, P, SZ]),
    "gfxinfer_artifact_open": (I32, [ctypes.c_char_p, I32, P]),
    "gfxinfer_artifact_close": (None, [P]),
    "gfxinfer_artifact_get_identity": (I32, [P, P]),
    "gfxinfer_artifact_tensor_count": (SZ, [P]),
    "gfxinfer_artifact_tensor_at": (I32, [P, SZ, P]),
    "gfxinfer_artifact_find": (I32, [P, ctypes.c_char_p, P]),
    "gfxinfer_artifact_bytes": (P, [P, ctypes.c_uint64, ctypes.c_uint64]),
    "gfxinfer_crc64_ecma": (ctypes.c_uint64, [ctypes.c_uint64, P, SZ]),
    "gfxinfer_artifact_resource": (I32, [P, ctypes.c_char_p, ctypes.POINTER(P), ctypes.POINTER(ctypes.c_uint64)]),
    "gfxinfer_tokenizer_create": (I32, [P, SZ, ctypes.POINTER(P)]),
    "gfxinfer_tokenizer_destroy": (None, [P]),
    "gfxinfer_tokenizer_vocabulary_size": (SZ, [P]),
    "gfxinfer_tokenizer_encode": (I32, [P, ctypes.c_char_p, SZ, P, SZ, ctypes.POINTER(SZ)]),
    "gfxinfer_tokenizer_decode": (I32, [P, P, SZ, P, SZ, ctypes.POINTER(SZ)]),
    "gfxinfer_render_chat_prompt": (I32, [ctypes.c_char_p, SZ, P, SZ, ctypes.POINTER(SZ)]),
    "gfxinfer_retile_gfx12_for_gfx950": (I32, [I32, P, SZ, P]),
    "gfxinfer_model_create_from_artifact": (I32, [P, ctypes.c_char_p, I32, I32, P]),
    "gfxinfer_model_write_artifact": (I32, [P, ctypes.c_char_p, ctypes.c_char_p, P, SZ]),
    "gfxinfer_session_create": (I32, [P, P, P]),
    "gfxinfer_session_destroy": (None, [P]),
    "gfxinfer_session_greedy_step": (I32, [P, U32, P]),
    "gfxinfer_session_block_step": (I32, [P, P, SZ, P]),
    "gfxinfer_session_mtp_draft": (I32, [P, U32, P]),
    "gfxinfer_session_speculative_step": (I32, [P, U32, SZ, P]),
    "gfxinfer_session_speculative_step_forced": (I32, [P, U32, SZ, U32, P]),
    "gfxinfer_session_speculative_step_planted": (I32, [P, U32, SZ, P, P]),
    "gfxinfer_session_position": (SZ, [P]),
    "gfxinfer_session_mtp_position": (SZ, [P]),
    "gfxinfer_session_get_summary": (I32, [P, P]),
    "gfxinfer_session_copy_buffer": (I32, [P, ctypes.c_char_p, SZ, P, SZ]),
    "gfxinfer_session_buffer_bytes": (SZ, [P, ctypes.c_char_p]),
    "gfxinfer_session_set_layer_trace": (I32, [P, P, SZ]),
    "gfxinfer_session_layer_trace_bytes": (SZ, [P]),
    "gfxinfer_session_prefill": (I32, [P, P, SZ, I32, P]),
    "gfxinfer_debug_model_wide_scratch": (SZ, [P, I32]),
    "gfxinfer_session_generate": (I32, [P, P, SZ, P, P, P, P]),
    "gfxinfer_depth_policy_create": (I32, [U32, P]),
    "gfxinfer_depth_policy_destroy": (None, [P]),
    "gfxinfer_depth_policy_choose": (U32, [P, U32]),
    "gfxinfer_depth_policy_record": (I32, [P, U32, U32, ctypes.c_double]),
}


class FusedMatrix(ctypes.Structure):
    """gfxinfer_fused_matrix (lowbit_gemv.h:128-133 Gfx12I4FusedMatrix)."""
    _fields_ = [("tiled_weights", P), ("tiled_weight_scales", P), ("output", P), ("rows", SZ)]


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIBRARY):
            raise RuntimeError(
                f"{LIBRARY} is not built; run __graft_entry__.build() (hipcc for gfx950)")
        # PyTorch-ROCm ships its own libamdhip64 (soname libamdhip64.so.7).  Loading it
        # first lets this library bind to that same HIP runtime; loading
        # /opt/rocm's copy first would put two HIP runtimes in one process.
        try:
            import torch
            global _current_device, _raw_stream, _half, _real, _word
            _current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
            _half, _real, _word = (torch.float16, torch.int16, torch.uint16), (torch.float32,), (torch.int32, torch.uint32)
        except ImportError:
            pass
        L = ctypes.CDLL(LIBRARY)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def header_functions() -> list[str]:
    """Names of every function declared in include/*.h."""
    text = "\n".join(open(h).read() for h in HEADERS)
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(gfxinfer_[a-z0-9_]+)\s*\(", text)))


def last_error() -> str:
    return lib().gfxinfer_last_error().decode()


def check(status: int) -> None:
    if status != OK:
        raise GfxinferError(status, last_error())


def _p(x) -> int | None:
    """Device/host address of a torch tensor, numpy array or raw int."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    return x.ctypes.data


# This thread's device and its current stream there, and the element types of checked operands (fp16 numbers also as their
# bits); set by lib().
_current_device = _raw_stream = None
_half = _real = _word = ()


def _device_of(tensors, what):
    """The device all tensors are on: its number, -1 for memory that no GPU reaches.  Pinned host memory goes with any (None)."""
    found = {t.get_device() for t in tensors if t.is_cuda or not t.is_pinned()}
    if len(found) > 1:
        raise ValueError(f"{what}: tensors of different devices")
    return found.pop() if found else None


def _operand(x, types, size, device, what):
    """Address of an operand of `size` bytes: a contiguous tensor of one of the types in memory of that device (None: of any),
    or an address, which is the caller's to know.  0.16 us more than taking the address (0.3 of an append's 4.5 us)."""
    try:
        if x.get_device() == device and x.dtype in types and x.nbytes >= size and x.is_contiguous():
            return x.data_ptr()
    except AttributeError:
        if x is None or isinstance(x, int):
            return x
        raise ValueError(f"{what}: a tensor or an address") from None
    if x.dtype not in types or x.nbytes < size or not x.is_contiguous():
        raise ValueError(f"{what}: a contiguous tensor of {size} bytes or more, {' / '.join(str(t)[6:] for t in types)}")
    if not (x.is_pinned() if not x.is_cuda else device is None):
        raise ValueError(f"{what} is not in the memory of the GPU that the call runs on")
    return x.data_ptr()


def _scratch(workspace, device):
    """Address and bytes of a workspace, which may be of any type."""
    if workspace is None:
        return None, 0
    return _operand(workspace, (workspace.dtype,), 0, device, "workspace"), workspace.nbytes


def _launch_stream(device, stream):
    """The stream's handle, if a launch there reaches the memory of that device (None: not known)."""
    if device is not None:
        if stream is None and device == _current_device():
            return _raw_stream(device)
        if stream is None or device < 0:
            raise GfxinferError(INVALID_ARGUMENT, "the tensors of the call are not in the memory of the current device")
    return _stream(stream)


_current_stream = None


def _stream(stream) -> int | None:
    if stream is None:
        # The handle of torch.cuda.current_stream() without its Stream object (2.8 us a call,
        # as much as the launch itself; looking torch's modules up each time takes 0.3 us).
        global _current_stream
        if _current_stream is None:
            import torch
            torch.cuda.current_device()  # initializes, or raises without a GPU
            device, raw = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
            _current_stream = lambda: raw(device())  # noqa: E731
        return _current_stream()
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


# ---- wrappers (reference launcher names, lowbit_gemv.h) ---------------------

def launch_quantize_activation_i4(x, packed, scales, columns, batch, stream=None):
    check(lib().gfxinfer_launch_quantize_activation_i4(_p(x), _p(packed), _p(scales), columns, batch, _stream(stream)))


def launch_quantize_activation_i8(x, codes, scales, columns, batch, stream=None):
    check(lib().gfxinfer_launch_quantize_activation_i8(_p(x), _p(codes), _p(scales), columns, batch, _stream(stream)))


def launch_quantize_group128(fmt, weights, rows, columns, codes, scales, flag=None, stream=None):
    check(lib().gfxinfer_launch_quantize_group128_gfx950(fmt, _p(weights), rows, columns, _p(codes), _p(scales), _p(flag), _stream(stream)))


def launch_i4_gemm(fmt, w, ws, a, as_, out, rows, columns, batch, stream=None):
    check(lib().gfxinfer_launch_gfx950_i4_gemm(fmt, _p(w), _p(ws), _p(a), _p(as_), _p(out), rows, columns, batch, 1, _stream(stream)))


def launch_i4_gemm_split(fmt, w, ws, a, as_, planes, rows, columns, batch, splits, stream=None):
    """Split-K GEMM: `splits` fp32 planes [splits, batch, rows] whose sum is the product."""
    check(lib().gfxinfer_launch_gfx950_i4_gemm_split(fmt, _p(w), _p(ws), _p(a), _p(as_), _p(planes), rows, columns, batch, splits, _stream(stream)))


def gemm_split_count(rows, columns, batch):
    return int(lib().gfxinfer_gemm_split_count(rows, columns, batch))


def launch_i4_gemm_half(fmt, w, ws, a, as_, out, rows, columns, batch, stream=None):
    check(lib().gfxinfer_launch_gfx950_i4_gemm_half(fmt, _p(w), _p(ws), _p(a), _p(as_), _p(out), rows, columns, batch, 1, _stream(stream)))


def launch_i4_gemm_fused(fmt, matrices, a, as_, columns, batch, stream=None):
    """matrices: list of (weights, scales, output, rows)."""
    arr = (FusedMatrix * len(matrices))(*[FusedMatrix(_p(w), _p(s), _p(o), r) for (w, s, o, r) in matrices])
    check(lib().gfxinfer_launch_gfx950_i4_gemm_fused(fmt, ctypes.cast(arr, P), len(matrices), _p(a), _p(as_), columns, batch, 1, _stream(stream)))


def launch_i8_gemm(fmt, w, ws, a, as_, out, rows, columns, batch, stream=None):
    check(lib().gfxinfer_launch_gfx950_i8_gemm(fmt, _p(w), _p(ws), _p(a), _p(as_), _p(out), rows, columns, batch, _stream(stream)))


def debug_gemm_partials(fmt, w, abits, a, rows, columns, batch, partials, stream=None):
    check(lib().gfxinfer_debug_gemm_partials(fmt, _p(w), abits, _p(a), rows, columns, batch, _p(partials), _stream(stream)))


GEMM_MFMA, GEMM_DOT = 1, 2


def debug_gemm_family(family, fmt, w, ws, a, as_, rows, columns, batch, out=None, half_output=False,
                      partials=None, argmax_keys=None, argmax_rows=0, splits=1, stream=None):
    """One A4 GEMM launch through a named kernel family (GEMM_MFMA or GEMM_DOT); returns the status."""
    return int(lib().gfxinfer_debug_gemm_family(family, fmt, _p(w), _p(ws), _p(a), _p(as_), _p(out),
                                                1 if half_output else 0, _p(partials), _p(argmax_keys),
                                                argmax_rows, rows, columns, batch, splits, _stream(stream)))


def debug_stream_read(data, nbytes, sink, workgroups, stream=None):
    check(lib().gfxinfer_debug_stream_read(_p(data), nbytes, _p(sink), workgroups, _stream(stream)))


def debug_stream_read_oneshot(data, nbytes, sink, loads_per_lane, stream=None):
    check(lib().gfxinfer_debug_stream_read_oneshot(_p(data), nbytes, _p(sink), loads_per_lane, _stream(stream)))


def launch_row_gather_tiled(fmt, w, ws, out, row, rows, columns, stream=None):
    check(lib().gfxinfer_launch_lowbit_row_gather_tiled(fmt, _p(w), _p(ws), _p(out), row, rows, columns, _stream(stream)))


def launch_row_gather_tiled_batch(fmt, w, ws, out, host_rows, first_row, rest_rows, count, rows, columns,
                                  stream=None):
    """host_rows: a sequence of ints or None; first_row / rest_rows: device uint32 tensors or None."""
    array = (ctypes.c_uint32 * count)(*host_rows) if host_rows is not None else None
    host = ctypes.cast(array, ctypes.c_void_p) if array is not None else None
    check(lib().gfxinfer_launch_lowbit_row_gather_tiled_batch(fmt, _p(w), _p(ws), _p(out), host, _p(first_row),
                                                              _p(rest_rows), count, rows, columns,
                                                              _stream(stream)))


def launch_row_gather_tiled_indirect(fmt, w, ws, out, row_ptr, rows, columns, stream=None):
    check(lib().gfxinfer_launch_lowbit_row_gather_tiled_indirect(fmt, _p(w), _p(ws), _p(out), _p(row_ptr), rows, columns, _stream(stream)))


# ---- pages of a K/V cache ------------------------------------------------------

class KvPages(ctypes.Structure):
    """gfxinfer_kv_pages.  `of` describes tensors (fp16 pools, int32 state) and keeps them alive."""
    _fields_ = [("key_pages", P), ("value_pages", P), ("page_table", P), ("lengths", P), ("references", P),
                ("layers", U32), ("page_count", U32), ("page_tokens", U32), ("kv_heads", U32), ("head_size", U32),
                ("sequences", U32), ("table_stride", U32)]
    device = None  # of tensors given to `of`

    @classmethod
    def of(cls, key_pages, value_pages, page_table, lengths, references):
        """key_pages, value_pages [layers, pages, page_tokens, kv_heads, head_size]; page_table
        [sequences, pages per sequence]; lengths [sequences]; references [pages].  All contiguous."""
        tensors = (key_pages, value_pages, page_table, lengths, references)
        layers, pages, page_tokens, kv_heads, head_size = key_pages.shape
        sequences, stride = page_table.shape
        if (tuple(value_pages.shape) != tuple(key_pages.shape) or tuple(lengths.shape) != (sequences,)
                or tuple(references.shape) != (pages,) or not all(t.is_contiguous() for t in tensors)
                or any(t.element_size() != size for t, size in zip(tensors, (2, 2, 4, 4, 4)))
                or any(str(t.dtype) == "torch.bfloat16" for t in tensors) or any(t.is_floating_point() for t in tensors[2:])):
            raise ValueError("K/V pages: fp16 pools of one shape, 32-bit integer state, all contiguous")
        self = cls(*(_p(t) for t in tensors), layers, pages, page_tokens, kv_heads, head_size, sequences, stride)
        self.tensors, self.device = tensors, _device_of(tensors, "K/V pages")
        return self


def _host_ids(values):
    """A host list of uint32 in memory the caller keeps for the call (an array is passed as it is)."""
    return values if isinstance(values, array) and values.typecode == "I" else array("I", values)


def kv_pages_workspace_bytes(pages) -> int:
    return int(lib().gfxinfer_kv_pages_workspace_bytes(ctypes.byref(pages)))


def launch_kv_pages_reset(pages, stream=None):
    check(lib().gfxinfer_launch_kv_pages_reset(ctypes.byref(pages), _launch_stream(pages.device, stream)))


def launch_kv_pages_fork(pages, parent, children, stream=None):
    L, ids = lib(), _host_ids(children)
    at, count = ids.buffer_info()
    check(L.gfxinfer_launch_kv_pages_fork(ctypes.byref(pages), parent, at, count, _launch_stream(pages.device, stream)))


def launch_kv_pages_reserve(pages, sequences, tokens, status, workspace, stream=None):
    """status: a device int32."""
    L, ids, device = lib(), _host_ids(sequences), pages.device
    at, count = ids.buffer_info()
    check(L.gfxinfer_launch_kv_pages_reserve(ctypes.byref(pages), at, count, tokens, _operand(status, _word, 4, device, "status"),
                                             *_scratch(workspace, device), _launch_stream(device, stream)))


def launch_kv_pages_append(pages, layer, key, value, sequences, tokens, stream=None):
    """key fp16, value fp32: [len(sequences), tokens, kv_heads * head_size]."""
    L, ids, device = lib(), _host_ids(sequences), pages.device
    at, count = ids.buffer_info()
    size = 2 * count * tokens * pages.kv_heads * pages.head_size
    check(L.gfxinfer_launch_kv_pages_append(ctypes.byref(pages), layer, _operand(key, _half, size, device, "key"),
                                            _operand(value, _real, 2 * size, device, "value"), at, count, tokens,
                                            _launch_stream(device, stream)))


def launch_kv_pages_advance(pages, sequences, tokens, token_counts=None, stream=None):
    """token_counts: device 32-bit integers, one per listed sequence, or None for `tokens` each."""
    L, ids, device = lib(), _host_ids(sequences), pages.device
    at, count = ids.buffer_info()
    counts = None if token_counts is None else _operand(token_counts, _word, 4 * count, device, "token_counts")
    check(L.gfxinfer_launch_kv_pages_advance(ctypes.byref(pages), at, count, tokens, counts, _launch_stream(device, stream)))


def launch_kv_pages_free(pages, sequences, keep_tokens=None, stream=None):
    L, ids, keep = lib(), _host_ids(sequences), None if keep_tokens is None else _host_ids(keep_tokens)
    if keep is not None and len(keep) != len(ids):
        raise ValueError("one length to keep per sequence")
    at, count = ids.buffer_info()
    check(L.gfxinfer_launch_kv_pages_free(ctypes.byref(pages), at, None if keep is None else keep.buffer_info()[0], count,
                                          _launch_stream(pages.device, stream)))


def launch_kv_pages_copy(pages, sources, destinations, stream=None):
    a, b = _host_ids(sources), _host_ids(destinations)
    if len(a) != len(b):
        raise ValueError("as many destinations as sources")
    check(lib().gfxinfer_launch_kv_pages_copy(ctypes.byref(pages), a.buffer_info()[0], b.buffer_info()[0], len(a),
                                              _launch_stream(pages.device, stream)))


def launch_kv_pages_compact(pages, live_pages, workspace, stream=None):
    """live_pages: a device int32, or None."""
    L, device = lib(), pages.device
    check(L.gfxinfer_launch_kv_pages_compact(ctypes.byref(pages), _operand(live_pages, _word, 4, device, "live_pages"),
                                             *_scratch(workspace, device), _launch_stream(device, stream)))


def kv_pages_attention_workspace_bytes(pages, count, tokens, q_heads, shared_tokens) -> int:
    return int(lib().gfxinfer_kv_pages_attention_workspace_bytes(ctypes.byref(pages), count, tokens, q_heads, shared_tokens))


def launch_kv_pages_gated_attention(pages, layer, query, gate, output, sequences, tokens, q_heads, shared_tokens, workspace,
                                    stream=None):
    """query and output fp16 [len(sequences), tokens, q_heads, head_size]; gate fp32 with rows of 2 head_size, or None."""
    L, ids, device = lib(), _host_ids(sequences), pages.device
    at, count = ids.buffer_info()
    size = 2 * count * tokens * q_heads * pages.head_size
    check(L.gfxinfer_launch_kv_pages_gated_attention(ctypes.byref(pages), layer, _operand(query, _half, size, device, "query"),
                                                     None if gate is None else _operand(gate, _real, 4 * size, device, "gate"),
                                                     _operand(output, _half, size, device, "output"), at, count, tokens, q_heads,
                                                     shared_tokens, *_scratch(workspace, device), _launch_stream(device, stream)))


# ---- prompts in chunks, in a cache that stays within a budget --------------------

class KvWeights(ctypes.Structure):
    """gfxinfer_kv_weights.  `of` describes tensors beside the pages and keeps them alive."""
    _fields_ = [("weight", P), ("position", P), ("dropped", P)]
    device = shape = None  # of tensors given to `of`

    @classmethod
    def of(cls, pages, weight, position, dropped):
        """weight fp32 and position int32 [sequences, table columns * page_tokens]; dropped int32 [sequences]."""
        tensors, shape = (weight, position, dropped), (pages.sequences, pages.table_stride * pages.page_tokens)
        if (tuple(weight.shape) != shape or tuple(position.shape) != shape or tuple(dropped.shape) != shape[:1]
                or not all(t.is_contiguous() and t.element_size() == 4 for t in tensors) or not weight.is_floating_point()
                or any(t.is_floating_point() for t in tensors[1:])):
            raise ValueError("K/V weights: contiguous fp32 weight and int32 position for every row of the table, int32 dropped")
        self = cls(*(_p(t) for t in tensors))
        self.tensors, self.shape, self.device = tensors, shape, _device_of(tensors, "K/V weights")
        if pages.device is not None and self.device not in (None, pages.device):
            raise ValueError("K/V weights: tensors of another device than the pages")
        return self


def _weights_of(weights, pages):
    """The address of weights that fit the pages: those of another cache have other rows."""
    if weights.shape not in (None, (pages.sequences, pages.table_stride * pages.page_tokens)):
        raise ValueError("K/V weights: made for pages with other sequences or another table")
    if None not in (weights.device, pages.device) and weights.device != pages.device:
        raise ValueError("K/V weights: tensors of another device than the pages")
    return ctypes.byref(weights)


def _chunk_lists(sequences, tokens):
    """Host lists of a chunk call, their addresses, the number of sequences and of rows."""
    ids, counts = _host_ids(sequences), _host_ids(tokens)
    if len(ids) != len(counts):
        raise ValueError("one number of tokens per sequence")
    at, count = ids.buffer_info()
    return ids, counts, at, counts.buffer_info()[0], count, sum(counts)


def kv_pages_chunk_attention_workspace_bytes(pages, tokens, q_heads) -> int:
    counts = _host_ids(tokens)
    return int(lib().gfxinfer_kv_pages_chunk_attention_workspace_bytes(ctypes.byref(pages), *counts.buffer_info(), q_heads))


def launch_kv_pages_chunk_attention(pages, layer, query, gate, output, log_sums, sequences, tokens, q_heads, workspace, stream=None):
    """tokens: host list, new tokens of each sequence.  query and output fp16 [rows, q_heads, head_size], gate fp32 with rows
    of 2 head_size or None, log_sums fp32 [rows, q_heads] or None; rows = sum(tokens)."""
    L, device = lib(), pages.device
    _ids, _counts, at, tokens_at, count, rows = _chunk_lists(sequences, tokens)
    size = 2 * rows * q_heads * pages.head_size
    check(L.gfxinfer_launch_kv_pages_chunk_attention(
        ctypes.byref(pages), layer, _operand(query, _half, size, device, "query"),
        None if gate is None else _operand(gate, _real, 4 * size, device, "gate"), _operand(output, _half, size, device, "output"),
        None if log_sums is None else _operand(log_sums, _real, 4 * rows * q_heads, device, "log_sums"), at, tokens_at, count,
        q_heads, *_scratch(workspace, device), _launch_stream(device, stream)))


def launch_kv_weights_begin(pages, weights, sequences, tokens, stream=None):
    L = lib()
    _ids, _counts, at, tokens_at, count, _ = _chunk_lists(sequences, tokens)
    check(L.gfxinfer_launch_kv_weights_begin(ctypes.byref(pages), _weights_of(weights, pages), at, tokens_at, count,
                                             _launch_stream(pages.device, stream)))


def kv_weights_workspace_bytes(pages, tokens, q_heads) -> int:
    counts = _host_ids(tokens)
    return int(lib().gfxinfer_kv_weights_workspace_bytes(ctypes.byref(pages), *counts.buffer_info(), q_heads))


def launch_kv_weights_add(pages, weights, layer, query, log_sums, sequences, tokens, q_heads, workspace, stream=None):
    """query and log_sums as of launch_kv_pages_chunk_attention."""
    L, device = lib(), pages.device
    _ids, _counts, at, tokens_at, count, rows = _chunk_lists(sequences, tokens)
    check(L.gfxinfer_launch_kv_weights_add(
        ctypes.byref(pages), _weights_of(weights, pages), layer, _operand(query, _half, 2 * rows * q_heads * pages.head_size, device, "query"),
        _operand(log_sums, _real, 4 * rows * q_heads, device, "log_sums"), at, tokens_at, count, q_heads,
        *_scratch(workspace, device), _launch_stream(device, stream)))


def kv_pages_evict_workspace_bytes(pages, count, budget) -> int:
    return int(lib().gfxinfer_kv_pages_evict_workspace_bytes(ctypes.byref(pages), count, budget))


def launch_kv_pages_evict(pages, weights, sequences, budget, first, recent, status, workspace, stream=None):
    """status: a device int32."""
    L, ids, device = lib(), _host_ids(sequences), pages.device
    at, count = ids.buffer_info()
    check(L.gfxinfer_launch_kv_pages_evict(ctypes.byref(pages), _weights_of(weights, pages), at, count, budget, first, recent,
                                           _operand(status, _word, 4, device, "status"), *_scratch(workspace, device),
                                           _launch_stream(device, stream)))


# ---- products in 8-bit integers, any number of tokens ----------------------------

@functools.cache
def _types():
    import torch
    return {torch.float16: TYPE_F16, torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16}, (torch.int8,)


def launch_quantize_rows_i8(x, codes, scales, stream=None):
    """x [rows, columns], fp16, fp32 or bf16 with dense rows; codes int8 [rows, columns]; scales fp32 [rows]."""
    types, integers = _types()
    rows, columns = x.shape
    L, device, kind = lib(), x.get_device(), types.get(x.dtype)
    if kind is None or x.stride(1) != 1 or device < 0:
        raise ValueError("row quantizer: x is fp16, fp32 or bf16 [rows, columns] on a GPU, with dense rows")
    check(L.gfxinfer_launch_quantize_rows_i8(
        x.data_ptr(), kind, rows, columns, x.stride(0) if rows > 1 else -(-columns // 8) * 8,
        _operand(codes, integers, rows * columns, device, "codes"), _operand(scales, _real, 4 * rows, device, "scales"),
        _launch_stream(device, stream)))


def w8a8_gemm_workspace_bytes(rows, columns, tokens) -> int:
    return int(lib().gfxinfer_w8a8_gemm_workspace_bytes(rows, columns, tokens))


def launch_w8a8_gemm(weights, weight_scales, codes, scales, output, workspace, stream=None):
    """weights int8 [rows, columns], weight_scales fp32 [rows], codes int8 [tokens, columns], scales fp32 [tokens], output fp32
    or fp16 [tokens, rows]; workspace may be None where w8a8_gemm_workspace_bytes is 0."""
    types, integers = _types()
    (rows, columns), tokens, L = weights.shape, codes.shape[0], lib()
    device, kind = weights.get_device(), types.get(output.dtype)
    if device < 0 or codes.shape != (tokens, columns) or output.shape != (tokens, rows) or kind is None or kind == TYPE_BF16:
        raise ValueError("8-bit product: weights [rows, columns] on a GPU, codes [tokens, columns], output fp32 or fp16 [tokens, rows]")
    check(L.gfxinfer_launch_w8a8_gemm(
        _operand(weights, integers, rows * columns, device, "weights"), _operand(weight_scales, _real, 4 * rows, device, "weight_scales"),
        _operand(codes, integers, tokens * columns, device, "codes"), _operand(scales, _real, 4 * tokens, device, "scales"),
        _operand(output, (output.dtype,), tokens * rows * output.element_size(), device, "output"), kind, rows, columns, tokens,
        *_scratch(workspace, device), _launch_stream(device, stream)))


# ---- rules on logits -------------------------------------------------------------

class LogitRules(ctypes.Structure):
    """gfxinfer_logit_rules.  `of` describes tensors and keeps them alive."""
    _fields_ = [(n, P) for n in ("history", "history_rows", "history_lengths", "prompt_lengths", "repetition", "presence",
                                 "frequency", "bias_tokens", "bias_values", "bias_counts", "allowed", "allowed_rows")]
    _fields_ += [(n, U32) for n in ("history_row_count", "history_stride", "bias_stride", "allowed_row_count",
                                    "allowed_stride")]
    device = None  # of tensors given to `of`

    @classmethod
    def of(cls, **tensors):
        """Contiguous 32-bit tensors by the names of the fields: history [rows, tokens], bias_tokens and
        bias_values [batch, entries], allowed [masks, words], the others [batch]."""
        self = cls()
        wide = ("history", "bias_tokens", "bias_values", "allowed")
        real = ("repetition", "presence", "frequency", "bias_values")
        for name, t in tensors.items():
            if name not in dict(cls._fields_[:12]):
                raise TypeError(f"no logit rule is called {name}")
            if t is None:
                continue
            if not t.is_contiguous() or t.element_size() != 4 or t.dim() != (2 if name in wide else 1):
                raise ValueError(f"logit rules: {name} is a contiguous 32-bit {'matrix' if name in wide else 'vector'}")
            if t.is_floating_point() != (name in real):
                raise ValueError(f"logit rules: {name} holds {'fp32 numbers' if name in real else '32-bit integers'}")
            setattr(self, name, _p(t))
        shape = lambda name: tuple(tensors[name].shape) if tensors.get(name) is not None else (0, 0)  # noqa: E731
        if shape("bias_tokens") != shape("bias_values"):
            raise ValueError("logit rules: as many bias values as tokens")
        (self.history_row_count, self.history_stride), self.bias_stride = shape("history"), shape("bias_tokens")[1]
        self.allowed_row_count, self.allowed_stride = shape("allowed")
        vectors = {tuple(t.shape)[0] for n, t in tensors.items() if t is not None and n not in wide}
        vectors |= {shape("bias_tokens")[0]} - {0}
        if len(vectors) > 1:
            raise ValueError("logit rules: one entry per row of the logits")
        self.batch = next(iter(vectors), None)
        self.tensors, self.device = tensors, _device_of([t for t in tensors.values() if t is not None], "logit rules")
        return self


def logit_rules_workspace_bytes(vocabulary, batch) -> int:
    return int(lib().gfxinfer_logit_rules_workspace_bytes(vocabulary, batch))


def launch_logit_rules(logits, rules, output, tokens, workspace, vocabulary=None, stream=None):
    """logits, output: fp32 [batch, columns] (the last dimension dense); output, tokens and workspace may be None."""
    batch, columns = logits.shape
    if rules.batch not in (None, batch):
        raise ValueError("logit rules: made for another number of rows")
    L, device = lib(), logits.get_device()
    if device < 0 and logits.is_pinned():
        device = rules.device
    if rules.device is not None and rules.device != device:
        raise ValueError("logit rules: tensors of another device than the logits")
    vocabulary = columns if vocabulary is None else vocabulary
    for t in (logits,) if output is None else (logits, output):
        if t.stride(1) != 1 or t.dtype not in _real or t.shape[0] != batch or t.shape[1] < vocabulary:
            raise ValueError("logit rules: logits are fp32 [batch, columns] with dense rows that hold the vocabulary")
    if output is not None and output.get_device() != device and not (device is None if output.is_cuda else output.is_pinned()):
        raise ValueError("logit rules: logits and output are on different devices")
    picked = None if tokens is None else _operand(tokens, _word, 4 * batch, device, "logit rules: tokens")
    check(L.gfxinfer_launch_logit_rules(logits.data_ptr(), logits.stride(0), vocabulary, batch, ctypes.byref(rules), _p(output),
                                        0 if output is None else output.stride(0), picked, *_scratch(workspace, device),
                                        _launch_stream(device, stream)))


# ---- host-side layout (numpy) -------------------------------------------------

def packed_row_bytes(fmt: int, columns: int) -> int:
    return int(lib().gfxinfer_packed_row_bytes(fmt, columns))


def tile_bytes(fmt: int, rows: int, columns: int) -> int:
    return rows * columns * {W2G128: 2, W3G128: 3}.get(fmt, 4) // 8


def tile_group128(fmt, packed_codes, scales, rows, columns):
    """Reference-packed codes + float scales -> (tiled codes, fp16 scale bits)."""
    import numpy as np
    packed_codes = np.ascontiguousarray(packed_codes, dtype=np.uint8)
    scales = np.ascontiguousarray(scales, dtype=np.float32)
    codes = np.zeros(tile_bytes(fmt, rows, columns), dtype=np.uint8)
    tscales = np.zeros(rows * (columns // 128), dtype=np.uint16)
    check(lib().gfxinfer_tile_group128_for_gfx950(fmt, _p(packed_codes), _p(scales), rows, columns, _p(codes), _p(tscales)))
    return codes, tscales


def untile_group128(fmt, codes, tscales, rows, columns):
    """Tiled codes (+ fp16 scales) -> (int8 weights [rows, columns], fp16 scale bits [rows, G])."""
    import numpy as np
    codes = np.ascontiguousarray(codes, dtype=np.uint8)
    w = np.empty((rows, columns), dtype=np.int8)
    s = np.empty((rows, columns // 128), dtype=np.uint16)
    ts = None if tscales is None else np.ascontiguousarray(tscales, dtype=np.uint16)
    check(lib().gfxinfer_untile_group128_for_gfx950(fmt, _p(codes), _p(ts), rows, columns, _p(w), _p(s) if ts is not None else None))
    return w, s
