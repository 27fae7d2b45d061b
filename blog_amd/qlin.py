"""ctypes binding of ``blog_amd/libqlin.so`` (the C ABI declared in ``include/qlin.h``).

Plumbing for the tests and the benchmark: device memory comes from torch tensors, every compute
call goes through the C ABI into the HIP kernels.  There is no fallback of any kind: if the
library is missing or a call is rejected, this module raises.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG, "libqlin.so")

Q4_0, Q5_0, Q8_0, Q8_1, Q4_K, Q6_K = 2, 6, 8, 9, 12, 14
STATUS = {0: "QLIN_OK", 1: "QLIN_ERR_UNSUPPORTED_TYPE", 2: "QLIN_ERR_SHAPE", 3: "QLIN_ERR_NULL",
          4: "QLIN_ERR_ROW_BYTES", 5: "QLIN_ERR_LIMIT", 6: "QLIN_ERR_LAUNCH", 7: "QLIN_ERR_ALIGN",
          8: "QLIN_ERR_IO", 9: "QLIN_ERR_FORMAT", 10: "QLIN_ERR_NOT_FOUND", 11: "QLIN_ERR_ALLOC"}

P, I, I64, SZ, F = C.c_void_p, C.c_int, C.c_int64, C.c_size_t, C.c_float
S, U32, U64 = C.c_char_p, C.c_uint32, C.c_uint64
PP, PI, PI64, PU64, PSZ, PD = (C.POINTER(C.c_void_p), C.POINTER(C.c_int), C.POINTER(C.c_int64),
                               C.POINTER(C.c_uint64), C.POINTER(C.c_size_t), C.POINTER(C.c_double))


class GgufTensorInfo(C.Structure):
    """struct qlin_gguf_tensor (include/qlin_gguf.h)."""
    _fields_ = [("name", C.c_char_p), ("type", C.c_int), ("n_dims", C.c_int), ("shape", C.c_int64 * 4),
                ("nbytes", C.c_uint64), ("offset", C.c_uint64), ("data", C.c_void_p)]


class QkRopeArgs(C.Structure):
    """struct qlin_qk_rope (include/qlin_decoder.h)."""
    _fields_ = [("q_norm", P), ("k_norm", P), ("norm_type", I), ("eps", F), ("one_plus", I), ("table", P),
                ("table_len", I), ("rotary_dim", I), ("pairing", I)]


class Kv8CacheArgs(C.Structure):
    """struct qlin_kv8_cache (include/qlin_decoder.h)."""
    _fields_ = [("pages", P), ("recent", P), ("block_table", P), ("n_pages", I), ("n_seqs", I), ("blocks_per_seq", I),
                ("kv_heads", I), ("head_dim", I)]


class LogitsControlsArgs(C.Structure):
    """struct qlin_logits_controls (include/qlin_decoder.h)."""
    _fields_ = [("history", P), ("history_lens", P), ("repetition", P), ("frequency", P), ("presence", P),
                ("bias_ids", P), ("bias_values", P), ("mask", P), ("mask_stride", SZ), ("max_history", I),
                ("max_bias", I)]


class MoeRoutingArgs(C.Structure):
    """struct qlin_moe_routing (include/qlin.h)."""
    _fields_ = [("bias", P), ("sigmoid", I), ("n_groups", I), ("top_groups", I), ("group_pairs", I), ("renormalise", I),
                ("scaling", F)]


class LoraArgs(C.Structure):
    """struct qlin_lora (include/qlin_decoder.h)."""
    _fields_ = [("a", P), ("b", P), ("base", P), ("y", P), ("base_stride", SZ), ("y_stride", SZ), ("out_dim", I)]


# name -> (restype, argtypes); every symbol of include/qlin.h
SIGNATURES = {
    "qlin_status_string": (C.c_char_p, [I]),
    "qlin_version": (C.c_char_p, []),
    "qlin_set_stream": (I, [P]),
    "qlin_get_stream": (P, []),
    "qlin_block_elems": (I, [I]),
    "qlin_block_bytes": (I, [I]),
    "qlin_row_bytes": (SZ, [I, I]),
    "qlin_launch_quant_gemv": (I, [I, P, SZ, P, P, I, I, I]),
    "qlin_launch_quant_gemv_add": (I, [I, P, SZ, P, P, I, I]),
    "qlin_launch_quant_matmul": (I, [I, P, SZ, P, P, I, I, I]),
    "qlin_launch_quant_matmul_add": (I, [I, P, SZ, P, P, I, I, I]),
    "qlin_launch_quant_gemv_q8_1": (I, [I, P, SZ, P, P, I, I]),
    "qlin_launch_moe_accumulate": (I, [P, F, P, I]),
    "qlin_launch_moe_accumulate_device": (I, [P, P, P, I]),
    "qlin_launch_argmax": (I, [P, I, P]),
    "qlin_launch_quantize_q8_1_mmq": (I, [P, P, I, I, I]),
    "qlin_launch_quant_matmul_q8_1_mmq": (I, [I, P, SZ, P, P, I, I, I]),
    "qlin_launch_quant_swiglu_indexed_block": (I, [I, P, P, SZ, SZ, SZ, SZ, P, P, P, I, I, I, I]),
    "qlin_launch_quant_swiglu_indexed_q8_1": (I, [I, P, P, SZ, SZ, SZ, SZ, P, P, P, I, I, I]),
    "qlin_launch_quant_down_q8_1_indexed_accum": (I, [I, P, SZ, SZ, P, P, P, P, I, I, I]),
    "qlin_launch_quant_down_q8_1_indexed_accum_shared": (I, [I, P, SZ, SZ, P, P, P, P, I, I, I]),
    "qlin_launch_quant_down_f32_indexed_accum": (I, [I, P, SZ, SZ, P, P, P, P, I, I, I]),
    "qlin_launch_quant_swiglu_rows": (I, [I, P, P, SZ, SZ, P, P, I, I, I]),
    "qlin_launch_quant_gemv_multi": (I, [I, I, P, SZ, P, P, P, I]),
    "qlin_q8_1_row_bytes": (SZ, [I]),
    "qlin_launch_quantize_q8_1": (I, [P, P, I, I, I]),
    "qlin_launch_quant_matmul_q8_1": (I, [I, P, SZ, P, P, I, I, I]),
    "qlin_launch_quant_swiglu": (I, [I, P, P, SZ, SZ, P, P, I, I]),
    "qlin_launch_quant_swiglu_indexed": (I, [I, P, P, SZ, SZ, SZ, SZ, P, P, P, I, I, I]),
    "qlin_launch_quant_down_f32_indexed_accum_ordered": (I, [I, P, SZ, SZ, P, P, P, P, I, I, I]),
    "qlin_launch_moe_router_topk": (I, [P, P, P, I, I, I, F]),
    "qlin_launch_moe_route": (I, [P, P, SZ, P, P, I, I, I]),
    "qlin_launch_dequantize_q8_1": (I, [P, P, I, I, I]),
    "qlin_launch_dequantize_to_f16": (I, [I, P, P, I64]),
    "qlin_launch_dequantize_q4k_to_f16": (I, [P, P, I64]),
    "qlin_launch_dequantize_q80_to_f16": (I, [P, P, I64]),
    "qlin_launch_dequantize_q50_to_f16": (I, [P, P, I64]),
    "qlin_launch_dequantize_q6k_to_f16": (I, [P, P, I64]),
    "qlin_launch_dequantize_to_f32": (I, [I, P, P, I64]),
    "qlin_gemm": (I, [I, P, SZ, P, P, I, I, I]),
    "qlin_moe_routed_decode_indexed": (I, [I, P, P, SZ, I, P, SZ, I, I, I, I, P, P, P, P, P, I]),
    "qlin_moe_routed_decode_indexed_logits": (I, [I, P, P, SZ, I, P, SZ, I, I, I, I, P, P, F, P, P, P, P, I]),
    "qlin_moe_ffn_decode_indexed_logits": (I, [I, P, P, SZ, I, P, SZ, I, I, I, I, I, P, P, SZ, P, SZ, I, P, P, F, P, P,
                                               P, P, I]),
    "qlin_moe_grouped_workspace_bytes": (SZ, [I, I, I, I, I]),
    "qlin_moe_routed_decode_grouped": (I, [I, P, P, SZ, I, P, SZ, I, I, I, I, P, P, P, P, SZ, P, I, I]),
    "qlin_moe_routed_decode_grouped_logits": (I, [I, P, P, SZ, I, P, SZ, I, I, I, I, P, P, F, P, P, P, SZ, P, I, I]),
    "qlin_moe_ffn_workspace_bytes": (SZ, [I, I, I, I, I, I]),
    "qlin_moe_ffn_decode_grouped_logits": (I, [I, P, P, SZ, I, P, SZ, I, I, I, I, I, P, P, SZ, P, SZ, I, P, P, F, P, P,
                                               P, SZ, P, I, I]),
    "qlin_moe_routed_decode_grouped_noalloc": (I, [I, P, P, SZ, I, P, SZ, I, I, I, I, P, P, P, P, I, I]),
    # include/qlin_decoder.h
    "qlin_launch_rms_norm": (I, [P, P, P, I, I, I, F, I]),
    "qlin_launch_rope_store_kv": (I, [P, P, P, P, P, I, I, I, I, I, P, F]),
    "qlin_launch_attend": (I, [P, P, P, P, I, I, I, I, I, P]),
    "qlin_launch_rope_attend": (I, [P, P, P, P, P, P, I, I, I, I, P, F]),
    "qlin_launch_rms_norm_quant_gemv_multi": (I, [I, I, P, SZ, P, P, I, F, I, P, P, I]),
    "qlin_launch_rms_norm_quant_swiglu": (I, [I, P, P, SZ, P, P, I, F, I, P, I, I]),
    "qlin_launch_quant_gemv_argmax": (I, [I, P, SZ, P, P, I, F, I, P, I, I, P, P]),
    "qlin_launch_rope_table": (I, [P, I, I, F]),
    "qlin_launch_qk_norm_rope_store_kv": (I, [P, P, SZ, P, SZ, P, SZ, P, P, P, I, I, I, I, I, P]),
    "qlin_launch_qk_norm_rope_store_kv8": (I, [P, P, P, SZ, P, SZ, P, SZ, P, I, I, P, P]),
    "qlin_launch_kv8_read": (I, [P, P, P, I, P, P]),
    "qlin_attend_kv8_workspace_bytes": (SZ, [I, I, I, I, I, I]),
    "qlin_launch_attend_kv8": (I, [P, P, P, I, I, P, P, F, P, SZ]),
    "qlin_logits_controls_scratch_bytes": (SZ, [I, I]),
    "qlin_launch_logits_controls": (I, [P, P, SZ, P, SZ, I, I, P, P, SZ]),
    "qlin_launch_add_rms_norm": (I, [P, SZ, P, SZ, P, SZ, P, I, F, I, P, SZ, P, I, I, I, I]),
    "qlin_lora_workspace_bytes": (SZ, [I, I, I, I, I]),
    "qlin_launch_lora_add": (I, [P, I, I, I, I, I, P, P, P, SZ, P, I, P, SZ]),
    "qlin_verify_drafts_workspace_bytes": (SZ, [I, I, I]),
    "qlin_launch_verify_drafts": (I, [P, SZ, P, SZ, P, P, P, P, P, P, P, P, I, I, I, P, SZ]),
    "qlin_launch_quant_embedding": (I, [I, P, P, P, SZ, I, I]),
    "qlin_launch_mla_absorb_q_nope": (I, [I, P, P, SZ, P, I, I, I, I, I]),
    "qlin_launch_mla_absorb_q4_xsum_delta": (I, [P, P, SZ, P, I, I, I, I, I]),
    "qlin_launch_mla_absorb_v": (I, [I, P, SZ, P, P, P, I, I, I, I]),
    "qlin_launch_mla_store_latent_q8_1_device_pos": (I, [P, P, I, I, SZ, P]),
    "qlin_launch_mla_absorb_scores_device_pos": (I, [P, P, P, SZ, P, P, P, I, I, I, I, P, I, F]),
    "qlin_launch_mla_absorb_context_device_pos": (I, [P, P, SZ, P, P, I, I, P, I]),
    "qlin_launch_mla_absorb_attend_device_pos": (I, [P, P, P, SZ, P, P, P, P, I, I, I, I, P, I, F]),
    "qlin_launch_mla_project_v_device_pos": (I, [I, P, SZ, P, SZ, P, I, I, I, I, P]),
    "qlin_launch_mla_absorb_context_v_device_pos": (I, [P, P, P, I, I, I, P, I]),
    # include/qlin_gguf.h
    "qlin_gguf_open": (I, [S, PP]),
    "qlin_gguf_close": (None, [P]),
    "qlin_gguf_version": (U32, [P]),
    "qlin_gguf_alignment": (U32, [P]),
    "qlin_gguf_tensor_count": (I64, [P]),
    "qlin_gguf_find_tensor": (I64, [P, S]),
    "qlin_gguf_tensor_info": (I, [P, I64, C.POINTER(GgufTensorInfo)]),
    "qlin_gguf_metadata_count": (I64, [P]),
    "qlin_gguf_metadata_key": (S, [P, I64]),
    "qlin_gguf_metadata_type": (I, [P, S]),
    "qlin_gguf_get_i64": (I, [P, S, PI64]),
    "qlin_gguf_get_f64": (I, [P, S, PD]),
    "qlin_gguf_get_str": (I, [P, S, PP, PSZ]),
    "qlin_gguf_get_array_info": (I, [P, S, PI, PI64]),
    "qlin_gguf_get_array_i64": (I, [P, S, I64, PI64]),
    "qlin_gguf_get_array_f64": (I, [P, S, I64, PD]),
    "qlin_gguf_get_array_str": (I, [P, S, I64, PP, PSZ]),
    "qlin_pool_create": (I, [PP]),
    "qlin_pool_destroy": (None, [P]),
    "qlin_pool_weight": (I, [P, P, S, PP, PU64]),
    "qlin_pool_expert_view": (I, [P, P, S, I, PP, PU64, PI64, PI64]),
    "qlin_pool_resident_bytes": (U64, [P]),
}


class QlinError(RuntimeError):
    def __init__(self, fn: str, rc: int):
        super().__init__(f"{fn} returned {rc} ({STATUS.get(rc, '?')})")
        self.rc = rc


_lib = None
_F32 = _I32 = _U32 = _U8 = None  # torch's types
_BF16 = _F16 = None
_LORA_TYPES = {}
_current_device = None


def lib() -> C.CDLL:
    """Loads the HIP library; raises if it has not been built (no fallback path exists)."""
    global _lib, _F32, _I32, _U32, _U8, _BF16, _F16, _LORA_TYPES, _current_device
    if _lib is None:
        # torch ships its own HIP runtime (torch/lib/libamdhip64.so, soname libamdhip64.so.7).  Loaded
        # first, it satisfies this library's libamdhip64.so.7 dependency, so the process has one HIP
        # runtime; loaded after, it would bring a second one next to /opt/rocm's, and device memory of
        # one is unusable from the other.
        try:
            import torch
            _F32, _I32, _U32, _U8 = torch.float32, torch.int32, torch.uint32, torch.uint8
            _LORA_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
            _BF16, _F16 = torch.bfloat16, torch.float16
            # (what torch.cuda.current_device calls after its own look at whether the GPU has been met; a tensor there has)
            _current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        except ImportError:
            pass
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: run `python -m blog_amd.build` (HIP/gfx950 build)")
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
    return _lib


def ptr(t) -> int:
    """Device address of a torch tensor (or an int address, or None -> 0)."""
    if t is None:
        return 0
    if isinstance(t, int):
        return t
    return t.data_ptr()


def call(name: str, *args) -> int:
    """Calls an entry point with tensors converted to addresses; raises on a non-zero status."""
    rc = getattr(lib(), name)(*[ptr(a) if not isinstance(a, (float, bool)) and hasattr(a, "data_ptr") else a
                                for a in args])
    if rc != 0:
        raise QlinError(name, rc)
    return rc


def status(name: str, *args) -> int:
    """Calls an entry point and returns its status without raising."""
    return getattr(lib(), name)(*[ptr(a) if hasattr(a, "data_ptr") else a for a in args])


def set_stream(stream) -> None:
    """Launch on a torch.cuda.Stream (or a raw hipStream_t address, or None)."""
    handle = 0 if stream is None else (stream if isinstance(stream, int) else stream.cuda_stream)
    lib().qlin_set_stream(handle or None)


def row_bytes(qtype: int, in_dim: int) -> int:
    return int(lib().qlin_row_bytes(qtype, in_dim))


# ---- convenience wrappers (tensors in, launches on the current library stream) --------------

def quant_gemv(qtype, w, rb, x, y, out_dim, in_dim, m=1):
    call("qlin_launch_quant_gemv", qtype, w, rb, x, y, out_dim, in_dim, m)


def quant_gemv_add(qtype, w, rb, x, y, out_dim, in_dim):
    call("qlin_launch_quant_gemv_add", qtype, w, rb, x, y, out_dim, in_dim)


def quant_gemv_multi(qtype, ws, rb, x, ys, out_dims, in_dim):
    """Several GEMVs sharing x in one launch (lists of tensors / device addresses)."""
    n = len(ws)
    wa = (C.c_void_p * n)(*[ptr(w) for w in ws])
    ya = (C.c_void_p * n)(*[ptr(y) for y in ys])
    da = (C.c_int * n)(*out_dims)
    call("qlin_launch_quant_gemv_multi", qtype, n, C.addressof(wa), rb, x, C.addressof(ya), C.addressof(da), in_dim)


def rms_norm_quant_gemv_multi(qtype, ws, rb, x, norm_w, norm_type, eps, one_plus, ys, out_dims, in_dim):
    """quant_gemv_multi of rms_norm(x), in one launch (lists of tensors / device addresses)."""
    n = len(ws)
    wa = (C.c_void_p * n)(*[ptr(w) for w in ws])
    ya = (C.c_void_p * n)(*[ptr(y) for y in ys])
    da = (C.c_int * n)(*out_dims)
    call("qlin_launch_rms_norm_quant_gemv_multi", qtype, n, C.addressof(wa), rb, x, norm_w, norm_type, eps, one_plus,
         C.addressof(ya), C.addressof(da), in_dim)


def quant_swiglu(qtype, wg, wu, g_rb, u_rb, x, act, ffn_dim, in_dim):
    call("qlin_launch_quant_swiglu", qtype, wg, wu, g_rb, u_rb, x, act, ffn_dim, in_dim)


def quant_matmul(qtype, w, rb, x, y, out_dim, in_dim, m):
    call("qlin_launch_quant_matmul", qtype, w, rb, x, y, out_dim, in_dim, m)


def quant_matmul_add(qtype, w, rb, x, y, out_dim, in_dim, m):
    call("qlin_launch_quant_matmul_add", qtype, w, rb, x, y, out_dim, in_dim, m)


def quant_swiglu_rows(qtype, wg, wu, g_rb, u_rb, x, act, ffn_dim, in_dim, m):
    call("qlin_launch_quant_swiglu_rows", qtype, wg, wu, g_rb, u_rb, x, act, ffn_dim, in_dim, m)


def quantize_q8_1(x, xq, in_dim, m, store_raw_sum=False):
    call("qlin_launch_quantize_q8_1", x, xq, in_dim, m, int(store_raw_sum))


def quant_matmul_q8_1(qtype, w, rb, xq, y, out_dim, in_dim, m):
    call("qlin_launch_quant_matmul_q8_1", qtype, w, rb, xq, y, out_dim, in_dim, m)


def dequantize(qtype, src, out, n, f16=True):
    if f16:
        call("qlin_launch_dequantize_to_f16", qtype, src, out, n)
    else:
        call("qlin_launch_dequantize_to_f32", qtype, src, out, n)


# ---- head norms with the rotation, the 8-bit attention cache, controls on logits (qlin_decoder.h) ---

KV8_BLOCK, KV8_RECENT = 32, 64
MAX_BIAS = 4096  # biases of a row of logits


# (call() looks at every argument twice: 2 to 4 us of a launch of 5)
def _at(t):
    return t if t is None or t.__class__ is int else t.data_ptr()


def _done(name, rc):
    if rc != 0:
        raise QlinError(name, rc)


def kv8_record_bytes(head_dim):
    """Bytes of one block of one key head in a page."""
    return 64 * head_dim + 16


def rope_table(table, theta):
    """Fills table ([n_pos, rotary_dim] f32) with the cosines and sines of every position."""
    if table.element_size() != 4 or not table.is_contiguous():
        raise ValueError("the table is contiguous f32")
    call("qlin_launch_rope_table", table, table.shape[0], table.shape[1], theta)


class QkRope:
    """How heads are normed and rotated (struct qlin_qk_rope): norm weights (bf16 or f16 bits, or None) and the
    rotation table [positions, rotary_dim] (None: no rotation).  Holds on to the tensors."""

    def __init__(self, q_norm, k_norm, norm_type, eps, one_plus, table, rotary_dim, pairing=0):
        if table is not None and (table.element_size() != 4 or not table.is_contiguous() or table.shape[1] != rotary_dim):
            raise ValueError(f"a table {tuple(table.shape)} of {table.dtype} for rotary_dim {rotary_dim}: contiguous f32 rows of it")
        self.norm_dims = 1 << 30  # of the shorter weights, as far as they are known
        for w in (q_norm, k_norm):
            if hasattr(w, "data_ptr"):
                if w.element_size() != 2 or not w.is_contiguous():
                    raise ValueError("norm weights are contiguous and of 16 bits")
                self.norm_dims = min(self.norm_dims, w.numel())
        self.tensors = (q_norm, k_norm, table)
        self.args = QkRopeArgs(ptr(q_norm), ptr(k_norm), norm_type, eps, int(one_plus), ptr(table),
                               table.shape[0] if table is not None else 0, rotary_dim, pairing)
        self.address = C.addressof(self.args)


def _of_sequences(t, n, name):
    """The address of positions or counts, int32, one for each of n sequences (or an address, or None, as it is)."""
    if t is None or t.__class__ is int:
        return t
    if t.dtype is not _I32 or n > 1 and (t.numel() < n or not t.is_contiguous()) or not (at := t.data_ptr()) and n:
        raise ValueError(f"{name}: {tuple(t.shape)} of {t.dtype}, not {n} contiguous values of int32")
    return at


def _short_norms(how, head_dim):
    return ValueError(f"norm weights of {how.norm_dims} values for heads of {head_dim}")


class Kv8Cache:
    """One layer's 8-bit cache (struct qlin_kv8_cache): pages [n_pages, kv_heads, kv8_record_bytes(head_dim)] uint8,
    recent [n_seqs, kv_heads, 2, 64, head_dim] f32, and the block table [n_seqs, blocks_per_seq] int32, or None with
    blocks_per_seq given.  Holds on to the tensors."""

    def __init__(self, pages, recent, block_table=None, blocks_per_seq=0):
        n_seqs, kv_heads, _, ring, head_dim = recent.shape
        if ring != KV8_RECENT or tuple(pages.shape[1:]) != (kv_heads, kv8_record_bytes(head_dim)):
            raise ValueError(f"pages {tuple(pages.shape)} and recent {tuple(recent.shape)} are not one cache's")
        for name, t, size in (("pages", pages, 1), ("recent", recent, 4), ("block_table", block_table, 4)):
            if t is not None and not t.is_contiguous():
                raise ValueError(f"{name} is not contiguous")
            if t is not None and t.element_size() != size:
                raise ValueError(f"{name} has elements of {t.element_size()} bytes, not of {size}")
        if block_table is not None:
            if block_table.shape[0] != n_seqs:
                raise ValueError(f"a block table of {block_table.shape[0]} sequences for {n_seqs}")
            blocks_per_seq = block_table.shape[1]
        self.pages, self.recent, self.block_table = pages, recent, block_table
        self.n_seqs, self.kv_heads, self.head_dim, self.blocks_per_seq = n_seqs, kv_heads, head_dim, blocks_per_seq
        self.args = Kv8CacheArgs(ptr(pages), ptr(recent), ptr(block_table), pages.shape[0], n_seqs, blocks_per_seq,
                                 kv_heads, head_dim)
        self.address = C.addressof(self.args)

    @classmethod
    def empty(cls, torch, n_seqs, kv_heads, head_dim, max_seq, device="cuda"):
        """A cache of max_seq positions (in whole blocks) for each sequence, its pages in order."""
        blocks = (max_seq + KV8_BLOCK - 1) // KV8_BLOCK
        pages = torch.zeros(n_seqs * blocks, kv_heads, kv8_record_bytes(head_dim), dtype=torch.uint8, device=device)
        recent = torch.zeros(n_seqs, kv_heads, 2, KV8_RECENT, head_dim, device=device)
        return cls(pages, recent, None, blocks)


def qk_norm_rope_store_kv(how, q, q_stride, k, k_stride, v, v_stride, q_out, kc, vc, rows, n_heads, kv_heads, head_dim,
                          max_seq, start_pos):
    if how.norm_dims < head_dim:
        raise _short_norms(how, head_dim)
    library = _lib or lib()
    _done("qlin_launch_qk_norm_rope_store_kv", library.qlin_launch_qk_norm_rope_store_kv(
        how.address, _at(q), q_stride, _at(k), k_stride, _at(v), v_stride, _at(q_out), _at(kc), _at(vc), rows, n_heads,
        kv_heads, head_dim, max_seq, _of_sequences(start_pos, 1, "start_pos")))


def qk_norm_rope_store_kv8(how, cache, q, q_stride, k, k_stride, v, v_stride, q_out, rows, n_heads, start_pos,
                           n_rows=None):
    if how.norm_dims < cache.head_dim:
        raise _short_norms(how, cache.head_dim)
    library, n = _lib or lib(), cache.n_seqs
    _done("qlin_launch_qk_norm_rope_store_kv8", library.qlin_launch_qk_norm_rope_store_kv8(
        how.address, cache.address, _at(q), q_stride, _at(k), k_stride, _at(v), v_stride, _at(q_out), rows, n_heads,
        _of_sequences(start_pos, n, "start_pos"), _of_sequences(n_rows, n, "n_rows")))


def kv8_read(cache, first, lens, count, k_out, v_out):
    library, n = _lib or lib(), cache.n_seqs
    _done("qlin_launch_kv8_read", library.qlin_launch_kv8_read(
        cache.address, _of_sequences(first, n, "first"), _of_sequences(lens, n, "lens"), count, _at(k_out), _at(v_out)))


def attend_kv8_workspace_bytes(n_seqs, rows, n_heads, kv_heads, head_dim, blocks_per_seq):
    return int(lib().qlin_attend_kv8_workspace_bytes(n_seqs, rows, n_heads, kv_heads, head_dim, blocks_per_seq))


def attend_kv8(cache, q, attn, rows, n_heads, start_pos, n_rows, softmax_scale, workspace):
    """workspace: a uint8 tensor of at least attend_kv8_workspace_bytes(...) (None where that is 0)."""
    library, n = _lib or lib(), cache.n_seqs
    _done("qlin_launch_attend_kv8", library.qlin_launch_attend_kv8(
        cache.address, _at(q), _at(attn), rows, n_heads, _of_sequences(start_pos, n, "start_pos"),
        _of_sequences(n_rows, n, "n_rows"), softmax_scale, _at(workspace), 0 if workspace is None else workspace.numel()))


def _wrong(name, t, dtype, rows):
    return ValueError(f"{name}: {tuple(t.shape)} of {t.dtype}, not {rows} contiguous values of {dtype}")


# struct qlin_logits_controls, packed (filling a ctypes structure takes 0.4 us longer)
_LOGITS_CONTROLS = struct.Struct("@8PNii")
assert _LOGITS_CONTROLS.size == C.sizeof(LogitsControlsArgs)


def logits_controls_scratch_bytes(rows, vocab):
    return int(lib().qlin_logits_controls_scratch_bytes(rows, vocab))


def logits_controls(logits, out, rows, vocab, *, history=None, history_lens=None, repetition=None, frequency=None,
                    presence=None, bias_ids=None, bias_values=None, mask=None, picks=None, scratch=None):
    """Penalties, biases and a mask on logits [rows, >= vocab] into out (which may be logits), and the greedy picks.
    history [rows, max_history], bias_ids / bias_values [rows, max_bias] and mask [rows, words] (32 tokens a word) are
    2-D and contiguous, with at least `rows` rows; history_lens, repetition, frequency, presence and picks hold a value for
    each row.  Token ids, lengths and picks are int32, the mask int32 or uint32, the rest float32.  scratch: a uint8 tensor of
    logits_controls_scratch_bytes(...), needed with picks."""
    library = _lib or lib()
    f32, i32 = _F32, _I32
    # (strides and sizes as whole tuples: stride(0) or size(1) take 0.15 us longer each)
    n, width = logits.shape
    out_n, out_width = out.shape
    row, out_row = width, out_width
    if not (logits.is_contiguous() and out.is_contiguous()):
        row, one = logits.stride()
        out_row, out_one = out.stride()
        if not one == out_one == 1 and vocab > 1:
            raise ValueError("a row of logits is contiguous")
    if n < rows or width < vocab or out_n < rows or out_width < vocab or logits.dtype is not f32 or out.dtype is not f32:
        raise ValueError(f"{tuple(logits.shape)} logits of {logits.dtype} into {tuple(out.shape)} of {out.dtype}: "
                         f"float32 [>= {rows}, >= {vocab}] both")
    words = max_history = max_bias = p_mask = p_history = p_ids = p_values = 0
    if mask is not None:
        n, words = mask.shape
        if n < rows or mask.dtype is not i32 and mask.dtype is not _U32 or not mask.is_contiguous():
            raise ValueError(f"the mask: {tuple(mask.shape)} of {mask.dtype}, not contiguous int32 or uint32 [{rows}, words]")
        p_mask = mask.data_ptr()
    if history is not None:
        n, max_history = history.shape
        if n < rows or history.dtype is not i32 or not history.is_contiguous():
            raise ValueError(f"the history: {tuple(history.shape)} of {history.dtype}, not contiguous int32 [{rows}, tokens]")
        p_history = history.data_ptr()
    if bias_ids is not None:
        shape = bias_ids.shape
        n, max_bias = shape
        if n < rows or bias_ids.dtype is not i32 or not bias_ids.is_contiguous() or bias_values is not None and (
                bias_values.dtype is not f32 or not bias_values.is_contiguous() or bias_values.shape != shape):
            raise ValueError(f"biases: int32 tokens and float32 values of one shape [{rows}, entries], contiguous")
        p_ids = bias_ids.data_ptr()
        p_values = 0 if bias_values is None else bias_values.data_ptr()
    # (what has a value for each row, written out: a function's call for each takes 0.3 us more.  An address stands for
    # itself; a tensor without values has none)
    p_lens = p_repetition = p_frequency = p_presence = p_picks = 0
    if history_lens is not None:
        if history_lens.__class__ is int:
            p_lens = history_lens
        elif history_lens.dtype is not i32 or not (p_lens := history_lens.data_ptr()) and rows or rows > 1 and (
                history_lens.numel() < rows or not history_lens.is_contiguous()):
            raise _wrong("history_lens", history_lens, i32, rows)
    if repetition is not None:
        if repetition.__class__ is int:
            p_repetition = repetition
        elif repetition.dtype is not f32 or not (p_repetition := repetition.data_ptr()) and rows or rows > 1 and (
                repetition.numel() < rows or not repetition.is_contiguous()):
            raise _wrong("repetition", repetition, f32, rows)
    if frequency is not None:
        if frequency.__class__ is int:
            p_frequency = frequency
        elif frequency.dtype is not f32 or not (p_frequency := frequency.data_ptr()) and rows or rows > 1 and (
                frequency.numel() < rows or not frequency.is_contiguous()):
            raise _wrong("frequency", frequency, f32, rows)
    if presence is not None:
        if presence.__class__ is int:
            p_presence = presence
        elif presence.dtype is not f32 or not (p_presence := presence.data_ptr()) and rows or rows > 1 and (
                presence.numel() < rows or not presence.is_contiguous()):
            raise _wrong("presence", presence, f32, rows)
    if picks is not None:
        if picks.__class__ is int:
            p_picks = picks
        elif picks.dtype is not i32 or not (p_picks := picks.data_ptr()) and rows or rows > 1 and (
                picks.numel() < rows or not picks.is_contiguous()):
            raise _wrong("picks", picks, i32, rows)
    a = _LOGITS_CONTROLS.pack(p_history, p_lens, p_repetition, p_frequency, p_presence, p_ids, p_values, p_mask, words,
                              max_history, max_bias)
    p_scratch = scratch_bytes = 0
    if scratch is not None:
        p_scratch, scratch_bytes = scratch.data_ptr(), scratch.numel()
    rc = library.qlin_launch_logits_controls(a, logits.data_ptr(), row, out.data_ptr(), out_row, rows, vocab, p_picks, p_scratch,
                                             scratch_bytes)
    if rc != 0:
        raise QlinError("qlin_launch_logits_controls", rc)


# ---- a server's step around the linears: norms with the residual's addition, adapters, routing, drafts -------
#
# These take tensors of one GPU (the current device's, whose stream set_stream was given) and refuse others, and types,
# shapes and layouts that would be read as something else.

# (A launch takes about 2 us of the host, looking at a tensor from all sides as much again: the usual layouts are told by few
# looks, and what one function would do for all tensors is written out where there are many.)

def _rows_of(t, shape, name, device):
    """The address and the row stride of t: f32 of at least shape whose rows are contiguous."""
    if t.shape == shape and t.is_contiguous() and t.dtype is _F32 and t.get_device() == device:
        return t.data_ptr(), shape[1]
    rows, width = shape
    n, have = t.shape
    row, one = t.stride()
    if t.dtype is not _F32 or n < rows or have < width or one != 1 and width > 1 or t.get_device() != device:
        raise ValueError(f"{name}: {tuple(t.shape)} of {t.dtype} on {t.device}, not float32 [{rows}, {width}] with contiguous rows "
                         f"on device {device}")
    return t.data_ptr(), row if n > 1 else max(row, width)


def _values_of(t, n, dtype, name, device):
    """The address of n values of dtype, one for each row or adapter: contiguous, alone or the first ones of a longer line."""
    have = t.numel()
    if t.dtype is not dtype or have != n and (have < n or t.dim() > 1 and t.shape[-1] != 1) or not t.is_contiguous() or t.get_device() != device:
        raise _not(t, f"{n} contiguous values of {dtype}", name, device)
    return t.data_ptr()


def _table_of(t, n, width, dtype, name, device):
    """The address of n rows of width values of dtype that stand one after the other: [>= n, width] (or a flat buffer of them)."""
    shape = t.shape
    if t.dtype is not dtype or shape != (n, width) and (t.numel() < n * width or n > 1 and width and len(shape) > 1 and shape[-1] != width) or (
            not t.is_contiguous() or t.get_device() != device):
        raise _not(t, f"contiguous {dtype} [{n}, {width}]", name, device)
    return t.data_ptr()


def _bytes_of(t, n, name, device):
    """The address of at least n bytes, in whatever shape."""
    if t.dtype is not _U8 or t.numel() < n or not t.is_contiguous() or t.get_device() != device:
        raise _not(t, f"{n} contiguous bytes (uint8)", name, device)
    return t.data_ptr()


def _not(t, what, name, device):
    return ValueError(f"{name}: {tuple(t.shape)} of {t.dtype} on {t.device}, not {what} on device {device}")


def _device_of(t, name):
    device = t.get_device()
    if device < 0:
        raise ValueError(f"{name} is on {t.device}, not on a GPU")
    if device != _current_device():  # (a launch goes to the current device)
        raise ValueError(f"{name} is on {t.device}, not on the current device {_current_device()}")
    return device


def q8_1_bytes(in_dim, rows, mmq=False):
    """Bytes of rows rows of in_dim values in Q8_1 blocks."""
    return (in_dim + 127) // 128 * rows * 144 if mmq else rows * ((in_dim + 31) // 32) * 36


def add_rms_norm(x, delta, sum, weight, norm_type, eps, one_plus, *, normed=None, q8_1=None, mmq=False, raw_sum=False):
    """sum = x + delta, and its RMSNorm into normed [rows, hidden], into Q8_1 blocks (uint8), or both.  x, delta, sum and normed
    are float32 [rows, hidden] with contiguous rows; delta and sum may be None, sum may be x or delta."""
    library, device, shape = _lib or lib(), _device_of(x, "x"), x.shape
    rows, hidden = shape
    p_x, n_x = (x.data_ptr(), hidden) if x.dtype is _F32 and x.is_contiguous() else _rows_of(x, shape, "x", device)
    p_delta, n_delta = (0, 0) if delta is None else _rows_of(delta, shape, "delta", device)
    p_sum, n_sum = (0, 0) if sum is None else _rows_of(sum, shape, "sum", device)
    p_normed, n_normed = (0, 0) if normed is None else _rows_of(normed, shape, "normed", device)
    if weight.element_size() != 2 or weight.numel() != hidden and (weight.numel() < hidden or weight.dim() > 1) or not weight.is_contiguous() or (
            weight.get_device() != device):
        raise ValueError(f"weight: {tuple(weight.shape)} of {weight.dtype} on {weight.device}, not {hidden} contiguous values of 16 bits")
    if weight.dtype is (_BF16 if norm_type else _F16):  # (whole numbers are patterns of either type)
        raise ValueError(f"weight: {weight.dtype} with norm_type {norm_type} (0 bfloat16, 1 float16)")
    p_q8 = 0 if q8_1 is None else _bytes_of(q8_1, q8_1_bytes(hidden, rows, mmq), "q8_1", device)
    rc = library.qlin_launch_add_rms_norm(p_x, n_x, p_delta, n_delta, p_sum, n_sum, weight.data_ptr(), norm_type, eps, int(one_plus),
                                          p_normed, n_normed, p_q8, int(mmq), int(raw_sum), rows, hidden)
    if rc != 0:
        raise QlinError("qlin_launch_add_rms_norm", rc)


def dequantize_q8_1(x_q8_1, x, in_dim, m, mmq=False):
    """The values that m rows of Q8_1 blocks (uint8) stand for, into x (float32 [m, in_dim], contiguous)."""
    library, device = _lib or lib(), _device_of(x, "x")
    rc = library.qlin_launch_dequantize_q8_1(_bytes_of(x_q8_1, q8_1_bytes(in_dim, m, mmq), "x_q8_1", device),
                                             _table_of(x, m, in_dim, _F32, "x", device), in_dim, m, int(mmq))
    if rc != 0:
        raise QlinError("qlin_launch_dequantize_q8_1", rc)


class Lora:
    """Adapters of one projection in slots: a [n_adapters, max_rank, in_dim] and b [n_adapters, out_dim, max_rank], both
    bfloat16, float16 or float32.  Holds on to the tensors."""

    def __init__(self, a, b):
        lib()
        (n, rank, n_in), (n_b, out, rank_b) = a.shape, b.shape
        if a.dtype is not b.dtype or a.dtype not in _LORA_TYPES or n_b != n or rank_b != rank or a.device != b.device:
            raise ValueError(f"a {tuple(a.shape)} of {a.dtype} and b {tuple(b.shape)} of {b.dtype} are not one projection's adapters")
        if not a.is_contiguous() or not b.is_contiguous():
            raise ValueError("a and b are contiguous")
        self.a, self.b, self.type = a, b, _LORA_TYPES[a.dtype]
        self.n_adapters, self.max_rank, self.in_dim, self.out_dim = n, rank, n_in, out
        self.like, self.device = (self.type, n, rank, n_in), a.get_device()
        self.addresses = a.data_ptr(), b.data_ptr()


def lora_workspace_bytes(rows, n_mats, n_adapters, max_rank, in_dim):
    return int(lib().qlin_lora_workspace_bytes(rows, n_mats, n_adapters, max_rank, in_dim))


# structs qlin_lora, packed (filling ctypes structures takes several times as long)
_LORAS = [struct.Struct("@" + "4PNNi4x" * n) for n in range(5)]
assert _LORAS[1].size == C.sizeof(LoraArgs) and _LORAS[3].size == 3 * C.sizeof(LoraArgs)


def lora_add(x, adapter_ids, mats, *, ranks=None, scales=None, workspace=None):
    """mats: up to 4 (Lora, base, y) whose adapters read the same x: y = base + scale B (A x) of each row's adapter, y = base in
    rows without one (id < 0, or no slot's).  x [rows, in_dim], base and y [rows, out_dim] are float32 with contiguous rows, y may
    be base; adapter_ids [rows] and ranks [n_adapters] int32, scales [n_adapters] float32.  workspace: a uint8 tensor of
    lora_workspace_bytes(...)."""
    library, device = _lib or lib(), _device_of(x, "x")
    if not 1 <= len(mats) <= 4:
        raise ValueError(f"{len(mats)} projections: 1 to 4")
    like, rows = mats[0][0].like, x.shape[0]
    kind, slots, rank, width = like
    p_x, n_x = _rows_of(x, (rows, width), "x", device)
    each = []
    for w, base, y in mats:
        if w.like != like:
            raise ValueError("the projections' adapters have one type, number of slots, rank and input")
        if w.device != device:
            raise ValueError(f"adapters on {w.a.device}, x on device {device}")
        shape = rows, w.out_dim
        p_base, n_base = _rows_of(base, shape, "base", device)
        p_y, n_y = (p_base, n_base) if y is base else _rows_of(y, shape, "y", device)
        each += (*w.addresses, p_base, p_y, n_base, n_y, w.out_dim)
    p_ws = ws_bytes = 0
    if workspace is not None:
        p_ws, ws_bytes = _bytes_of(workspace, 0, "workspace", device), workspace.numel()
    rc = library.qlin_launch_lora_add(_LORAS[len(mats)].pack(*each), len(mats), kind, slots, rank, width,
                                      0 if ranks is None else _values_of(ranks, slots, _I32, "ranks", device),
                                      0 if scales is None else _values_of(scales, slots, _F32, "scales", device), p_x, n_x,
                                      _values_of(adapter_ids, rows, _I32, "adapter_ids", device), rows, p_ws, ws_bytes)
    if rc != 0:
        raise QlinError("qlin_launch_lora_add", rc)


class MoeRouting:
    """How experts are chosen (struct qlin_moe_routing).  bias: float32 [n_experts] or None.  Holds on to the tensor."""

    def __init__(self, *, sigmoid=False, bias=None, n_groups=1, top_groups=1, group_pairs=False, renormalise=False, scaling=1.0):
        lib()
        if bias is not None and (bias.dtype is not _F32 or not bias.is_contiguous()):
            raise ValueError(f"a bias of {bias.dtype}: contiguous float32")
        self.bias = bias
        self.args = MoeRoutingArgs(ptr(bias), int(sigmoid), n_groups, top_groups, int(group_pairs), int(renormalise), scaling)
        self.address = C.addressof(self.args)


def moe_route(how, logits, ids, weights):
    """The k experts of each token and their weights: logits float32 [tokens, n_experts] with contiguous rows into ids int32 and
    weights float32, both [tokens, k] and contiguous."""
    library, device = _lib or lib(), _device_of(logits, "logits")
    tokens, n_experts = logits.shape
    contiguous = logits.dtype is _F32 and logits.is_contiguous()
    p_logits, stride = (logits.data_ptr(), n_experts) if contiguous else _rows_of(logits, logits.shape, "logits", device)
    shape = ids.shape
    k = shape[1]
    if how.bias is not None:
        _values_of(how.bias, n_experts, _F32, "the bias", device)
    if shape[0] < tokens or weights.shape != shape:
        raise ValueError(f"ids {tuple(ids.shape)} and weights {tuple(weights.shape)} for {tokens} tokens")
    rc = library.qlin_launch_moe_route(how.address, p_logits, stride, _table_of(ids, tokens, k, _I32, "ids", device),
                                       _table_of(weights, tokens, k, _F32, "weights", device), tokens, n_experts, k)
    if rc != 0:
        raise QlinError("qlin_launch_moe_route", rc)


def verify_drafts_workspace_bytes(n_seqs, max_drafts, vocab):
    return int(lib().qlin_verify_drafts_workspace_bytes(n_seqs, max_drafts, vocab))


def _logits_of(t, shape, name, device):
    """The address and the row stride of [n, rows, vocab] logits that lie row after row."""
    if t.shape == shape and t.is_contiguous() and t.dtype is _F32 and t.get_device() == device:
        return t.data_ptr(), shape[2]
    n, rows, vocab = shape
    seq, row, one = t.stride() if t.dim() == 3 else (0, 0, 0)
    if t.dtype is not _F32 or tuple(t.shape) != tuple(shape) or t.get_device() != device or one != 1 and vocab > 1 or (
            n > 1 and rows > 0 and seq != rows * row):
        raise ValueError(f"{name}: {tuple(t.shape)} of {t.dtype}, strides {t.stride()}, on {t.device}, not float32 [{n}, {rows}, "
                         f"{vocab}] row after row on device {device}")
    return t.data_ptr(), row if rows > 1 else seq if n > 1 else max(row, vocab)


def verify_drafts(target, drafts, uniform, tokens, accepted, *, draft_logits=None, n_drafts=None, temperature=None, logprobs=None,
                  rates=None, workspace=None):
    """Drafted tokens checked against the target's probabilities, and the next token of each sequence.  target float32
    [n_seqs, max_drafts + 1, vocab] and draft_logits [n_seqs, max_drafts, vocab] (None: drafted by lookup) row after row; drafts
    int32 [n_seqs, max_drafts] (None with max_drafts 0), uniform float32 [n_seqs, max_drafts + 1]; n_drafts int32 and
    temperature float32 [n_seqs] or None.  Into tokens int32 [n_seqs, max_drafts + 1], accepted int32 [n_seqs], and, where given,
    logprobs float32 [n_seqs, max_drafts + 1] and rates float32 [n_seqs, max_drafts].  workspace: a uint8 tensor of
    verify_drafts_workspace_bytes(...)."""
    library, device, shape = _lib or lib(), _device_of(target, "target"), target.shape
    n, rows, vocab = shape
    d = rows - 1
    contiguous = target.dtype is _F32 and target.is_contiguous()
    p_target, target_stride = (target.data_ptr(), vocab) if contiguous else _logits_of(target, shape, "target", device)
    p_draft = draft_stride = p_ws = ws_bytes = 0
    if draft_logits is not None:
        p_draft, draft_stride = _logits_of(draft_logits, (n, d, vocab), "draft_logits", device)
    if workspace is not None:
        p_ws, ws_bytes = _bytes_of(workspace, 0, "workspace", device), workspace.numel()
    rc = library.qlin_launch_verify_drafts(
        p_target, target_stride, p_draft if d else 0, draft_stride, 0 if drafts is None else _table_of(drafts, n, d, _I32, "drafts", device),
        0 if n_drafts is None else _values_of(n_drafts, n, _I32, "n_drafts", device),
        0 if temperature is None else _values_of(temperature, n, _F32, "temperature", device),
        _table_of(uniform, n, rows, _F32, "uniform", device), _table_of(tokens, n, rows, _I32, "tokens", device),
        _values_of(accepted, n, _I32, "accepted", device), 0 if logprobs is None else _table_of(logprobs, n, rows, _F32, "logprobs", device),
        0 if rates is None else _table_of(rates, n, d, _F32, "rates", device), n, d, vocab, p_ws, ws_bytes)
    if rc != 0:
        raise QlinError("qlin_launch_verify_drafts", rc)
