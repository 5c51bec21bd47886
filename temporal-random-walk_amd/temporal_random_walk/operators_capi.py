"""The C ABI of the operators (include/trw_operators.h) by ctypes, for callers
with device pointers of their own.  Programs on PyTorch tensors use
``temporal_random_walk.operators``."""
from __future__ import annotations

import ctypes as C
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libtrw_operators.so")
ABI_VERSION = 1  # TRW_OPS_ABI_VERSION

# every symbol the header declares
EXPORTS = [
    "trw_ops_walk_mask", "trw_ops_attention_workspace", "trw_ops_attention_forward",
    "trw_ops_attention_backward", "trw_ops_attention_step_workspace", "trw_ops_attention_step",
    "trw_ops_relative_bias", "trw_ops_relative_bias_workspace", "trw_ops_relative_bias_backward",
    "trw_ops_paged_write", "trw_ops_paged_read", "trw_ops_paged_step_workspace",
    "trw_ops_paged_step", "trw_ops_beam_select_workspace", "trw_ops_beam_select",
    "trw_ops_beam_reorder",
    "trw_ops_last_error", "trw_ops_abi_version",
]


class Rows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("row_stride", C.c_int64), ("head_stride", C.c_int64)]


class MaskParams(C.Structure):
    _fields_ = [("docs", C.c_int64), ("q_rows", C.c_int64), ("k_rows", C.c_int64),
                ("q_length", C.c_int64), ("k_length", C.c_int64),
                ("q_lens", C.c_void_p), ("k_lens", C.c_void_p),
                ("q_offsets", C.c_void_p), ("k_offsets", C.c_void_p), ("prefix", C.c_void_p),
                ("kind", C.c_int32), ("q_rows_info", C.c_void_p), ("k_rows_info", C.c_void_p),
                ("docs_info", C.c_void_p)]


class Score(C.Structure):
    _fields_ = [("scale", C.c_float), ("softcap", C.c_float), ("table", C.c_void_p),
                ("buckets", C.c_void_p), ("num_buckets", C.c_int32), ("reach", C.c_int32),
                ("slopes", C.c_void_p), ("q_times", C.c_void_p), ("k_times", C.c_void_p)]


class AttentionParams(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32),
                ("dim", C.c_int32), ("q_rows", C.c_int64), ("k_rows", C.c_int64),
                ("q_rows_info", C.c_void_p), ("k_rows_info", C.c_void_p),
                ("docs_info", C.c_void_p), ("docs", C.c_int64), ("longest", C.c_int64),
                ("own_causal", C.c_int32), ("covered", C.c_int32),
                ("score", Score),
                ("q", Rows), ("k", Rows), ("v", Rows), ("out", Rows), ("stats", C.c_void_p),
                ("out_low", Rows), ("d_out", Rows), ("d_q", Rows), ("d_k", Rows), ("d_v", Rows),
                ("d_table", C.c_void_p), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_uint64)]


class StepParams(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32),
                ("dim", C.c_int32), ("batch", C.c_int64), ("capacity", C.c_int64),
                ("lens", C.c_void_p), ("score", Score),
                ("q", Rows), ("k", Rows), ("v", Rows), ("out", Rows),
                ("k_cache", C.c_void_p), ("v_cache", C.c_void_p),
                ("k_batch_stride", C.c_int64), ("k_pos_stride", C.c_int64),
                ("k_head_stride", C.c_int64), ("v_batch_stride", C.c_int64),
                ("v_pos_stride", C.c_int64), ("v_head_stride", C.c_int64),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


class BiasParams(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("heads", C.c_int32), ("num_buckets", C.c_int32),
                ("reach", C.c_int32), ("q_len", C.c_int64), ("k_len", C.c_int64),
                ("q_offset", C.c_int64), ("table", C.c_void_p), ("buckets", C.c_void_p),
                ("out", C.c_void_p), ("d_out", C.c_void_p), ("d_out_head_stride", C.c_int64),
                ("d_out_row_stride", C.c_int64), ("d_table", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


class Pages(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("kv_heads", C.c_int32), ("dim", C.c_int32),
                ("page_rows", C.c_int32), ("pages", C.c_int64), ("k", C.c_void_p),
                ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("k_stride", C.c_int64), ("v_stride", C.c_int64),
                ("k_scale_stride", C.c_int64), ("v_scale_stride", C.c_int64),
                ("table", C.c_void_p), ("table_stride", C.c_int64), ("table_pages", C.c_int64),
                ("walks", C.c_int64)]


class PagedCopyParams(C.Structure):
    _fields_ = [("pages", Pages), ("dtype", C.c_int32), ("rows", C.c_int64),
                ("length", C.c_int64), ("counts", C.c_void_p), ("offsets", C.c_void_p),
                ("starts", C.c_void_p), ("k", Rows), ("v", Rows), ("times", C.c_void_p),
                ("k_times", C.c_void_p)]


class PagedStepParams(C.Structure):
    _fields_ = [("pages", Pages), ("dtype", C.c_int32), ("heads", C.c_int32),
                ("lens", C.c_void_p), ("first", C.c_void_p), ("score", Score),
                ("q", Rows), ("k", Rows), ("v", Rows), ("out", Rows),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


class BeamSelectParams(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("beams", C.c_int32), ("width", C.c_int32),
                ("groups", C.c_int64), ("nodes", C.c_int64), ("logits", C.c_void_p),
                ("group_stride", C.c_int64), ("beam_stride", C.c_int64),
                ("scores", C.c_void_p), ("ended", C.c_void_p), ("end_token", C.c_int64),
                ("out_scores", C.c_void_p), ("out_tokens", C.c_void_p),
                ("out_parents", C.c_void_p), ("out_ended", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


class BeamReorderParams(C.Structure):
    _fields_ = [("beams", C.c_int32), ("page_rows", C.c_int32), ("count", C.c_int32),
                ("groups", C.c_int64), ("pages", C.c_int64), ("table_pages", C.c_int64),
                ("table_stride", C.c_int64), ("table", C.c_void_p), ("out_table", C.c_void_p),
                ("lens", C.c_void_p), ("out_lens", C.c_void_p), ("parents", C.c_void_p),
                ("caches", C.POINTER(Pages)), ("k_times", C.c_void_p)]


_lib = None


def lib():
    """Load libtrw_operators.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: build it first "
                              "(python temporal-random-walk_amd/build.py)")
        L = C.CDLL(LIB_PATH)
        P = C.c_void_p
        size = C.POINTER(C.c_uint64)
        L.trw_ops_walk_mask.argtypes = [C.POINTER(MaskParams), P]
        L.trw_ops_attention_workspace.argtypes = [C.POINTER(AttentionParams), C.c_int32, size]
        L.trw_ops_attention_forward.argtypes = [C.POINTER(AttentionParams), P]
        L.trw_ops_attention_backward.argtypes = [C.POINTER(AttentionParams), P]
        L.trw_ops_attention_step_workspace.argtypes = [C.POINTER(StepParams), size]
        L.trw_ops_attention_step.argtypes = [C.POINTER(StepParams), P]
        L.trw_ops_relative_bias.argtypes = [C.POINTER(BiasParams), P]
        L.trw_ops_relative_bias_workspace.argtypes = [C.POINTER(BiasParams), size]
        L.trw_ops_relative_bias_backward.argtypes = [C.POINTER(BiasParams), P]
        L.trw_ops_paged_write.argtypes = [C.POINTER(PagedCopyParams), P]
        L.trw_ops_paged_read.argtypes = [C.POINTER(PagedCopyParams), P]
        L.trw_ops_paged_step_workspace.argtypes = [C.POINTER(PagedStepParams), size]
        L.trw_ops_paged_step.argtypes = [C.POINTER(PagedStepParams), P]
        L.trw_ops_beam_select_workspace.argtypes = [C.POINTER(BeamSelectParams), size]
        L.trw_ops_beam_select.argtypes = [C.POINTER(BeamSelectParams), P]
        L.trw_ops_beam_reorder.argtypes = [C.POINTER(BeamReorderParams), P]
        L.trw_ops_last_error.restype = C.c_char_p
        L.trw_ops_abi_version.restype = C.c_int32
        if L.trw_ops_abi_version() != ABI_VERSION:
            raise ImportError(f"{LIB_PATH} has ABI {L.trw_ops_abi_version()}, these bindings "
                              f"expect {ABI_VERSION}: rebuild it")
        _lib = L
    return _lib


def call(function, *args):
    """A function of the library; a failure's status and message as an exception."""
    rc = function(*args)
    if rc != 0:
        message = lib().trw_ops_last_error().decode()
        raise {1: ValueError, 3: MemoryError}.get(rc, RuntimeError)(message)
