"""ctypes binding of include/kda_b200.h.  The library is the only compute path: a missing or unloadable
libkda_b200.so raises, there is no fallback."""
from __future__ import annotations

import ctypes as C
from pathlib import Path

PKG = Path(__file__).resolve().parent
LIB_PATH = PKG / "libkda_b200.so"

FRONTEND_RAW, FRONTEND_PLAIN = 0, 1
STATE_VALUE_FIRST, STATE_KEY_FIRST = 0, 1
NOALLOC_MAX_SEQS, NOALLOC_MAX_HEADS = 64, 16
KERNEL_TCGEN05, KERNEL_MMA_SYNC, KERNEL_TCGEN05_TWO_TASK = 0, 1, 2
MAX_CUT_PIECES = 128
EXPORTS = ["kda_prefill_workspace_bytes", "kda_prefill_workspace_bytes_cuts", "kda_prefill_workspace_clear_bytes", "kda_prefill_launch", "kda_prefill_plan_counts", "kda_prefill_launch_noalloc", "kda_segment_launch", "kda_scan_launch", "kda_scan_strided_launch",
           "kda_fixup_launch", "kda_fixup_tiles_launch", "kda_segment_tiles", "kda_state_rows_copy", "kda_error_string", "kda_abi_struct_bytes", "kda_version",
           "kda_debug_configure", "kda_short_conv_launch", "kda_short_conv_step_launch", "kda_selective_scan_workspace_bytes",
           "kda_selective_scan_launch", "kda_selective_scan_step_launch", "kda_step_launch", "kda_pool_workspace_bytes",
           "kda_pool_copy_launch", "kda_pool_fork_launch", "kda_pool_free_launch", "kda_pool_compact_launch",
           "kda_gated_scan_launch", "kda_gated_scan_step_launch", "kda_gated_scan_grad_launch", "kda_group_norm_workspace_bytes",
           "kda_group_norm_launch", "kda_group_norm_grad_launch"]
TYPE_BF16, TYPE_FP16, TYPE_FP32 = 0, 1, 2
SCAN_MAX_STATE, MAX_POOLS, MAX_TABLES = 128, 8, 8
GATED_SCAN_TILE, GROUP_NORM_MAX_WIDTH = 48, 16384
ACT_NONE, ACT_SILU, ACT_SIGMOID = 0, 1, 2


class KdaPrefillArgs(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("g", C.c_void_p), ("beta", C.c_void_p),
        ("out", C.c_void_p),
        ("ldq", C.c_int64), ("ldk", C.c_int64), ("ldv", C.c_int64), ("ldg", C.c_int64), ("ldbeta", C.c_int64),
        ("ldo", C.c_int64),
        ("A_log", C.c_void_p), ("dt_bias", C.c_void_p),
        ("scale", C.c_float), ("lower_bound", C.c_float),
        ("frontend", C.c_int32), ("state_layout", C.c_int32), ("H", C.c_int32), ("N", C.c_int32),
        ("T", C.c_int64),
        ("cu_seqlens", C.c_void_p), ("cu_is64", C.c_int32),
        ("src_base", C.c_void_p), ("src_slot_stride", C.c_int64), ("src_idx", C.c_void_p), ("src_idx_is64", C.c_int32),
        ("src_slots", C.c_int64),
        ("dst_base", C.c_void_p), ("dst_slot_stride", C.c_int64), ("dst_idx", C.c_void_p), ("dst_idx_is64", C.c_int32),
        ("dst_slots", C.c_int64),
        ("ck_base", C.c_void_p), ("ck_is_bf16", C.c_int32), ("ck_every", C.c_int32), ("ck_rows", C.c_int64),
        ("ck_starts", C.c_void_p), ("ck_starts_is64", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("status", C.c_void_p),
        ("kernel", C.c_int32),
        ("max_cut_pieces", C.c_int32),
    ]


class KdaSegmentArgs(C.Structure):
    _fields_ = [
        ("base", KdaPrefillArgs),
        ("n_seg", C.c_int32),
        ("seg_t0", C.c_void_p), ("seg_t1", C.c_void_p), ("seg_need_map", C.c_void_p),
        ("qt", C.c_void_p), ("P", C.c_void_p), ("S_loc", C.c_void_p),
        ("tiles", C.c_void_p), ("n_tiles", C.c_int64),
    ]


class KdaSequences(C.Structure):
    _fields_ = [
        ("cu_seqlens", C.c_void_p), ("slots", C.c_void_p), ("n_slots", C.c_int64), ("T", C.c_int64), ("status", C.c_void_p),
        ("cu_is64", C.c_int32), ("slots_is64", C.c_int32), ("N", C.c_int32), ("zero_rest", C.c_int32),
    ]


class KdaConvArgs(C.Structure):
    _fields_ = [
        ("x", C.c_void_p), ("weight", C.c_void_p), ("bias", C.c_void_p), ("out", C.c_void_p), ("src", C.c_void_p),
        ("dst", C.c_void_p),
        ("ldx", C.c_int64), ("ldo", C.c_int64), ("src_slot_stride", C.c_int64), ("dst_slot_stride", C.c_int64),
        ("seq", KdaSequences),
        ("C", C.c_int32), ("W", C.c_int32), ("type", C.c_int32), ("weight_type", C.c_int32), ("silu", C.c_int32),
    ]


class KdaScanArgs(C.Structure):
    _fields_ = [
        ("u", C.c_void_p), ("dt", C.c_void_p), ("B", C.c_void_p), ("C", C.c_void_p), ("z", C.c_void_p), ("out", C.c_void_p),
        ("A", C.c_void_p), ("D", C.c_void_p), ("dt_bias", C.c_void_p), ("src", C.c_void_p), ("dst", C.c_void_p),
        ("ldu", C.c_int64), ("lddt", C.c_int64), ("ldb", C.c_int64), ("ldc", C.c_int64), ("ldz", C.c_int64),
        ("ldo", C.c_int64), ("src_slot_stride", C.c_int64), ("dst_slot_stride", C.c_int64),
        ("seq", KdaSequences),
        ("Dm", C.c_int32), ("Ns", C.c_int32), ("groups", C.c_int32), ("type", C.c_int32), ("softplus", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class KdaStepArgs(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("g", C.c_void_p), ("beta", C.c_void_p),
        ("out", C.c_void_p), ("A_log", C.c_void_p), ("dt_bias", C.c_void_p), ("pool", C.c_void_p),
        ("ldq", C.c_int64), ("ldk", C.c_int64), ("ldv", C.c_int64), ("ldg", C.c_int64), ("ldbeta", C.c_int64),
        ("ldo", C.c_int64), ("slot_stride", C.c_int64),
        ("seq", KdaSequences),
        ("scale", C.c_float), ("lower_bound", C.c_float), ("frontend", C.c_int32), ("H", C.c_int32),
    ]


class KdaPoolArgs(C.Structure):
    _fields_ = [
        ("base", C.c_void_p * MAX_POOLS), ("stride", C.c_int64 * MAX_POOLS), ("bytes", C.c_int64 * MAX_POOLS),
        ("slots", C.c_int64), ("n_pools", C.c_int32), ("n_tables", C.c_int32), ("used", C.c_void_p), ("src", C.c_void_p),
        ("dst", C.c_void_p), ("n", C.c_int64), ("src_is64", C.c_int32), ("dst_is64", C.c_int32), ("slots_out", C.c_void_p),
        ("remap", C.c_void_p), ("tables", C.c_void_p * MAX_TABLES), ("table_n", C.c_int64 * MAX_TABLES),
        ("table_is64", C.c_int32 * MAX_TABLES), ("status", C.c_void_p), ("workspace", C.c_void_p),
        ("workspace_bytes", C.c_size_t),
    ]


class KdaGatedScanArgs(C.Structure):
    _fields_ = [
        ("x", C.c_void_p), ("r", C.c_void_p), ("i", C.c_void_p), ("out", C.c_void_p), ("rate", C.c_void_p),
        ("r_bias", C.c_void_p), ("i_bias", C.c_void_p), ("src", C.c_void_p), ("dst", C.c_void_p), ("tiles", C.c_void_p),
        ("ldx", C.c_int64), ("ldr", C.c_int64), ("ldi", C.c_int64), ("ldo", C.c_int64), ("src_slot_stride", C.c_int64),
        ("dst_slot_stride", C.c_int64),
        ("seq", KdaSequences),
        ("rate_scale", C.c_float), ("C", C.c_int32), ("type", C.c_int32),
    ]


class KdaGatedScanGradArgs(C.Structure):
    _fields_ = [
        ("x", C.c_void_p), ("r", C.c_void_p), ("i", C.c_void_p), ("dy", C.c_void_p), ("dx", C.c_void_p), ("dr", C.c_void_p),
        ("di", C.c_void_p), ("rate", C.c_void_p), ("r_bias", C.c_void_p), ("i_bias", C.c_void_p), ("tiles", C.c_void_p),
        ("src", C.c_void_p), ("dfinal", C.c_void_p), ("dsrc", C.c_void_p), ("drate", C.c_void_p), ("dr_bias", C.c_void_p),
        ("di_bias", C.c_void_p),
        ("ldx", C.c_int64), ("ldr", C.c_int64), ("ldi", C.c_int64), ("lddy", C.c_int64), ("lddx", C.c_int64),
        ("lddr", C.c_int64), ("lddi", C.c_int64),
        ("seq", KdaSequences),
        ("rate_scale", C.c_float), ("C", C.c_int32), ("type", C.c_int32),
    ]


class KdaGroupNormArgs(C.Structure):
    _fields_ = [
        ("x", C.c_void_p), ("z", C.c_void_p), ("dy", C.c_void_p), ("out", C.c_void_p), ("dz", C.c_void_p), ("weight", C.c_void_p),
        ("bias", C.c_void_p), ("dweight", C.c_void_p), ("dbias", C.c_void_p), ("workspace", C.c_void_p),
        ("workspace_bytes", C.c_size_t),
        ("T", C.c_int64), ("ldx", C.c_int64), ("ldz", C.c_int64), ("lddy", C.c_int64), ("ldo", C.c_int64), ("lddz", C.c_int64),
        ("eps", C.c_float), ("G", C.c_int32), ("D", C.c_int32), ("act", C.c_int32), ("center", C.c_int32), ("shared", C.c_int32),
        ("type", C.c_int32),
    ]


STRUCTS = [KdaPrefillArgs, KdaSegmentArgs, KdaConvArgs, KdaScanArgs, KdaStepArgs, KdaPoolArgs, KdaGatedScanArgs, KdaGatedScanGradArgs,
           KdaGroupNormArgs]
_lib = None


def lib():
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                "(nvcc, sm_100a). kda_b200 has no other compute path.")
        L = C.CDLL(str(LIB_PATH))
        L.kda_prefill_workspace_bytes.argtypes = [C.c_int32, C.c_int32]
        L.kda_prefill_workspace_bytes.restype = C.c_size_t
        L.kda_prefill_workspace_bytes_cuts.argtypes = [C.c_int32, C.c_int32, C.c_int32]
        L.kda_prefill_workspace_bytes_cuts.restype = C.c_size_t
        L.kda_prefill_workspace_clear_bytes.argtypes = []
        L.kda_prefill_workspace_clear_bytes.restype = C.c_size_t
        L.kda_prefill_launch.argtypes = [C.POINTER(KdaPrefillArgs), C.c_void_p]
        L.kda_prefill_launch.restype = C.c_int
        L.kda_prefill_plan_counts.argtypes = [C.POINTER(KdaPrefillArgs), C.POINTER(C.c_int32), C.c_void_p]
        L.kda_prefill_plan_counts.restype = C.c_int
        L.kda_prefill_launch_noalloc.argtypes = [C.POINTER(KdaPrefillArgs), C.c_void_p]
        L.kda_prefill_launch_noalloc.restype = C.c_int
        L.kda_segment_launch.argtypes = [C.POINTER(KdaSegmentArgs), C.c_void_p]
        L.kda_segment_launch.restype = C.c_int
        L.kda_scan_launch.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_int32,
                                      C.c_void_p]
        L.kda_scan_launch.restype = C.c_int
        L.kda_scan_strided_launch.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_int32,
                                              C.c_int64, C.c_void_p]
        L.kda_scan_strided_launch.restype = C.c_int
        L.kda_fixup_launch.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                       C.c_int32, C.c_int32, C.c_void_p]
        L.kda_fixup_launch.restype = C.c_int
        L.kda_fixup_tiles_launch.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p,
                                             C.c_void_p, C.c_int32, C.c_int32, C.c_int64, C.c_void_p]
        L.kda_fixup_tiles_launch.restype = C.c_int
        L.kda_segment_tiles.argtypes = [C.c_void_p, C.c_void_p, C.c_int32, C.c_int64]
        L.kda_segment_tiles.restype = C.c_int64
        L.kda_state_rows_copy.argtypes = [C.c_void_p, C.c_int64, C.c_int32, C.c_void_p, C.c_int64, C.c_void_p, C.c_int32,
                                          C.c_int32, C.c_void_p]
        L.kda_state_rows_copy.restype = C.c_int
        L.kda_error_string.argtypes = [C.c_int]
        L.kda_error_string.restype = C.c_char_p
        L.kda_version.restype = C.c_char_p
        L.kda_debug_configure.argtypes = [C.c_int64, C.c_int32, C.c_void_p]
        L.kda_debug_configure.restype = C.c_int
        L.kda_abi_struct_bytes.argtypes = [C.c_int]
        L.kda_abi_struct_bytes.restype = C.c_size_t
        for name, block in (("short_conv", KdaConvArgs), ("short_conv_step", KdaConvArgs), ("selective_scan", KdaScanArgs),
                            ("selective_scan_step", KdaScanArgs), ("step", KdaStepArgs), ("pool_copy", KdaPoolArgs),
                            ("pool_fork", KdaPoolArgs), ("pool_free", KdaPoolArgs), ("pool_compact", KdaPoolArgs),
                            ("gated_scan", KdaGatedScanArgs), ("gated_scan_step", KdaGatedScanArgs),
                            ("gated_scan_grad", KdaGatedScanGradArgs), ("group_norm", KdaGroupNormArgs),
                            ("group_norm_grad", KdaGroupNormArgs)):
            entry = getattr(L, f"kda_{name}_launch")
            entry.argtypes, entry.restype = [C.POINTER(block), C.c_void_p], C.c_int
        L.kda_selective_scan_workspace_bytes.argtypes = [C.c_int64, C.c_int32, C.c_int32, C.c_int32]
        L.kda_selective_scan_workspace_bytes.restype = C.c_size_t
        L.kda_group_norm_workspace_bytes.argtypes = [C.c_int64, C.c_int32, C.c_int32, C.c_int32, C.c_int32]
        L.kda_group_norm_workspace_bytes.restype = C.c_size_t
        L.kda_pool_workspace_bytes.argtypes = [C.c_int64, C.c_int64]
        L.kda_pool_workspace_bytes.restype = C.c_size_t
        if any(L.kda_abi_struct_bytes(i) != C.sizeof(block) for i, block in enumerate(STRUCTS)):
            raise RuntimeError("libkda_b200.so and the Python binding disagree on the argument struct layout: rebuild")
        _lib = L
    return _lib


def check(rc: int, what: str):
    if rc != 0:
        raise RuntimeError(f"{what} failed: {lib().kda_error_string(rc).decode()} (code {rc})")


_raw = {}


def raw(name):
    """The entry point with an untyped argument block (words instead of the struct)."""
    f = _raw.get(name)
    if f is None:
        f = lib()[name]
        f.argtypes, f.restype = [C.c_void_p, C.c_void_p], C.c_int
        _raw[name] = f
    return f
