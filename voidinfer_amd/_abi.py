"""ctypes view of include/voidinfer_sampling.h (the C ABI of libvoidinfer_sampling.so).

Struct layouts are mirrored twice: as numpy dtypes (for building device arrays of
parameters / reading outputs) and as ctypes structures (for by-pointer host
arguments).  ``load()`` raises ImportError when the built library is missing, so
no caller can silently fall back to a CPU path.
"""
from __future__ import annotations

import ctypes as C
import struct
from pathlib import Path

import numpy as np

import os

# VOIDINFER_AMD_LIB selects another build of the same library (e.g. an instrumented one).
LIB_PATH = Path(os.environ.get("VOIDINFER_AMD_LIB", Path(__file__).resolve().parent / "libvoidinfer_sampling.so"))
BINDING_PATH = Path(__file__).resolve().parent / "_binding.so"   # tensors to the host structs (csrc/binding.cpp)

BF16, F16, F32 = 0, 1, 2
OK, ERR_INVALID, ERR_UNSUPPORTED, ERR_WORKSPACE, ERR_LAUNCH, ERR_DEVICE = range(6)
FLAG_NONFINITE, FLAG_EMPTY, FLAG_ZERO_Q, FLAG_NO_RESIDUAL, FLAG_BAD_HISTORY = 1, 2, 4, 8, 16
FLAG_ERROR = 0x80000000
VERIFY_GREEDY, VERIFY_SAMPLED, VERIFY_SAMPLED_TOPK = 0, 1, 2
ROUTE_TOPK, ROUTE_FULL, ROUTE_ALL = 1, 2, 3
ABSENT_OCCURRENCE = 0x7F7F7F7F

GREEDY_ROW = np.dtype([("serial", "<u8"), ("token", "<i4"), ("nonfinite", "<u4")])
ROW_PARAMS = np.dtype([
    ("temperature", "<f4"), ("top_p", "<f4"), ("min_p", "<f4"),
    ("repetition_penalty", "<f4"), ("presence_penalty", "<f4"), ("frequency_penalty", "<f4"),
    ("top_k", "<i4"), ("lane", "<u4"), ("seed", "<u8"), ("position", "<i4"), ("reserved", "<u4"),
])
SAMPLE_STATS = np.dtype([
    ("flags", "<u4"), ("support", "<u4"), ("finite", "<u4"), ("reserved", "<u4"),
    ("support_mass", "<f8"), ("uniform", "<f8"),
])
assert GREEDY_ROW.itemsize == 16 and ROW_PARAMS.itemsize == 48 and SAMPLE_STATS.itemsize == 32


DRAFT_SAMPLING = np.dtype([   # vi_draft_sampling == DraftSelectSampling (dflash2_draft.cu:2562-2572)
    ("inv_temperature", "<f4"), ("top_p", "<f4"), ("min_p", "<f4"), ("top_k", "<i4"), ("seed", "<u8"),
    ("key_base", "<i4"), ("reserved", "<i4"), ("presence_penalty", "<f4"), ("reserved2", "<i4"),
    ("first_occurrence", "<u8"),
])
assert DRAFT_SAMPLING.itemsize == 48


class DeviceSampling(C.Structure):
    """vi_device_sampling == Exl3DeviceSampling (src/exl3/sampled_select.h:17-28)."""
    _fields_ = [
        ("temperature", C.c_float), ("top_k", C.c_int32), ("top_p", C.c_float), ("min_p", C.c_float),
        ("seed", C.c_uint64), ("presence_penalty", C.c_float), ("reserved", C.c_int32),
        ("first_occurrence", C.c_void_p),
    ]


assert C.sizeof(DeviceSampling) == 40

# Host structs of the logit rules and of the paged cache (field order and padding as in
# the header); the calls on tensors pack all but the first in csrc/binding.cpp.
LOGIT_RULES = struct.Struct("<12Qqiiii")     # vi_logit_rules
KV_CACHE = struct.Struct("<2Q3qiiiiii")      # vi_kv_cache
LANE_ROWS = struct.Struct("<3Qqiiii")        # vi_lane_rows
HEAD_ROWS = struct.Struct("<Qqq")            # vi_head_rows
ROTATION = struct.Struct("<3Qiiii")          # vi_rotation
PAGE_MAP = struct.Struct("<4Qqiiii")         # vi_page_map
PAGE_POOL = struct.Struct("<Qqqii")          # vi_page_pool
assert (LOGIT_RULES.size, KV_CACHE.size, LANE_ROWS.size, HEAD_ROWS.size, ROTATION.size, PAGE_MAP.size,
        PAGE_POOL.size) == (120, 64, 48, 24, 40, 56, 32)

_vp, _i, _i64, _u64, _sz, _u32 = C.c_void_p, C.c_int, C.c_int64, C.c_uint64, C.c_size_t, C.c_uint32

SIGNATURES = {
    "vi_init": ([], _i),
    "vi_status_string": ([_i], C.c_char_p),
    "vi_abi_version": ([], _u32),
    "vi_greedy_workspace_bytes": ([_i, _i], _sz),
    "vi_greedy_rows": ([_vp, _i, _i, _i, _i64, _u64, _vp, _vp, _sz, _vp], _i),
    "vi_greedy_rows_noalloc": ([_vp, _i, _i, _i, _i64, _u64, _vp, _vp], _i),
    "vi_topk_workspace_bytes": ([_i, _i, _i], _sz),
    "vi_topk_rows": ([_vp, _i, _i, _i, _i64, _i, _vp, _vp, _vp, _vp, _vp, _sz, _vp], _i),
    "vi_topk16_for_test": ([_vp, _i, _i, _vp, _vp, _vp, _vp], _i),
    "vi_sampled_packet_workspace_bytes": ([_i, _i], _sz),
    "vi_sampled_packet": ([_vp, _i, _i, _i, _i64, C.POINTER(DeviceSampling), _i, _vp, _i, _vp, _i, _u64,
                           _vp, _vp, _sz, _vp], _i),
    "vi_row_scores_workspace_bytes": ([_i, _i], _sz),
    "vi_row_scores": ([_vp, _i, _i, _i, _i64, _vp, _vp, _vp, _vp, _sz, _vp], _i),
    "vi_sampled_scores_workspace_bytes": ([_i, _i], _sz),
    "vi_sampled_scores": ([_vp, _i, _i, _i, _i64, C.POINTER(DeviceSampling), _i, C.c_float, _vp, _vp, _vp, _vp,
                           _sz, _vp], _i),
    "vi_draft_choice": ([_i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp], _i),
    "vi_selector_chain": ([_i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp], _i),
    "vi_build_verification_tree": ([_vp, _i, _vp, _vp, _i, _i, C.c_float, _vp, _vp, _vp, _vp], _i),
    "vi_penalty_state_bytes": ([_i, _i], _sz),
    "vi_penalty_state_reset": ([_vp, _i, _i, _i, _vp], _i),
    "vi_penalty_state_update": ([_vp, _i, _i, _i, _vp, _vp, _i, _vp], _i),
    "vi_sample_rows_state": ([_vp, _i, _i, _i, _i64, _vp, _vp, _i, _i, _vp, _vp, _vp, _i64, _vp, _u32, _vp, _sz,
                              _vp], _i),
    "vi_packet_transport_create": ([_i, _i, C.POINTER(C.c_void_p)], _i),
    "vi_packet_transport_destroy": ([_vp], _i),
    "vi_packet_submit": ([_vp, _vp, _i, _vp, C.POINTER(C.c_int)], _i),
    "vi_packet_query": ([_vp, _i, C.POINTER(C.c_int)], _i),
    "vi_packet_finish": ([_vp, _i, _vp, _i], _i),
    "vi_presence_reset": ([_vp, _i, _vp], _i),
    "vi_presence_truncate": ([_vp, _i, _i, _vp], _i),
    "vi_presence_record": ([_vp, _i, _i, _vp, _sz, _vp], _i),
    "vi_sample_workspace_bytes": ([_i, _i, _i64], _sz),
    "vi_sample_rows": ([_vp, _i, _i, _i, _i64, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _i64, _vp, _u32, _vp, _sz,
                        _vp], _i),
    "vi_verify_workspace_bytes": ([_i, _i, _i], _sz),
    "vi_verify_rows": ([_i, _vp, _i, _i64, _i, _vp, _i, _i64, _i, _i, _i, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp,
                        _vp, _sz, _vp], _i),
    "vi_process_logits": ([_vp, _i, _i, _i, _i64, _vp, _vp, _i64, _vp, _vp], _i),
    "vi_norm_rotate_append": ([_vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, C.c_float, _vp, _vp, _i64, _i64, _vp, _vp], _i),
    "vi_prefix_attention_workspace_bytes": ([_i, _i, _i, _i, _i, _i, _i, _i, _i64, _i64], _sz),
    "vi_prefix_attention": ([_vp, _vp, _i, _vp, C.c_float, _i, _vp, _vp, _i, _i, _i64, _i64, _vp, _vp, _i64, _i64, _vp,
                             _vp, _sz, _vp], _i),
    "vi_pages_fork": ([_vp, _vp, _vp, _i, _vp], _i),
    "vi_pages_extend_workspace_bytes": ([_i], _sz),
    "vi_pages_extend": ([_vp, _vp, _vp, _vp, _i, _vp, _sz, _vp], _i),
    "vi_pages_truncate": ([_vp, _vp, _vp, _i, _vp], _i),
    "vi_pages_copy": ([_vp, _i, _vp, _vp, _i, _vp], _i),
    "vi_pages_compact_workspace_bytes": ([_i], _sz),
    "vi_pages_compact": ([_vp, _vp, _vp, _sz, _vp], _i),
    "vi_keep_rows": ([_vp, _vp, _i, _vp, _vp, _vp, _i, _vp, _i, _vp], _i),
    "vi_probe_read": ([_vp, _sz, _vp, _vp], _i),
    "vi_probe_copy": ([_vp, _vp, _sz, _vp], _i),
}

_lib = None


def load() -> C.CDLL:
    """Load the in-tree library (ImportError if it has not been built)."""
    global _lib
    if _lib is None:
        for path in (LIB_PATH, BINDING_PATH):
            if not path.exists():
                raise ImportError(
                    f"{path} is missing: build it with `python voidinfer_amd/build.py` "
                    "(there is no CPU fallback)")
        lib = C.CDLL(str(LIB_PATH))
        for name, (args, res) in SIGNATURES.items():
            try:
                fn = getattr(lib, name)
            except AttributeError as e:
                raise ImportError(f"{LIB_PATH} lacks {name}: it is older than its sources, rebuild it with "
                                  "`python voidinfer_amd/build.py`") from e
            fn.argtypes = args
            fn.restype = res
        _lib = lib
    return _lib


class VIError(RuntimeError):
    def __init__(self, status: int, what: str):
        self.status = status
        msg = load().vi_status_string(status).decode()
        super().__init__(f"{what}: {msg} (status {status})")


def check(status: int, what: str) -> None:
    if status != OK:
        if status == ERR_INVALID:
            raise ValueError(f"{what}: invalid argument")
        raise VIError(status, what)
