"""Python plumbing over the C ABI of libuocr_rswa_b200.so (tests and benchmark only).

The product is the shared library (hand-written sm_100a kernels behind `include/uocr_rswa_b200.h`)
plus the C++17 host classes under `include/uocr/`.  This module only loads the library with ctypes,
mirrors the structs of the header, and offers thin wrappers that take torch CUDA tensors (used here
purely as device-memory handles) and launch on torch's current stream.  There is no fallback: if
the library is missing or a call fails, an exception is raised.

The directory name is not a Python identifier; load it with

    importlib.util.spec_from_file_location("uocr_b200", "<repo>/unlimited-ocr.cpp_b200/__init__.py")
"""
from __future__ import annotations

import ctypes as C
import os
import struct
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB_PATH = os.path.join(HERE, "libuocr_rswa_b200.so")

F32, BF16 = 0, 1
BLOCK_TOKENS = 16
STATUS_BAD_BLOCK, STATUS_WAIT_TIMEOUT, STATUS_BAD_SLOT = 1, 2, 4

NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC,-fvisibility=hidden", "-shared", "-t", "0"]


def sources():
    csrc = os.path.join(HERE, "csrc")
    return sorted(os.path.join(csrc, f) for f in os.listdir(csrc) if f.endswith((".cu", ".cpp")))


def build(verbose: bool = False) -> str:
    """Compile every source under csrc/ for sm_100a into libuocr_rswa_b200.so (in-tree)."""
    cmd = ["nvcc", *NVCC_FLAGS, "-I", os.path.join(ROOT, "include"), "-I", os.path.join(HERE, "include"),
           "-I", os.path.join(HERE, "csrc"), "-o", LIB_PATH, *sources()]
    if verbose:
        print(" ".join(cmd))
    subprocess.check_call(cmd)
    return LIB_PATH


class PagedKV(C.Structure):
    """uocr_b200_paged_kv"""
    _fields_ = [("k_pool", C.c_void_p), ("v_pool", C.c_void_p), ("block_table", C.c_void_p),
                ("table_stride", C.c_int32), ("num_blocks", C.c_int32), ("kv_heads", C.c_int32),
                ("head_dim", C.c_int32), ("dtype", C.c_int32)]


class RopeDesc(C.Structure):
    """uocr_b200_rope_desc"""
    _fields_ = [("layout", C.c_int32), ("rotary_dim", C.c_int32), ("scaling", C.c_int32), ("theta", C.c_float),
                ("factor", C.c_float), ("orig_context", C.c_float), ("low", C.c_float), ("high", C.c_float),
                ("amplitude", C.c_float)]


class QkvRows(C.Structure):
    """uocr_b200_qkv_rows"""
    _fields_ = [("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("q_out", C.c_void_p), ("q_stride", C.c_int64),
                ("k_stride", C.c_int64), ("v_stride", C.c_int64), ("q_out_stride", C.c_int64), ("dtype", C.c_int32),
                ("heads", C.c_int32)]


class ScoreDesc(C.Structure):
    """uocr_b200_score"""
    _fields_ = [("scale", C.c_float), ("softcap", C.c_float), ("slopes", C.c_void_p), ("d_q_pos", C.c_void_p), ("d_key_pos", C.c_void_p),
                ("key_pos_stride", C.c_int32), ("d_lo", C.c_void_p), ("d_hi", C.c_void_p)]


class MassDesc(C.Structure):
    """uocr_b200_mass"""
    _fields_ = [("mass_in", C.c_void_p), ("mass_out", C.c_void_p), ("stride", C.c_int32), ("decay", C.c_float), ("scratch", C.c_void_p),
                ("scratch_bytes", C.c_size_t)]


class Error(RuntimeError):
    def __init__(self, status, msg):
        super().__init__(f"uocr_b200 status {status}: {msg}")
        self.status = status


class ArgumentError(Error, ValueError):
    """Tensors a call would misread (type, layout, size, device): the library gets bare addresses, so they are refused before it is called."""

    def __init__(self, msg):
        super().__init__(1, msg)


_LIB = None

_vp, _i, _i64 = C.c_void_p, C.c_int, C.c_int64
_SIGS = {
    "uocr_b200_status_string": (C.c_char_p, [_i]),
    "uocr_b200_last_error": (C.c_char_p, []),
    "uocr_b200_version": (C.c_char_p, []),
    "uocr_b200_launch_count": (C.c_uint64, []),
    "uocr_b200_workspace_create": (_i, [_i, C.POINTER(_vp)]),
    "uocr_b200_workspace_destroy": (_i, [_vp]),
    "uocr_b200_workspace_status": (_i, [_vp, _vp, C.POINTER(_i)]),
    "uocr_b200_workspace_set_timing": (_i, [_vp, _i]),
    "uocr_b200_workspace_set_overlap": (_i, [_vp, _i]),
    "uocr_b200_workspace_set_wait_limit": (_i, [_vp, C.c_uint]),
    "uocr_b200_noalloc_status": (_i, [_vp, C.POINTER(_i)]),
    "uocr_b200_workspace_set_out_dtype": (_i, [_vp, _i]),
    "uocr_b200_workspace_stream_read_gbs": (_i, [_vp, _vp, C.POINTER(C.c_double)]),
    "uocr_b200_workspace_last_kernel_ms": (_i, [_vp, C.POINTER(C.c_float)]),
    "uocr_b200_rswa_append_decode_batch_f32": (_i, [_vp] * 8 + [_i] * 5 + [_vp]),
    "uocr_b200_rswa_append_decode_f32": (_i, [_vp] * 6 + [_i] * 4 + [_vp]),
    "uocr_b200_rswa_append_decode_batch_paged": (_i, [C.POINTER(PagedKV)] + [_vp] * 6 + [_i, _i, _vp, _vp]),
    "uocr_b200_rswa_append_decode_batch_paged_layers": (_i, [_vp, _i, _vp, _vp, C.c_longlong, _vp, _vp, C.c_longlong, _vp, _vp,
                                                              _i, _i, _vp, _vp]),
    "uocr_b200_rswa_gather_paged_layers": (_i, [_vp, _i, _vp, C.c_longlong, _vp, _vp, _i, _i, _vp, _vp, C.c_longlong, _i,
                                                 _vp, _vp]),
    "uocr_b200_rswa_write_prefill_ragged_f32": (_i, [_vp] * 6 + [_i] * 4 + [_vp]),
    "uocr_b200_rswa_write_prefill_ragged_paged": (_i, [C.POINTER(PagedKV)] + [_vp] * 4 + [_i, _vp, _vp]),
    "uocr_b200_rswa_publish_slots": (_i, [_vp, _i, _vp, _i, _vp, _vp, _vp, _i, _i, _vp, _vp]),
    "uocr_b200_rswa_attention_batch_f32": (_i, [_vp] * 5 + [_i] * 5 + [_vp, _vp, _vp]),
    "uocr_b200_rswa_attention_batch_paged": (_i, [C.POINTER(PagedKV)] + [_vp] * 4 + [_i, _i, _vp, _vp, _vp]),
    "uocr_b200_rswa_prefill_text_paged": (_i, [C.POINTER(PagedKV), _vp, _vp, _i] + [_vp] * 7 + [_i, _i, _i, _vp, _vp, _vp]),
    "uocr_b200_rswa_text_scatter_paged": (_i, [C.POINTER(PagedKV), _vp, _vp, _i] + [_vp] * 4 + [_i, _vp, _vp]),
    "uocr_b200_rswa_text_scatter_fill_paged": (_i, [C.POINTER(PagedKV), _vp, _vp, _i] + [_vp] * 9 + [_i, _i, _vp, _vp]),
    "uocr_b200_rswa_prefill_attention_tc": (_i, [C.POINTER(PagedKV), _vp, _vp, _i, _vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp]),
    "uocr_b200_rswa_prefill_plan_tc": (_i, [_vp, _i, _vp, _i, _vp, _vp]),
    "uocr_b200_workspace_prefill_plan_serial": (C.c_uint, [_vp]),
    "uocr_b200_rswa_ring_fill_paged": (_i, [C.POINTER(PagedKV), _vp, _vp, _i] + [_vp] * 7 + [_i, _i, _vp, _vp]),
    "uocr_b200_rswa_decode_step_paged": (_i, [C.POINTER(PagedKV)] + [_vp] * 7 + [_i, _i, _i, _vp, _vp, _vp]),
    "uocr_b200_rswa_decode_step_rope_paged": (_i, [C.POINTER(PagedKV)] + [_vp] * 4 + [C.c_float] + [_vp] * 4 +
                                              [_i, _i, _i, _vp, _vp, _vp]),
    "uocr_b200_rswa_attention_batch_paged_noalloc": (_i, [C.POINTER(PagedKV)] + [_vp] * 4 + [_i, _i, _vp, _vp]),
    "uocr_b200_rswa_attention_ragged_f32": (_i, [_vp] * 5 + [_i] * 5 + [_vp, _vp, _vp]),
    "uocr_b200_rswa_attention_ragged_paged": (_i, [C.POINTER(PagedKV)] + [_vp] * 4 + [_i, _i, _vp, _vp, _vp]),
    "uocr_b200_rswa_attention_f32": (_i, [_vp] * 3 + [_i, _vp] + [_i] * 6 + [_vp, _vp, _vp]),
    "uocr_b200_rswa_attention_paged": (_i, [C.POINTER(PagedKV), _i, _vp, _i, _vp, _i, _vp] + [_i] * 4 + [_vp, _vp, _vp]),
    "uocr_b200_rswa_gather_paged": (_i, [C.POINTER(PagedKV)] + [_vp] * 3 + [_i, _i, _vp, _vp, _i, _vp, _vp]),
    "uocr_b200_rswa_gather_heads_paged": (_i, [C.POINTER(PagedKV)] + [_vp] * 3 + [_i, _i, _vp, _vp, _vp, _vp]),
    "uocr_b200_rswa_mass_scratch_bytes": (C.c_size_t, [_i, _i, _i]),
    "uocr_b200_rswa_attention_scored_batch_paged": (_i, [C.POINTER(PagedKV), C.POINTER(ScoreDesc), _vp, _i] + [_vp] * 4 + [_i, _i, _i, _vp, _vp, _vp, _vp]),
    "uocr_b200_rswa_attention_scored_ragged_paged": (_i, [C.POINTER(PagedKV), C.POINTER(ScoreDesc), _vp, _i] + [_vp] * 3 + [_i, _i, _vp, _vp, _vp]),
    "uocr_b200_rswa_prefill_text_scored_paged": (_i, [C.POINTER(PagedKV), _vp, _vp, _i, C.POINTER(ScoreDesc), _vp, _i] + [_vp] * 4 +
                                                 [_i, _i, _i, _vp, _vp, _vp]),
    "uocr_b200_rswa_prefill_attention_scored_tc": (_i, [C.POINTER(PagedKV), _vp, _vp, _i, C.POINTER(ScoreDesc), _vp, _i, _vp, _vp, _i, _i, _i, _vp, _vp, _vp]),
    "uocr_b200_rswa_prefill_plan_scored_tc": (_i, [C.POINTER(ScoreDesc), _vp, _i, _vp, _i, _vp, _vp]),
    "uocr_b200_rswa_evict_select": (_i, [_vp, _i, _vp, _vp, _i, _i, _i, _i, _vp, _vp, _vp, _vp]),
    "uocr_b200_rswa_evict_compact_paged_layers": (_i, [_vp, _i, _vp, _vp, _i, _vp, _i, _vp, _vp, _i, _vp, _vp]),
    "uocr_b200_rswa_evict_publish": (_i, [_vp, _i, _vp, _i, _vp, _i, _vp, _vp, _i, _vp, C.c_longlong, _i, _vp, _i, _vp, _i, _vp, _i, _vp, _vp]),
    "uocr_b200_rope_create": (_i, [C.POINTER(RopeDesc), C.POINTER(_vp)]),
    "uocr_b200_rope_destroy": (_i, [_vp]),
    "uocr_b200_rswa_rope_rows": (_i, [_vp, _vp, _vp, _i64, _vp, _i, _i, _i, _vp]),
    "uocr_b200_rswa_rope_write_prefill_paged": (_i, [C.POINTER(PagedKV), _vp, _vp] + [_vp] * 3 + [_i, _vp, _vp]),
    "uocr_b200_rswa_rope_append_decode_batch_paged": (_i, [C.POINTER(PagedKV), _vp, _vp] + [_vp] * 5 + [_i, _i, _vp, _vp]),
}


_HOST_SYMBOLS = [
    "pool_create", "pool_destroy", "pool_reset", "pool_allocate", "pool_free", "pool_total", "pool_used",
    "pool_peak", "pool_num_free_blocks", "pool_fragmentation",
    "bm_create", "bm_destroy", "bm_acquire_prefix", "bm_release_prefix", "bm_allocate_ring", "bm_free_ring",
    "bm_live_prefixes", "bm_total_prefix_bytes", "bm_shared_prefix_bytes", "bm_peak_prefix_bytes", "bm_get_stats",
    "sched_create", "sched_destroy", "sched_add_request", "sched_build_batch", "sched_mark_prefilled",
    "sched_mark_prefilling", "sched_add_token", "sched_finish", "sched_state", "sched_num_outputs",
    "sched_has_work", "sched_running", "sched_get_stats",
    "cache_create", "cache_set_kv_dtype", "cache_destroy", "cache_reset", "cache_write_prefill",
    "cache_append_decode", "cache_attention", "cache_len", "cache_ring_pos", "cache_ring_started",
    "cache_capacity", "cache_prefill_len", "cache_keys", "cache_values", "cache_bytes",
]


def host_symbols():
    """Entry points of include/uocr_rswa_b200_host.h (host classes behind the C ABI)."""
    return ["uocr_b200_" + n for n in _HOST_SYMBOLS]


def declared_symbols():
    """Names of every function declared in include/uocr_rswa_b200.h (parsed from the header)."""
    import re
    out = []
    for name in ("uocr_rswa_b200.h", "uocr_rswa_b200_host.h"):
        text = open(os.path.join(ROOT, "include", name)).read()
        out += re.findall(r"UOCR_B200_API\s+[\w\s\*]+?\b(uocr_b200_\w+)\s*\(", text)
    return sorted(set(out))


def lib() -> C.CDLL:
    """Load the shared library (never builds it: a missing library is an error on a GPU box)."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(f"{LIB_PATH} is missing: run __graft_entry__.build() first "
                                    "(there is no Python or CPU fallback for the CUDA path)")
        L = C.CDLL(LIB_PATH, mode=os.RTLD_LOCAL)
        for name, (res, args) in _SIGS.items():
            f = getattr(L, name)
            f.restype, f.argtypes = res, args
        _LIB = L
    return _LIB


def check(status: int) -> None:
    if status != 0:
        L = lib()
        raise Error(status, f"{L.uocr_b200_status_string(status).decode()}: {L.uocr_b200_last_error().decode()}")


def _p(t):
    """Device (or host) address of a torch tensor / numpy array / None."""
    if t is None:
        return None
    if hasattr(t, "data_ptr"):
        return t.data_ptr()
    return t.ctypes.data


_current_raw_stream = None  # torch's raw handle of a device's current stream, without building a Stream object


def stream_handle(stream=None, device=None):
    if stream is not None:
        return stream.cuda_stream
    global _current_raw_stream
    if _current_raw_stream is None:
        import torch
        _current_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
    return _current_raw_stream(_current_device() if device is None else device)


class Workspace:
    def __init__(self, max_rows: int):
        h = _vp()
        check(lib().uocr_b200_workspace_create(max_rows, C.byref(h)))
        self.h = h
        self.out_dtype = F32
        self.plan_rows = None  # packed rows of the tile plan with modified scores

    def status(self, stream=None) -> int:
        v = _i(0)
        check(lib().uocr_b200_workspace_status(self.h, stream_handle(stream), C.byref(v)))
        return v.value

    def set_timing(self, enabled: bool) -> None:
        check(lib().uocr_b200_workspace_set_timing(self.h, 1 if enabled else 0))

    def set_out_dtype(self, dtype: int) -> None:
        """F32 (default) or BF16: type of the `out` tensor of every attention call using this workspace."""
        check(lib().uocr_b200_workspace_set_out_dtype(self.h, dtype))
        self.out_dtype = dtype

    def set_overlap(self, enabled: bool) -> None:
        check(lib().uocr_b200_workspace_set_overlap(self.h, 1 if enabled else 0))

    def set_wait_limit(self, polls: int) -> None:
        """Polls a tile wait may take before the warp gives up (0: every wait gives up at once)."""
        check(lib().uocr_b200_workspace_set_wait_limit(self.h, polls))

    def stream_read_gbs(self, stream=None) -> float:
        """Read-only HBM -> shared-memory streaming rate of this GPU in GB/s (bulk copies, one CTA per SM)."""
        v = C.c_double(0)
        check(lib().uocr_b200_workspace_stream_read_gbs(self.h, stream_handle(stream), C.byref(v)))
        return v.value

    def last_kernel_ms(self) -> float:
        v = C.c_float(0)
        check(lib().uocr_b200_workspace_last_kernel_ms(self.h, C.byref(v)))
        return v.value

    def close(self):
        if self.h:
            lib().uocr_b200_workspace_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def host_classes():
    """ctypes table + object wrappers over this library's host classes (MemoryPool, BlockManager,
    ContinuousBatchScheduler, RSWACache): see host_classes.py."""
    import importlib.util
    import sys
    name = "uocr_b200_host_classes"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, os.path.join(HERE, "host_classes.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    lib()  # a missing library is an error
    return sys.modules[name].FunctionTable(LIB_PATH, "uocr_b200")


def launch_count() -> int:
    return int(lib().uocr_b200_launch_count())


class PagedLayer:
    """Device storage of one layer's paged KV plus the descriptor the C ABI takes.  `pools`: K and V
    tensors the caller already holds, [num_blocks, kv_heads, 16, head_dim]; otherwise zero-filled ones are made."""

    def __init__(self, num_blocks, kv_heads, head_dim, dtype, table, device="cuda", pools=None):
        import torch
        self.dtype = dtype
        tdt = torch.bfloat16 if dtype == BF16 else torch.float32
        shape = (num_blocks, kv_heads, BLOCK_TOKENS, head_dim)
        if pools is None:
            pools = tuple(torch.zeros(shape, dtype=tdt, device=device) for _ in range(2))
        for t in pools:
            if tuple(t.shape) != shape or t.dtype != tdt or not t.is_contiguous():
                raise ValueError(f"a pool must be a contiguous {tdt} tensor of shape {shape}")
        self.k, self.v = pools
        self.table = table  # int32 [slots, stride], shared between layers
        self.desc = PagedKV(self.k.data_ptr(), self.v.data_ptr(), table.data_ptr(), table.shape[1],
                            num_blocks, kv_heads, head_dim, dtype)

    def ref(self):
        return C.byref(self.desc)


# ---- thin call wrappers (torch tensors in, status checked) ---------------------------------------

def append_decode_batch_paged(layer, k, v, d_len, d_ring, d_prefill, d_slots, batch, window, ws=None, stream=None):
    check(lib().uocr_b200_rswa_append_decode_batch_paged(layer.ref(), _p(k), _p(v), _p(d_len), _p(d_ring),
                                                          _p(d_prefill), _p(d_slots), batch, window,
                                                          ws.h if ws else None, stream_handle(stream)))


def layer_array(layers):
    """Contiguous array of uocr_b200_paged_kv for the entry points that take several layers at once."""
    arr = (PagedKV * len(layers))()
    for i, lay in enumerate(layers):
        arr[i] = lay.desc
    return arr


def append_decode_batch_paged_layers(layers, k, v, d_len, d_ring, d_prefill, d_slots, batch, window, ws=None, stream=None):
    """All layers of an append step in one launch: k, v are [L][rows >= batch][row], d_len / d_ring [L][slots]."""
    check(lib().uocr_b200_rswa_append_decode_batch_paged_layers(
        layer_array(layers), len(layers), _p(k), _p(v), k.stride(0), _p(d_len), _p(d_ring), d_len.stride(0), _p(d_prefill),
        _p(d_slots), batch, window, ws.h if ws else None, stream_handle(stream)))


def gather_paged_layers(layers, d_len, d_prefill, d_slots, n, capacity_rows, out_k, out_v, out_dtype, ws=None, stream=None):
    """All layers of a gather in one launch: out_k, out_v are [L][n][capacity_rows][row], d_len [L][slots]."""
    check(lib().uocr_b200_rswa_gather_paged_layers(
        layer_array(layers), len(layers), _p(d_len), d_len.stride(0), _p(d_prefill), _p(d_slots), n, capacity_rows,
        _p(out_k), _p(out_v), out_k.stride(0) * out_k.element_size(), out_dtype, ws.h if ws else None, stream_handle(stream)))


def attention_batch_paged(layer, q, d_len, d_prefill, d_slots, batch, heads, out, ws, stream=None):
    check(lib().uocr_b200_rswa_attention_batch_paged(layer.ref(), _p(q), _p(d_len), _p(d_prefill), _p(d_slots),
                                                      batch, heads, _p(out), ws.h, stream_handle(stream)))


def prefill_text_paged(layer, text_k, text_v, text_blocks, q, k, v, d_prefill, d_slots, d_pos, d_block0, total, window,
                       heads, out, ws, stream=None):
    check(lib().uocr_b200_rswa_prefill_text_paged(layer.ref(), _p(text_k), _p(text_v), text_blocks, _p(q), _p(k), _p(v),
                                                   _p(d_prefill), _p(d_slots), _p(d_pos), _p(d_block0), total, window,
                                                   heads, _p(out), ws.h, stream_handle(stream)))


def text_scatter_paged(layer, text_k, text_v, text_blocks, k, v, d_pos, d_block0, total, ws=None, stream=None):
    check(lib().uocr_b200_rswa_text_scatter_paged(layer.ref(), _p(text_k), _p(text_v), text_blocks, _p(k), _p(v),
                                                   _p(d_pos), _p(d_block0), total, ws.h if ws else None,
                                                   stream_handle(stream)))


def text_scatter_fill_paged(layer, text_k, text_v, text_blocks, k, v, d_slots, d_pos, d_block0, d_text_len, d_prefill,
                            d_len, d_ring, total, window, ws=None, stream=None):
    """text scatter + ring fill + cursor publication in one pass."""
    check(lib().uocr_b200_rswa_text_scatter_fill_paged(layer.ref(), _p(text_k), _p(text_v), text_blocks, _p(k), _p(v),
                                                        _p(d_slots), _p(d_pos), _p(d_block0), _p(d_text_len), _p(d_prefill),
                                                        _p(d_len), _p(d_ring), total, window, ws.h if ws else None,
                                                        stream_handle(stream)))


def prefill_attention_tc(layer, text_k, text_v, text_blocks, q, d_prefill, tiles, window, heads, out, ws, stream=None,
                         reuse_plan=False):
    """tiles: int32 numpy array [n, 6] = (row0, rows, slot, kind, pos0, block0) per query tile (host).
    reuse_plan: the workspace already holds the plan of exactly these tiles (prefill_plan_tc, or an earlier call)."""
    import numpy as np
    t = np.ascontiguousarray(tiles, dtype=np.int32)
    check(lib().uocr_b200_rswa_prefill_attention_tc(layer.ref(), _p(text_k), _p(text_v), text_blocks, _p(q),
                                                     _p(d_prefill), None if reuse_plan else t.ctypes.data, t.shape[0], window,
                                                     heads, _p(out), ws.h, stream_handle(stream)))


def prefill_plan_tc(tiles, d_prefill, window, ws, stream=None):
    """Uploads and orders the query tiles once; later prefill_attention_tc(..., reuse_plan=True) calls share the plan."""
    import numpy as np
    t = np.ascontiguousarray(tiles, dtype=np.int32)
    check(lib().uocr_b200_rswa_prefill_plan_tc(t.ctypes.data, t.shape[0], _p(d_prefill), window, ws.h, stream_handle(stream)))
    return lib().uocr_b200_workspace_prefill_plan_serial(ws.h)


def make_prefill_tiles(requests):
    """requests: iterable of (row0, n_rows, slot, kind, pos0, block0); cut into tiles of <= 128 rows."""
    import numpy as np
    out = []
    for row0, n, slot, kind, pos0, block0 in requests:
        for a in range(0, n, 128):
            out.append((row0 + a, min(128, n - a), slot, kind, pos0 + a, block0))
    return np.array(out, dtype=np.int32).reshape(-1, 6)


def ring_fill_paged(layer, text_k, text_v, text_blocks, d_slots, d_pos, d_block0, d_text_len, d_prefill, d_len, d_ring,
                    total, window, ws=None, stream=None):
    check(lib().uocr_b200_rswa_ring_fill_paged(layer.ref(), _p(text_k), _p(text_v), text_blocks, _p(d_slots), _p(d_pos),
                                                _p(d_block0), _p(d_text_len), _p(d_prefill), _p(d_len), _p(d_ring),
                                                total, window, ws.h if ws else None, stream_handle(stream)))


def decode_step_rope_paged(layer, q, k, v, d_positions, theta, d_len, d_ring, d_prefill, d_slots, batch, window, heads,
                           out, ws, stream=None):
    """rope + append + decode attention of one layer in one launch (q, k un-rotated)."""
    check(lib().uocr_b200_rswa_decode_step_rope_paged(layer.ref(), _p(q), _p(k), _p(v), _p(d_positions), float(theta),
                                                       _p(d_len), _p(d_ring), _p(d_prefill), _p(d_slots), batch, window,
                                                       heads, _p(out), ws.h, stream_handle(stream)))


def decode_step_paged(layer, q, k, v, d_len, d_ring, d_prefill, d_slots, batch, window, heads, out, ws, stream=None):
    """append + decode attention of one layer in one launch."""
    check(lib().uocr_b200_rswa_decode_step_paged(layer.ref(), _p(q), _p(k), _p(v), _p(d_len), _p(d_ring),
                                                  _p(d_prefill), _p(d_slots), batch, window, heads, _p(out), ws.h,
                                                  stream_handle(stream)))


def attention_batch_paged_noalloc(layer, q, d_len, d_prefill, d_slots, batch, heads, out, stream=None):
    """Same result as attention_batch_paged, scratch in the library's built-in device array."""
    check(lib().uocr_b200_rswa_attention_batch_paged_noalloc(layer.ref(), _p(q), _p(d_len), _p(d_prefill),
                                                              _p(d_slots), batch, heads, _p(out),
                                                              stream_handle(stream)))


def noalloc_status(stream=None) -> int:
    """Reads and clears the device status word of the allocation-free calls (synchronises the stream)."""
    v = _i(0)
    check(lib().uocr_b200_noalloc_status(stream_handle(stream), C.byref(v)))
    return v.value


def write_prefill_ragged_paged(layer, k, v, d_slots, d_pos, total, ws=None, stream=None):
    check(lib().uocr_b200_rswa_write_prefill_ragged_paged(layer.ref(), _p(k), _p(v), _p(d_slots), _p(d_pos), total,
                                                           ws.h if ws else None, stream_handle(stream)))


def attention_ragged_paged(layer, q, d_prefill, d_slots, d_pos, total, heads, out, ws, stream=None):
    check(lib().uocr_b200_rswa_attention_ragged_paged(layer.ref(), _p(q), _p(d_prefill), _p(d_slots), _p(d_pos),
                                                       total, heads, _p(out), ws.h, stream_handle(stream)))


def attention_paged(layer, slot, q, kv_len, d_len, prefill_len, d_prefill, seq, q_start, heads, causal, out, ws,
                    stream=None):
    check(lib().uocr_b200_rswa_attention_paged(layer.ref(), slot, _p(q), kv_len, _p(d_len), prefill_len,
                                                _p(d_prefill), seq, q_start, heads, 1 if causal else 0, _p(out),
                                                ws.h, stream_handle(stream)))


def gather_paged(layer, d_len, d_prefill, d_slots, n, capacity_rows, out_k, out_v, out_dtype, ws=None, stream=None):
    check(lib().uocr_b200_rswa_gather_paged(layer.ref(), _p(d_len), _p(d_prefill), _p(d_slots), n, capacity_rows,
                                             _p(out_k), _p(out_v), out_dtype, ws.h if ws else None,
                                             stream_handle(stream)))


def gather_heads_paged(layer, d_len, d_prefill, d_slots, n, capacity_rows, out_k, out_v, ws=None, stream=None):
    """fp32 out[n][kv_heads][capacity_rows][head_dim]: the layout of the reference's cache snapshots."""
    check(lib().uocr_b200_rswa_gather_heads_paged(layer.ref(), _p(d_len), _p(d_prefill), _p(d_slots), n, capacity_rows,
                                                   _p(out_k), _p(out_v), ws.h if ws else None, stream_handle(stream)))


def append_decode_batch_f32(k, v, kbase, vbase, d_len, d_ring, d_prefill, d_slots, batch, batch_cap, window,
                            kv_heads, head_dim, stream=None):
    check(lib().uocr_b200_rswa_append_decode_batch_f32(_p(k), _p(v), _p(kbase), _p(vbase), _p(d_len), _p(d_ring),
                                                        _p(d_prefill), _p(d_slots), batch, batch_cap, window,
                                                        kv_heads, head_dim, stream_handle(stream)))


def append_decode_f32(k, v, kcache, vcache, d_len, d_ring, prefill_len, window, kv_heads, head_dim, stream=None):
    check(lib().uocr_b200_rswa_append_decode_f32(_p(k), _p(v), _p(kcache), _p(vcache), _p(d_len), _p(d_ring),
                                                  prefill_len, window, kv_heads, head_dim, stream_handle(stream)))


def write_prefill_ragged_f32(k, v, kbase, vbase, d_slots, d_pos, total, batch_cap, kv_heads, head_dim, stream=None):
    check(lib().uocr_b200_rswa_write_prefill_ragged_f32(_p(k), _p(v), _p(kbase), _p(vbase), _p(d_slots), _p(d_pos),
                                                         total, batch_cap, kv_heads, head_dim, stream_handle(stream)))


def attention_batch_f32(q, kbase, vbase, d_len, d_slots, batch, batch_cap, heads, kv_heads, head_dim, out, ws,
                        stream=None):
    check(lib().uocr_b200_rswa_attention_batch_f32(_p(q), _p(kbase), _p(vbase), _p(d_len), _p(d_slots), batch,
                                                    batch_cap, heads, kv_heads, head_dim, _p(out), ws.h,
                                                    stream_handle(stream)))


def attention_ragged_f32(q, kbase, vbase, d_slots, d_pos, total, batch_cap, heads, kv_heads, head_dim, out, ws,
                         stream=None):
    check(lib().uocr_b200_rswa_attention_ragged_f32(_p(q), _p(kbase), _p(vbase), _p(d_slots), _p(d_pos), total,
                                                     batch_cap, heads, kv_heads, head_dim, _p(out), ws.h,
                                                     stream_handle(stream)))


def attention_f32(q, kcache, vcache, kv_len, d_len, seq, q_start, heads, kv_heads, head_dim, causal, out, ws,
                  stream=None):
    check(lib().uocr_b200_rswa_attention_f32(_p(q), _p(kcache), _p(vcache), kv_len, _p(d_len), seq, q_start, heads,
                                              kv_heads, head_dim, 1 if causal else 0, _p(out), ws.h,
                                              stream_handle(stream)))


# ---- rotary positions --------------------------------------------------------------------------------

_ROPE_LAYOUTS = {"half": 0, "interleaved": 1}
_ROPE_SCALINGS = {"none": 0, "linear": 1, "base": 2, "ramp": 3, "bands": 4}


class Rope:
    """Frequencies of one model (uocr_b200_rope): see the header for the layouts and scalings."""

    def __init__(self, layout="half", rotary_dim=128, theta=10000.0, scaling="none", factor=1.0, orig_context=0.0, low=0.0, high=0.0,
                 amplitude=1.0):
        desc = RopeDesc(_ROPE_LAYOUTS[layout], rotary_dim, _ROPE_SCALINGS[scaling], theta, factor, orig_context, low, high, amplitude)
        h = _vp()
        check(lib().uocr_b200_rope_create(C.byref(desc), C.byref(h)))
        self.h = h

    def __del__(self):
        try:
            lib().uocr_b200_rope_destroy(self.h)
        except Exception:
            pass


_I32 = _FLOAT = _HALF = None  # torch.int32, torch.float32, torch.bfloat16, once torch has been asked for
_device_index = None


def _current_device():
    """Index of the current device: launches go there, so the tensors of a call must be there."""
    if _device_index is None:
        _load_torch()
    return _device_index()


def _load_torch():
    global _I32, _FLOAT, _HALF, _device_index
    import torch
    _I32, _FLOAT, _HALF = torch.int32, torch.float32, torch.bfloat16
    _device_index = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _dp(t):
    """Device address of a tensor / None (the light form of _p for calls that are short themselves)."""
    return None if t is None else t.data_ptr()


def _dtype_of(t):
    dt = t.dtype
    if dt is _FLOAT:
        return F32
    if dt is _HALF:
        return BF16
    raise ArgumentError(f"rows must be float32 or bfloat16, got {dt}")


def _refuse(t, dtype, n, dev, name):
    """The error for a tensor that is not what `_array` or `_ints` wants."""
    return ArgumentError(f"{name}: wanted at least {n} contiguous {dtype} on cuda:{dev}, got {t.numel()} {t.dtype} {'contiguous' if t.is_contiguous() else 'strided'} on {t.device}")


def _array(t, dtype, n, dev, name):
    """Address of a contiguous tensor of at least n elements of the type (None passes: the library says where it wants one)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() < n or not t.is_contiguous() or t.get_device() != dev:
        raise _refuse(t, dtype, n, dev, name)
    return t.data_ptr()


def _ints(t, n, dev, name):
    if t is None:
        return None
    if t.dtype is not _I32 or t.numel() < n or not t.is_contiguous() or t.get_device() != dev:
        raise _refuse(t, _I32, n, dev, name)
    return t.data_ptr()


def _slot_ints(t, dev, name):
    """The same for one integer per slot, however many slots there are (an empty tensor has no address, which the library refuses)."""
    if t is None:
        return None
    if t.dtype is not _I32 or not t.is_contiguous() or t.get_device() != dev:
        raise _refuse(t, _I32, 1, dev, name)
    return t.data_ptr()


def _grid(t, dtype, rows, dev, name):
    """(address, width) of a contiguous [at least `rows`][width] matrix of the type; (None, 0) for None."""
    if t is None:
        return None, 0
    shape = t.shape
    if len(shape) != 2 or shape[0] < rows:
        raise ArgumentError(f"{name}: wanted a matrix of at least {rows} rows, got {tuple(shape)}")
    if t.dtype is not dtype or not t.is_contiguous() or t.get_device() != dev:
        raise _refuse(t, dtype, 0, dev, name)
    return t.data_ptr(), shape[1]


def _row_stride(t, dtype, n, width, dev):
    """Elements between the rows of t: an [n, width or more] matrix of the type on the device with contiguous rows."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != n or shape[1] < width or stride[1] != 1 or t.dtype is not dtype or t.get_device() != dev:
        raise ArgumentError(f"rows must be [{n}, at least {width}] {dtype} on cuda:{dev} with contiguous elements, got {tuple(shape)} {t.dtype} on {t.device}, strides {stride}")
    return stride[0] if n > 1 else width


_QKV_ROWS = struct.Struct("PPPPqqqqii")  # QkvRows (packing is a fifth of the time that filling a ctypes structure takes)


def _addr(t):
    return 0 if t is None else t.data_ptr()


def _qkv_rows(q, k, v, q_out, heads, kv_heads, head_dim, n, dev):
    """Packed rows, [n, width] each with its own row stride, as the bytes of a QkvRows; and the stride of k."""
    ref = q if q is not None else k
    dt = ref.dtype
    q_width, kv_width = heads * head_dim, kv_heads * head_dim
    qs = ks = vs = os = 0
    if q is not None:
        qs = _row_stride(q, dt, n, q_width, dev)
        if q_out is not None:
            os = qs if q_out is q else _row_stride(q_out, dt, n, q_width, dev)
    if k is not None:
        ks = _row_stride(k, dt, n, kv_width, dev)
        if v is not None:
            vs = _row_stride(v, dt, n, kv_width, dev)
    return _QKV_ROWS.pack(_addr(q), _addr(k), _addr(v), _addr(q_out), qs, ks, vs, os, _dtype_of(ref), heads), ks


def rope_rows(rope, q, k, q_out, k_out, d_positions, heads, kv_heads, head_dim, stream=None):
    """Rotates the packed rows of q and k (either may be None with 0 heads; outputs may be the inputs)."""
    n, dev = (q if q is not None else k).shape[0], _current_device()
    rows, k_stride = _qkv_rows(q, k, None, q_out, heads, kv_heads, head_dim, n, dev)
    if k_out is not None and k_out is not k:
        k_stride = _row_stride(k_out, (k if k is not None else k_out).dtype, n, kv_heads * head_dim, dev)
    check(lib().uocr_b200_rswa_rope_rows(rope.h, rows, _dp(k_out), k_stride, _ints(d_positions, n, dev, "d_positions"), n, kv_heads, head_dim,
                                         stream_handle(stream, dev)))


def _kv_rows(layer, q, k, v, q_out, heads, dev):
    """The rows of a call that writes K and V to the layer, and their count."""
    d, n = layer.desc, k.shape[0]
    if layer.k.get_device() != dev:
        raise ArgumentError(f"the layer is on {layer.k.device}, the current device is cuda:{dev}")
    return _qkv_rows(q, k, v, q_out, heads, d.kv_heads, d.head_dim, n, dev)[0], n


def rope_write_prefill_paged(layer, rope, q, k, v, q_out, d_positions, d_slots, d_pos, heads, ws=None, stream=None):
    """rope + write_prefill_ragged_paged in one pass."""
    dev = _current_device()
    rows, n = _kv_rows(layer, q, k, v, q_out, heads, dev)
    check(lib().uocr_b200_rswa_rope_write_prefill_paged(
        layer.desc, rope.h, rows, _ints(d_positions, n, dev, "d_positions"), _ints(d_slots, n, dev, "d_slots"), _ints(d_pos, n, dev, "d_pos"), n,
        ws.h if ws else None, stream_handle(stream, dev)))


def rope_append_decode_batch_paged(layer, rope, q, k, v, q_out, d_positions, d_len, d_ring, d_prefill, d_slots, window, heads, ws=None,
                                   stream=None):
    """rope + append_decode_batch_paged in one pass."""
    dev = _current_device()
    rows, n = _kv_rows(layer, q, k, v, q_out, heads, dev)
    check(lib().uocr_b200_rswa_rope_append_decode_batch_paged(
        layer.desc, rope.h, rows, _ints(d_positions, n, dev, "d_positions"), _slot_ints(d_len, dev, "d_len"), _slot_ints(d_ring, dev, "d_ring"),
        _slot_ints(d_prefill, dev, "d_prefill"), _ints(d_slots, n, dev, "d_slots"), n, window, ws.h if ws else None, stream_handle(stream, dev)))


# ---- attention with modified scores --------------------------------------------------------------------

class Score:
    """Scale, cap, distance bias and visible ranges of one call (uocr_b200_score); keeps its tensors alive."""

    def __init__(self, scale=0.0, softcap=0.0, slopes=None, d_q_pos=None, d_key_pos=None, d_lo=None, d_hi=None):
        import torch
        for t, dt in ((slopes, torch.float32), (d_q_pos, torch.int32), (d_key_pos, torch.int32), (d_lo, torch.int32), (d_hi, torch.int32)):
            if t is not None and (t.dtype != dt or not t.is_contiguous()):
                raise ArgumentError(f"expected a contiguous {dt} tensor")
        self.keep = (slopes, d_q_pos, d_key_pos, d_lo, d_hi)
        self.desc = ScoreDesc(scale, softcap, _p(slopes), _p(d_q_pos), _p(d_key_pos), d_key_pos.shape[1] if d_key_pos is not None else 0,
                              _p(d_lo), _p(d_hi))
        # what a call may read: rows and heads its tensors reach (None: no limit), and their device
        self.rows = min((t.numel() for t in (d_q_pos if slopes is not None else None, d_lo, d_hi) if t is not None), default=None)
        self.heads = slopes.numel() if slopes is not None else None
        self.device = _one_device(self.keep)


def _one_device(tensors):
    """Index of the device all of them are on; None for none."""
    found = {t.get_device() for t in tensors if t is not None}
    if len(found) > 1:
        raise ArgumentError("the tensors are on different devices")
    return found.pop() if found else None


class Mass:
    """Accumulated attention weights of the fixed region, [slots, stride] (uocr_b200_mass), with scratch for `batch` rows."""

    def __init__(self, mass_in, mass_out, batch, heads, decay=1.0):
        import torch
        for t in (mass_in, mass_out):
            if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.shape != mass_out.shape):
                raise ArgumentError("the mass must be contiguous float32, [slots, stride]")
        stride = mass_out.shape[1]
        n = lib().uocr_b200_rswa_mass_scratch_bytes(batch, heads, stride)
        self.scratch = torch.empty(n, dtype=torch.uint8, device=mass_out.device)
        self.keep = (mass_in, mass_out)
        self.desc = MassDesc(_p(mass_in), _p(mass_out), stride, decay, _p(self.scratch), n)
        self.device = _one_device(self.keep)


def _scored(layer, score, q, rows, heads, out, ws, dev):
    """Addresses of q and out and q's type, for a call of `rows` rows."""
    if (score.rows is not None and rows > score.rows) or (score.heads is not None and heads > score.heads):
        raise ArgumentError(f"the score's tensors are for {score.rows} rows and {score.heads} heads, the call has {rows} and {heads}")
    if (score.device is not None and score.device != dev) or layer.k.get_device() != dev:
        raise ArgumentError(f"score and layer must be on the current device, cuda:{dev}")
    dt, n = _dtype_of(q), rows * heads * layer.desc.head_dim
    return _array(q, q.dtype, n, dev, "q"), dt, _array(out, _HALF if ws.out_dtype == BF16 else _FLOAT, n, dev, "out")


def attention_scored_batch_paged(layer, score, q, d_len, d_ring, d_prefill, d_slots, batch, window, heads, out, ws, mass=None, stream=None):
    """Decode attention with modified scores; `mass` also accumulates the attention weights."""
    dev = _current_device()
    q, dt, out = _scored(layer, score, q, batch, heads, out, ws, dev)
    if mass is not None and mass.device != dev:
        raise ArgumentError(f"the mass must be on the current device, cuda:{dev}")
    check(lib().uocr_b200_rswa_attention_scored_batch_paged(
        layer.desc, score.desc, q, dt, _slot_ints(d_len, dev, "d_len"), _slot_ints(d_ring, dev, "d_ring"), _slot_ints(d_prefill, dev, "d_prefill"),
        _ints(d_slots, batch, dev, "d_slots"), batch, window, heads, out, C.addressof(mass.desc) if mass is not None else None, ws.h, stream_handle(stream, dev)))


def attention_scored_ragged_paged(layer, score, q, d_prefill, d_slots, d_pos, total, heads, out, ws, stream=None):
    """Packed vision rows with modified scores, any geometry."""
    dev = _current_device()
    q, dt, out = _scored(layer, score, q, total, heads, out, ws, dev)
    check(lib().uocr_b200_rswa_attention_scored_ragged_paged(
        layer.desc, score.desc, q, dt, _slot_ints(d_prefill, dev, "d_prefill"), _ints(d_slots, total, dev, "d_slots"), _ints(d_pos, total, dev, "d_pos"), total,
        heads, out, ws.h, stream_handle(stream, dev)))


def _text_pools(layer, text_k, text_v, text_blocks, dev):
    n = max(text_blocks, 0) * layer.desc.kv_heads * BLOCK_TOKENS * layer.desc.head_dim
    return _array(text_k, layer.k.dtype, n, dev, "text_k"), _array(text_v, layer.k.dtype, n, dev, "text_v")


def prefill_text_scored_paged(layer, text_k, text_v, text_blocks, score, q, d_prefill, d_slots, d_pos, d_block0, total, window, heads, out, ws,
                              stream=None):
    """Packed text rows over prefix + text window with modified scores, any geometry (K and V already in the text pool)."""
    dev = _current_device()
    q, dt, out = _scored(layer, score, q, total, heads, out, ws, dev)
    text_k, text_v = _text_pools(layer, text_k, text_v, text_blocks, dev)
    check(lib().uocr_b200_rswa_prefill_text_scored_paged(
        layer.desc, text_k, text_v, text_blocks, score.desc, q, dt, _slot_ints(d_prefill, dev, "d_prefill"), _ints(d_slots, total, dev, "d_slots"),
        _ints(d_pos, total, dev, "d_pos"), _ints(d_block0, total, dev, "d_block0"), total, window, heads, out, ws.h, stream_handle(stream, dev)))


def _tiles(tiles):
    """The query tiles as the library takes them, and the packed rows they reach."""
    import numpy as np
    t = np.ascontiguousarray(tiles, dtype=np.int32)
    if t.ndim != 2 or t.shape[1] != 6:
        raise ArgumentError(f"tiles must be [n, 6], got {t.shape}")
    return t, int((t[:, 0].astype(np.int64) + t[:, 1]).max(initial=0))


def prefill_plan_scored_tc(score, tiles, d_prefill, window, ws, stream=None):
    """Uploads and orders the query tiles for the score's visible ranges; later calls with reuse_plan=True share the plan."""
    dev = _current_device()
    t, rows = _tiles(tiles)
    if (score.rows is not None and rows > score.rows) or (score.device is not None and score.device != dev):
        raise ArgumentError(f"the score's tensors are for {score.rows} rows on device {score.device}, the tiles reach {rows} on cuda:{dev}")
    ws.plan_rows = max(rows, ws.plan_rows or 0)  # until the call has succeeded: the library may hold the old plan or the new one
    check(lib().uocr_b200_rswa_prefill_plan_scored_tc(score.desc, t.ctypes.data, t.shape[0], _slot_ints(d_prefill, dev, "d_prefill"), window, ws.h,
                                                      stream_handle(stream, dev)))
    ws.plan_rows = rows


def prefill_attention_scored_tc(layer, text_k, text_v, text_blocks, score, q, d_prefill, tiles, window, heads, out, ws, stream=None, reuse_plan=False):
    """prefill_attention_tc with modified scores; q fp32 or bf16."""
    dev = _current_device()
    t, rows = (tiles, ws.plan_rows) if reuse_plan and ws.plan_rows is not None else _tiles(tiles)  # the rows of a reused plan are the plan's
    q, dt, out = _scored(layer, score, q, rows, heads, out, ws, dev)
    text_k, text_v = _text_pools(layer, text_k, text_v, text_blocks, dev)
    if not reuse_plan:
        ws.plan_rows = max(rows, ws.plan_rows or 0)
    check(lib().uocr_b200_rswa_prefill_attention_scored_tc(
        layer.desc, text_k, text_v, text_blocks, score.desc, q, dt, _slot_ints(d_prefill, dev, "d_prefill"), None if reuse_plan else t.ctypes.data, len(t),
        window, heads, out, ws.h, stream_handle(stream, dev)))
    if not reuse_plan:
        ws.plan_rows = rows


# ---- eviction from the fixed region ----------------------------------------------------------------------

def evict_select(mass, d_prefill, d_slots, n, keep, sinks, recent, d_keep, d_keep_len, ws=None, stream=None):
    """The `keep` heaviest tokens of each slot's fixed region, ascending: d_keep int32 [n, keep], d_keep_len int32 [n].  Protected tokens
    that do not all fit (keep < sinks + recent) are kept from the front."""
    dev = _current_device()
    mass, stride = _grid(mass, _FLOAT, 1, dev, "mass")
    check(lib().uocr_b200_rswa_evict_select(
        mass, stride, _slot_ints(d_prefill, dev, "d_prefill"), _ints(d_slots, n, dev, "d_slots"), n, keep, sinks, recent,
        _ints(d_keep, n * keep, dev, "d_keep"), _ints(d_keep_len, n, dev, "d_keep_len"), ws.h if ws else None, stream_handle(stream, dev)))


def evict_compact_paged_layers(layers, d_prefill, d_slots, n, d_keep, d_keep_len, d_new_blocks=None, ws=None, stream=None):
    """Moves the kept rows of every layer to the new blocks (None: in place).  layers: PagedLayers, or their layer_array."""
    dev = _current_device()
    if isinstance(layers, C.Array):
        arr = layers
    else:
        arr = layer_array(layers)
        if any(lay.k.get_device() != dev for lay in layers):
            raise ArgumentError(f"the layers must be on the current device, cuda:{dev}")
    keep, width = _grid(d_keep, _I32, n, dev, "d_keep")
    new, new_width = _grid(d_new_blocks, _I32, n, dev, "d_new_blocks")
    check(lib().uocr_b200_rswa_evict_compact_paged_layers(
        arr, len(arr), _slot_ints(d_prefill, dev, "d_prefill"), _ints(d_slots, n, dev, "d_slots"), n, keep, width, _ints(d_keep_len, n, dev, "d_keep_len"), new,
        new_width, ws.h if ws else None, stream_handle(stream, dev)))


def evict_publish(table, d_slots, n, d_keep, d_keep_len, d_len, d_prefill, window, d_new_blocks=None, mass=None, d_key_pos=None, ws=None,
                  stream=None):
    """Puts the new regions in force: table rows, d_len [layers, slots], d_prefill, and the per-token arrays."""
    dev = _current_device()
    table, table_width = _grid(table, _I32, 1, dev, "table")
    keep, width = _grid(d_keep, _I32, n, dev, "d_keep")
    new, new_width = _grid(d_new_blocks, _I32, n, dev, "d_new_blocks")
    mass, mass_width = _grid(mass, _FLOAT, 1, dev, "mass")
    key_pos, pos_width = _grid(d_key_pos, _I32, 1, dev, "d_key_pos")
    if d_len.dim() != 2 or (d_len.size(1) > 1 and d_len.stride(1) != 1) or d_len.dtype is not _I32 or d_len.get_device() != dev:
        raise ArgumentError(f"d_len must be [layers, slots] int32 on cuda:{dev} with contiguous rows, got {tuple(d_len.shape)} {d_len.dtype} on {d_len.device}")
    check(lib().uocr_b200_rswa_evict_publish(
        table, table_width, _ints(d_slots, n, dev, "d_slots"), n, keep, width, _ints(d_keep_len, n, dev, "d_keep_len"), new, new_width, d_len.data_ptr(),
        d_len.stride(0), d_len.size(0), _slot_ints(d_prefill, dev, "d_prefill"), window, mass, mass_width, key_pos, pos_width, ws.h if ws else None,
        stream_handle(stream, dev)))
