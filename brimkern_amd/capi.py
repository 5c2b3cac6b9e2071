"""ctypes binding of ``libbrik.so`` (the C ABI in ``include/brik.h``).

This is the Python-side host of the drop-in boundary (tests, bench, smoke); the JavaScript host is
``brimkern_amd/js`` over the N-API addon. Both call the same C entry points. Nothing here falls
back to CPU: if the library is missing or no gfx950 device is present, construction raises.
"""
from __future__ import annotations

import ctypes
import os

import numpy as np

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "libbrik.so")

BRIK_OK, BRIK_EINVAL, BRIK_EALIGN, BRIK_EHIP, BRIK_ENOMEM, BRIK_ENODEV, BRIK_EMODULE = 0, -1, -2, -3, -4, -5, -6
BRIK_EVALID = -7
BRIK_OPT_PATH, BRIK_OPT_GEMV_VARIANT = 1, 2
BRIK_GEMV_VARIANTS = 11
BRIK_OPT_GEMM_TILE, BRIK_GEMM_TILES = 3, 23
BRIK_OPT_PLAN_STAGE, BRIK_OPT_PLAN_SETS, BRIK_OPT_SPLITK, BRIK_OPT_GEMV_BLOCKS = 4, 5, 6, 7
BRIK_OPT_ATTN_ROWS, BRIK_OPT_ATTN_SPLITS = 8, 9
BRIK_OPT_I8_KERNEL, BRIK_OPT_I8_SPLITS = 10, 11
PATH_AUTO, PATH_GEMV, PATH_GEMM = 0, 1, 2
BRIK_PATH_GEMV, BRIK_PATH_GEMV_STAGED, BRIK_PATH_TILED, BRIK_PATH_SPLITK = 1, 2, 3, 4

# every exported symbol of include/brik.h with (restype, argtypes)
_P, _I, _Z, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.POINTER(ctypes.c_float)
SIGNATURES = {
    "brik_create": (_I, [_I, ctypes.POINTER(_P)]),
    "brik_destroy": (None, [_P]),
    "brik_last_error": (ctypes.c_char_p, [_P]),
    "brik_last_path": (_I, [_P]),
    "brik_last_kernel": (ctypes.c_char_p, [_P]),
    "brik_strerror": (ctypes.c_char_p, [_I]),
    "brik_device_count": (_I, [ctypes.POINTER(_I)]),
    "brik_alloc": (_I, [_P, _Z, ctypes.POINTER(_P)]),
    "brik_free": (_I, [_P, _P]),
    "brik_h2d": (_I, [_P, _P, _P, _Z]),
    "brik_d2h": (_I, [_P, _P, _P, _Z]),
    "brik_d2d": (_I, [_P, _P, _P, _Z]),
    "brik_h2d_async": (_I, [_P, _P, _P, _Z]),
    "brik_sync": (_I, [_P]),
    "brik_fence_record": (_I, [_P, ctypes.POINTER(_P)]),
    "brik_fence_d2h": (_I, [_P, _P, _P, _Z]),
    "brik_fence_error": (ctypes.c_char_p, [_P]),
    "brik_fence_destroy": (None, [_P]),
    "brik_self_validate": (_I, [_P, ctypes.c_char_p, _Z]),
    "brik_matmul_t_q8": (_I, [_P, _P, _P, _P, _P, _I, _I, _I]),
    "brik_matmul_t_q4": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I]),
    "brik_matmul_t_q3": (_I, [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I]),
    "brik_matmul_t_q4_noalloc": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I]),
    "brik_moe_matmul_t_q4": (_I, [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I]),
    "brik_moe_matmul_t_q4_x2": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I]),
    "brik_dequant_q8_f32": (_I, [_P, _P, _P, _P, _Z]),
    "brik_dequant_q4_f32": (_I, [_P, _P, _P, _P, _P, _Z]),
    "brik_dequant_q3_f32": (_I, [_P, _P, _P, _P, _P, _P, _Z]),
    "brik_quantize_q8": (_I, [_P, _P, _P, _P, _Z]),
    "brik_quantize_q4": (_I, [_P, _P, _P, _P, _P, _Z]),
    "brik_quantize_q3": (_I, [_P, _P, _P, _P, _P, _P, _Z]),
    "brik_f16_to_f32": (_I, [_P, _P, _P, _Z]),
    "brik_matmul_t_f16w": (_I, [_P, _P, _P, _P, _I, _I, _I]),
    "brik_conv2d_q8": (_I, [_P, _P, _P, _P, _P, _P] + [_I] * 8),
    "brik_conv2d_q4": (_I, [_P, _P, _P, _P, _P, _P, _P] + [_I] * 8),
    "brik_timer_begin": (_I, [_P]),
    "brik_timer_end": (_I, [_P, _F]),
    "brik_set_option": (_I, [_P, _I, _I]),
    "brik_gemv_plan_create": (_I, [_P, _I, _P, _I, ctypes.POINTER(_P)]),
    "brik_gemv_plan_run": (_I, [_P, _P]),
    "brik_gemv_plan_destroy": (None, [_P, _P]),
    "brik_gemv_plan_create_ex": (_I, [_P, _I, _P, _I, ctypes.POINTER(_P)]),
    "brik_gemv_plan_create_glu": (_I, [_P, _I, _P, _P, _P, ctypes.POINTER(_P), ctypes.POINTER(_P)]),
    "brik_graph_begin": (_I, [_P]),
    "brik_graph_end": (_I, [_P, ctypes.POINTER(_P)]),
    "brik_graph_launch": (_I, [_P, _P]),
    "brik_graph_destroy": (None, [_P, _P]),
    "brik_logits_topk": (_I, [_P, _P, _I, _P, _I, ctypes.c_float, ctypes.c_float, _I, _P, _P]),
    "brik_lm_head_topk_q8": (_I, [_P, _P, _P, _P, _I, _I, _P, _I, ctypes.c_float, ctypes.c_float, _I, _P, _P]),
    "brik_lm_head_topk_q4": (_I, [_P, _P, _P, _P, _P, _I, _I, _P, _I, ctypes.c_float, ctypes.c_float, _I, _P, _P]),
    "brik_lm_head_topk_q3": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _P, _I, ctypes.c_float, ctypes.c_float, _I, _P,
                                  _P]),
    "brik_qk_norm_rope": (_I, [_P, _P, _P]),
    "brik_kv_write": (_I, [_P, _P, _P, _P]),
    "brik_kv_read": (_I, [_P, _P, _P, _P, _P]),
    "brik_attention": (_I, [_P, _P, _P, _P]),
    "brik_moe_route": (_I, [_P, _P]),
    "brik_moe_route_grad": (_I, [_P, _P, _P, _P]),
    "brik_moe_sort": (_I, [_P, _P, _I, _I, _I, _P, _P, _P]),
    "brik_moe_dispatch": (_I, [_P, _P, _P, _P, _P, _I, _I, _I]),
    "brik_moe_combine": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I]),
    "brik_moe_combine_grad": (_I, [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I]),
    "brik_quantize_i8": (_I, [_P, _P, ctypes.c_int64, _P, ctypes.c_int64, _I, _P, _P, _I, _I]),
    "brik_matmul_t_i8": (_I, [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I]),
    "brik_moe_matmul_t_i8": (_I, [_P, _P, _P, _I, _P, _I, _P, _P, _P, _P, _I, _I, _I, _I]),
}
BRIK_TOPK_MAX = 64
BRIK_NOALLOC_SCRATCH_BYTES = 16 << 20
BRIK_STAGING_RING_BYTES = 32 << 20

FMT_CODES = {"q8": 8, "q4": 4, "q3": 3}


class GemvJob(ctypes.Structure):
    """``brik_gemv_job`` of include/brik.h."""
    _fields_ = [("x", _P), ("p0", _P), ("p1", _P), ("scales", _P), ("mins", _P), ("y", _P),
                ("K", ctypes.c_int32), ("N", ctypes.c_int32)]


class GemvJobEx(ctypes.Structure):
    """``brik_gemv_job_ex`` of include/brik.h (fused input transform and residual)."""
    _fields_ = [("job", GemvJob), ("gate", _P), ("norm_w", _P), ("res", _P), ("eps", ctypes.c_float),
                ("flags", ctypes.c_int32)]


BRIK_JOB_GAIN_ONE_PLUS, BRIK_JOB_ACT_GELU = 1, 2


_I32, _I64, _F32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class KvCache(ctypes.Structure):
    """``brik_kv_cache`` of include/brik.h."""
    _fields_ = [("fmt", _I32), ("heads", _I32), ("head_dim", _I32), ("page", _I32), ("pages", _I32), ("reserved", _I32),
                ("k", _P), ("v", _P), ("k_scales", _P), ("v_scales", _P), ("k_mins", _P), ("v_mins", _P)]


class KvBatch(ctypes.Structure):
    """``brik_kv_batch`` of include/brik.h."""
    _fields_ = [("seqs", _I32), ("rows", _I32), ("row_off", _P), ("kv_len", _P), ("table", _P), ("table_cols", _I32),
                ("max_len", _I32), ("max_rows", _I32), ("prefix_len", _I32), ("prefix_table", _P)]


class QkvRows(ctypes.Structure):
    """``brik_qkv_rows`` of include/brik.h."""
    _fields_ = [("q", _P), ("k", _P), ("v", _P), ("q_out", _P), ("k_out", _P), ("q_stride", _I64), ("k_stride", _I64),
                ("v_stride", _I64), ("q_out_stride", _I64), ("k_out_stride", _I64), ("q_norm", _P), ("k_norm", _P),
                ("inv_freq", _P), ("positions", _P), ("heads", _I32), ("kv_heads", _I32), ("head_dim", _I32),
                ("rot_dim", _I32), ("flags", _I32), ("eps", _F32)]


class AttnArgs(ctypes.Structure):
    """``brik_attn_args`` of include/brik.h."""
    _fields_ = [("q", _P), ("out", _P), ("q_stride", _I64), ("out_stride", _I64), ("heads", _I32), ("window", _I32),
                ("scale", _F32), ("softcap", _F32)]


BRIK_QKV_GAIN_ONE_PLUS, BRIK_QKV_INTERLEAVED = 1, 2


class MoeRouteArgs(ctypes.Structure):
    """``brik_moe_route_args`` of include/brik.h."""
    _fields_ = [("logits", _P), ("bias", _P), ("logit_stride", _I64), ("ids", _P), ("weights", _P), ("row_off", _P), ("src", _P),
                ("slot", _P), ("tokens", _I32), ("experts", _I32), ("k", _I32), ("flags", _I32), ("scale", _F32), ("reserved", _I32)]


BRIK_ROUTE_SIGMOID, BRIK_ROUTE_RENORM = 1, 2
BRIK_MOE_EXPERTS, BRIK_MOE_K, BRIK_I8_K = 1024, 64, 131040


class BrikError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"brik error {code}: {msg}")
        self.code = code


_lib = None


def load_library(path: str = LIB_PATH):
    """Load libbrik.so and declare every entry point. Raises if it was never built."""
    global _lib
    if _lib is None:
        if not os.path.exists(path):
            raise ImportError(f"{path} is missing: run `python -m brimkern_amd.build` (no CPU fallback exists)")
        lib = ctypes.CDLL(path)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def device_count() -> int:
    n = ctypes.c_int(0)
    load_library().brik_device_count(ctypes.byref(n))
    return n.value


class DeviceBuffer:
    """A device allocation owned by a :class:`Context`."""

    __slots__ = ("ctx", "ptr", "nbytes")

    def __init__(self, ctx: "Context", ptr: int, nbytes: int):
        self.ctx, self.ptr, self.nbytes = ctx, ptr, nbytes

    def offset(self, nbytes: int) -> int:
        """Raw device address ``nbytes`` into the buffer (for plane views into a packed blob)."""
        assert 0 <= nbytes <= self.nbytes
        return self.ptr + nbytes

    def free(self):
        if self.ptr:
            self.ctx._check(self.ctx.lib.brik_free(self.ctx.handle, _P(self.ptr)))
            self.ptr = 0

    def __int__(self):
        return self.ptr


def _addr(p) -> _P:
    if p is None:
        return _P(None)
    if isinstance(p, DeviceBuffer):
        return _P(p.ptr)
    return _P(int(p))


def _i32(*sizes):
    """The sizes of a call, refused where 32 bits do not hold them (ctypes would cut them off)."""
    for v in sizes:
        if not -(1 << 31) <= v < 1 << 31:
            raise BrikError(BRIK_EINVAL, f"{v} is no 32-bit integer")
    return sizes


class Context:
    """One device + one stream (``brik_ctx``)."""

    def __init__(self, device: int = 0):
        self.lib = load_library()
        h = _P()
        rc = self.lib.brik_create(device, ctypes.byref(h))
        if rc != BRIK_OK:
            raise BrikError(rc, f"brik_create({device}): {self.lib.brik_strerror(rc).decode()}")
        self.handle = h
        self._buffers = []

    def _check(self, rc: int):
        if rc != BRIK_OK:
            raise BrikError(rc, self.lib.brik_last_error(self.handle).decode())
        return rc

    def close(self):
        if getattr(self, "handle", None):
            for b in self._buffers:
                b.free()
            self._buffers.clear()
            self.lib.brik_destroy(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- memory -----------------------------------------------------------------------
    def alloc(self, nbytes: int) -> DeviceBuffer:
        p = _P()
        self._check(self.lib.brik_alloc(self.handle, max(int(nbytes), 1), ctypes.byref(p)))
        b = DeviceBuffer(self, p.value, int(nbytes))
        self._buffers.append(b)
        return b

    def free(self, buf: DeviceBuffer):
        buf.free()
        if buf in self._buffers:
            self._buffers.remove(buf)

    def upload(self, arr: np.ndarray) -> DeviceBuffer:
        a = np.ascontiguousarray(arr)
        b = self.alloc(a.nbytes)
        self.h2d(b, a)
        return b

    def h2d(self, dst, arr: np.ndarray, dst_offset: int = 0):
        a = np.ascontiguousarray(arr)
        self._check(self.lib.brik_h2d(self.handle, _P(int(_addr(dst).value or 0) + dst_offset),
                                      _P(a.ctypes.data), a.nbytes))

    def h2d_async(self, dst, arr: np.ndarray, dst_offset: int = 0):
        """Upload without waiting for earlier work (brik_h2d_async): ``arr`` may change on return."""
        a = np.ascontiguousarray(arr)
        self._check(self.lib.brik_h2d_async(self.handle, _P(int(_addr(dst).value or 0) + dst_offset),
                                            _P(a.ctypes.data), a.nbytes))

    def download(self, src, dtype, count: int, src_offset: int = 0) -> np.ndarray:
        out = np.empty(count, dtype=dtype)
        self._check(self.lib.brik_d2h(self.handle, _P(out.ctypes.data),
                                      _P(int(_addr(src).value or 0) + src_offset), out.nbytes))
        return out

    def sync(self):
        self._check(self.lib.brik_sync(self.handle))

    def fence(self) -> "Fence":
        """Mark the current end of the stream (brik_fence_record)."""
        h = _P()
        self._check(self.lib.brik_fence_record(self.handle, ctypes.byref(h)))
        return Fence(self, h)

    def self_validate(self):
        """The load-time kernel checks (brik_self_validate): returns None when every check passes, else
        the name of the first failing check (BRIK_EVALID); other errors raise."""
        buf = ctypes.create_string_buffer(64)
        rc = self.lib.brik_self_validate(self.handle, buf, 64)
        if rc == BRIK_EVALID:
            return buf.value.decode()
        self._check(rc)
        return None

    def set_option(self, key: int, value: int):
        self._check(self.lib.brik_set_option(self.handle, key, value))

    def last_path(self) -> int:
        """BRIK_PATH_* of the last matmul call on this context (0 before any, or for K = 0)."""
        return self.lib.brik_last_path(self.handle)

    def last_kernel(self) -> str:
        """The product kernel of the last matmul or convolution, by the stem of its name (brik_last_kernel)."""
        return self.lib.brik_last_kernel(self.handle).decode()

    def timer_begin(self):
        self._check(self.lib.brik_timer_begin(self.handle))

    def timer_end(self) -> float:
        ms = ctypes.c_float(0)
        self._check(self.lib.brik_timer_end(self.handle, ctypes.byref(ms)))
        return ms.value

    # ---- compute (device pointers, enqueue only) -------------------------------------------
    def matmul_t_q8(self, x, codes, sc, y, M, K, N):
        self._check(self.lib.brik_matmul_t_q8(self.handle, _addr(x), _addr(codes), _addr(sc), _addr(y), M, K, N))

    def matmul_t_q4(self, x, nib, sc, mn, y, M, K, N):
        self._check(self.lib.brik_matmul_t_q4(self.handle, _addr(x), _addr(nib), _addr(sc), _addr(mn),
                                              _addr(y), M, K, N))

    def matmul_t_q4_noalloc(self, x, nib, sc, mn, y, M, K, N):
        """:meth:`matmul_t_q4` on the library's fixed per-device scratch: no device allocation."""
        self._check(self.lib.brik_matmul_t_q4_noalloc(self.handle, _addr(x), _addr(nib), _addr(sc), _addr(mn),
                                                      _addr(y), M, K, N))

    def matmul_t_q3(self, x, lo, hi, sc, mn, y, M, K, N):
        self._check(self.lib.brik_matmul_t_q3(self.handle, _addr(x), _addr(lo), _addr(hi), _addr(sc),
                                              _addr(mn), _addr(y), M, K, N))

    def moe_matmul_t_q4(self, x, row_off, nib, sc, mn, y, E, R, K, N):
        self._check(self.lib.brik_moe_matmul_t_q4(self.handle, _addr(x), _addr(row_off), _addr(nib),
                                                  _addr(sc), _addr(mn), _addr(y), E, R, K, N))

    def moe_matmul_t_q4_x2(self, x, row_off, a, y_a, b, y_b, E, R, K, N):
        """Two stacked q4 tensors (``a``, ``b``: (nib, sc, mn) address triples) on the same routed rows,
        one launch (brik_moe_matmul_t_q4_x2)."""
        self._check(self.lib.brik_moe_matmul_t_q4_x2(self.handle, _addr(x), _addr(row_off), *map(_addr, a),
                                                     _addr(y_a), *map(_addr, b), _addr(y_b), E, R, K, N))

    def gemv_plan(self, fmt: str, jobs) -> "GemvPlan":
        """jobs: iterable of dicts with x, p0, p1, sc, mn, y (device addresses), K, N, and optionally the
        fusions of ``brik_gemv_job_ex``: gate, norm_w, eps, one_plus, gelu, res. Jobs without any
        fusion key go through ``brik_gemv_plan_create``, the others through the ``_ex`` form."""
        jobs = list(jobs)
        fused = any(k in j for j in jobs for k in ("gate", "norm_w", "res"))
        h = _P()
        if not fused:
            arr = (GemvJob * len(jobs))()
            for i, j in enumerate(jobs):
                arr[i] = GemvJob(_addr(j["x"]), _addr(j["p0"]), _addr(j.get("p1")), _addr(j["sc"]),
                                 _addr(j.get("mn")), _addr(j["y"]), j["K"], j["N"])
            self._check(self.lib.brik_gemv_plan_create(self.handle, FMT_CODES[fmt], ctypes.cast(arr, _P), len(jobs),
                                                       ctypes.byref(h)))
            return GemvPlan(self, h)
        arr = (GemvJobEx * len(jobs))()
        for i, j in enumerate(jobs):
            arr[i] = _job_ex(j)
        self._check(self.lib.brik_gemv_plan_create_ex(self.handle, FMT_CODES[fmt], ctypes.cast(arr, _P), len(jobs),
                                                      ctypes.byref(h)))
        return GemvPlan(self, h)

    def gemv_plan_glu(self, fmt: str, gate, up, down):
        """The linked (gate/up, down) plans of ``brik_gemv_plan_create_glu``; each job a dict as for
        :meth:`gemv_plan`. down must read gate's and up's outputs (``gate=gate["y"]``, ``x=up["y"]``).
        Returns ``(gate_up_plan, down_plan)``; run them in that order."""
        jobs = (GemvJobEx * 3)(_job_ex(gate), _job_ex(up), _job_ex(down))
        hg, hd = _P(), _P()
        base = ctypes.addressof(jobs)
        size = ctypes.sizeof(GemvJobEx)
        self._check(self.lib.brik_gemv_plan_create_glu(self.handle, FMT_CODES[fmt], _P(base), _P(base + size),
                                                       _P(base + 2 * size), ctypes.byref(hg), ctypes.byref(hd)))
        return GemvPlan(self, hg), GemvPlan(self, hd)

    # ---- recorded launches (HIP graphs) ---------------------------------------------------------
    def graph_begin(self):
        """Record (not run) every launch enqueued from now on until :meth:`graph_end`."""
        self._check(self.lib.brik_graph_begin(self.handle))

    def graph_end(self) -> "Graph":
        h = _P()
        self._check(self.lib.brik_graph_end(self.handle, ctypes.byref(h)))
        return Graph(self, h)

    # ---- sampling pre-work ----------------------------------------------------------------
    def logits_topk(self, logits, n, recent, n_recent, penalty, softcap, k, ids, vals):
        """Softcap, repetition penalty (in place on ``logits``) and the top ``k``, on the stream."""
        self._check(self.lib.brik_logits_topk(self.handle, _addr(logits), n, _addr(recent), n_recent, penalty,
                                              softcap, k, _addr(ids), _addr(vals)))

    def lm_head_topk(self, fmt: str, x, planes, K, vocab, recent, n_recent, penalty, softcap, k, ids, vals):
        """``x . deq(W)^T`` over the vocab, then :meth:`logits_topk` on the logits (a workspace)."""
        tail = (K, vocab, _addr(recent), n_recent, penalty, softcap, k, _addr(ids), _addr(vals))
        fn = getattr(self.lib, f"brik_lm_head_topk_{fmt}")
        self._check(fn(self.handle, _addr(x), *[_addr(p) for p in planes], *tail))

    # ---- the attention side of a decoder layer -------------------------------------------------
    # The structures below are made once and used in every step: they hold addresses, not contents.
    @staticmethod
    def kv_cache(fmt: str, heads, head_dim, page, pages, k, v) -> KvCache:
        """A paged cache over the planes of ``k`` and ``v``: q8 (codes, sc), q4 (nib, sc, mn)."""
        k, v = [_addr(p) for p in k], [_addr(p) for p in v]
        mins = (k[2], v[2]) if fmt == "q4" else (None, None)
        return KvCache(FMT_CODES[fmt], heads, head_dim, page, pages, 0, k[0], v[0], k[1], v[1], *mins)

    @staticmethod
    def kv_batch(seqs, rows, kv_len=None, table=None, table_cols=0, max_len=0, row_off=None, max_rows=0, prefix_len=0,
                 prefix_table=None) -> KvBatch:
        """The sequences of a step: device arrays ``kv_len`` [seqs], ``table`` [seqs, table_cols] and, unless every sequence
        has rows / seqs rows, ``row_off`` [seqs + 1]; ``prefix_table`` for a shared prefix of ``prefix_len`` tokens."""
        return KvBatch(seqs, rows, _addr(row_off), _addr(kv_len), _addr(table), table_cols, max_len, max_rows, prefix_len,
                       _addr(prefix_table))

    @staticmethod
    def qkv_rows(head_dim, heads=0, kv_heads=0, q=None, k=None, v=None, q_out=None, k_out=None, q_norm=None, k_norm=None,
                 eps=1e-6, inv_freq=None, rot_dim=0, positions=None, one_plus=False, interleaved=False, q_stride=0, k_stride=0,
                 v_stride=0, q_out_stride=0, k_out_stride=0) -> QkvRows:
        """The q / k / v rows of a step and what is done to them (``brik_qkv_rows``)."""
        flags = (BRIK_QKV_GAIN_ONE_PLUS if one_plus else 0) | (BRIK_QKV_INTERLEAVED if interleaved else 0)
        return QkvRows(_addr(q), _addr(k), _addr(v), _addr(q_out), _addr(k_out), q_stride, k_stride, v_stride, q_out_stride,
                       k_out_stride, _addr(q_norm), _addr(k_norm), _addr(inv_freq), _addr(positions), heads, kv_heads,
                       head_dim, rot_dim, flags, eps)

    @staticmethod
    def attn_args(q, out, heads, scale, window=0, softcap=0.0, q_stride=0, out_stride=0) -> AttnArgs:
        return AttnArgs(_addr(q), _addr(out), q_stride, out_stride, heads, window, scale, softcap)

    def qk_norm_rope(self, batch: KvBatch, rows: QkvRows):
        """Head norms and rotation of q and k (brik_qk_norm_rope)."""
        self._check(self.lib.brik_qk_norm_rope(self.handle, ctypes.addressof(batch), ctypes.addressof(rows)))

    def kv_write(self, cache: KvCache, batch: KvBatch, rows: QkvRows):
        """k and v quantized into the cache, q and k normed and rotated on the way (brik_kv_write)."""
        self._check(self.lib.brik_kv_write(self.handle, ctypes.addressof(cache), ctypes.addressof(batch), ctypes.addressof(rows)))

    def kv_read(self, cache: KvCache, batch: KvBatch, k, v):
        """The batch's tokens read back as f32 rows (brik_kv_read)."""
        self._check(self.lib.brik_kv_read(self.handle, ctypes.addressof(cache), ctypes.addressof(batch), _addr(k), _addr(v)))

    def attention(self, cache: KvCache, batch: KvBatch, args: AttnArgs):
        """Attention of the batch's rows over the cache (brik_attention)."""
        self._check(self.lib.brik_attention(self.handle, ctypes.addressof(cache), ctypes.addressof(batch), ctypes.addressof(args)))

    # ---- experts: routing, tokens to their experts and back ---------------------------------------
    @staticmethod
    def moe_route_args(logits, tokens, experts, k, ids, weights, bias=None, row_off=None, src=None, slot=None, sigmoid=False, renorm=False,
                       scale=1.0, logit_stride=0) -> MoeRouteArgs:
        """The routing of a step, made once and used in every one (``brik_moe_route_args``)."""
        flags = (BRIK_ROUTE_SIGMOID if sigmoid else 0) | (BRIK_ROUTE_RENORM if renorm else 0)
        return MoeRouteArgs(_addr(logits), _addr(bias), logit_stride, _addr(ids), _addr(weights), _addr(row_off), _addr(src), _addr(slot),
                            *_i32(tokens, experts, k), flags, scale, 0)

    def moe_route(self, args: MoeRouteArgs):
        """The k experts of every token, their weights and, if asked for, the sorted assignments (brik_moe_route)."""
        self._check(self.lib.brik_moe_route(self.handle, ctypes.addressof(args)))

    def moe_route_grad(self, args: MoeRouteArgs, dweights, dlogits):
        """The gradient of the logits from that of the weights (brik_moe_route_grad)."""
        self._check(self.lib.brik_moe_route_grad(self.handle, ctypes.addressof(args), _addr(dweights), _addr(dlogits)))

    def moe_sort(self, ids, tokens, k, experts, row_off, src, slot):
        """Assignments ``ids`` [tokens, k] sorted by expert (brik_moe_sort)."""
        self._check(self.lib.brik_moe_sort(self.handle, _addr(ids), *_i32(tokens, k, experts), _addr(row_off), _addr(src), _addr(slot)))

    def moe_dispatch(self, x, slot, weights, x_sorted, tokens, k, width):
        """The tokens' rows to their experts' rows, times ``weights`` unless None (brik_moe_dispatch)."""
        self._check(self.lib.brik_moe_dispatch(self.handle, _addr(x), _addr(slot), _addr(weights), _addr(x_sorted), *_i32(tokens, k, width)))

    def moe_combine(self, y_sorted, slot, weights, res, out, tokens, k, width):
        """The experts' rows back to the tokens, weighted and summed, plus ``res`` unless None (brik_moe_combine)."""
        self._check(self.lib.brik_moe_combine(self.handle, _addr(y_sorted), _addr(slot), _addr(weights), _addr(res), _addr(out),
                                              *_i32(tokens, k, width)))

    def moe_combine_grad(self, dout, y_sorted, slot, weights, dy_sorted, dweights, tokens, k, width):
        """The gradients of the experts' rows and of the weights (brik_moe_combine_grad)."""
        self._check(self.lib.brik_moe_combine_grad(self.handle, _addr(dout), _addr(y_sorted), _addr(slot), _addr(weights), _addr(dy_sorted),
                                                   _addr(dweights), *_i32(tokens, k, width)))

    # ---- products of 8-bit integers ---------------------------------------------------------------
    def quantize_i8(self, x, codes, scales, M, K, x_stride=0, gate=None, gate_stride=0, gelu=False):
        """Rows of x, or of act(gate) * x, to int8 codes and a scale each (brik_quantize_i8)."""
        self._check(self.lib.brik_quantize_i8(self.handle, _addr(x), x_stride, _addr(gate), gate_stride, BRIK_JOB_ACT_GELU if gelu else 0,
                                              _addr(codes), _addr(scales), *_i32(M, K)))

    def matmul_t_i8(self, x, x_scales, w, w_scales, y, M, K, N, res=None):
        """y = x . w^T of int8 codes, scaled by row and channel, plus ``res`` unless None (brik_matmul_t_i8)."""
        self._check(self.lib.brik_matmul_t_i8(self.handle, _addr(x), _addr(x_scales), _addr(w), _addr(w_scales), _addr(res), _addr(y),
                                              *_i32(M, K, N)))

    def moe_matmul_t_i8(self, x, x_scales, row_off, w, w_scales, y_sorted, E, rows, K, N, src=None, k=1, x_rows=None):
        """The same by experts (brik_moe_matmul_t_i8). x: the sorted rows or, with ``src`` and ``k``, the tokens (rows / k of them
        unless ``x_rows`` says otherwise)."""
        if x_rows is None:
            x_rows = rows if src is None else rows // max(k, 1)
        self._check(self.lib.brik_moe_matmul_t_i8(self.handle, _addr(x), _addr(x_scales), *_i32(x_rows), _addr(src), *_i32(k), _addr(row_off),
                                                  _addr(w), _addr(w_scales), _addr(y_sorted), *_i32(E, rows, K, N)))

    def dequant_q8(self, codes, sc, out, n):
        self._check(self.lib.brik_dequant_q8_f32(self.handle, _addr(codes), _addr(sc), _addr(out), n))

    def dequant_q4(self, nib, sc, mn, out, n):
        self._check(self.lib.brik_dequant_q4_f32(self.handle, _addr(nib), _addr(sc), _addr(mn), _addr(out), n))

    def dequant_q3(self, lo, hi, sc, mn, out, n):
        self._check(self.lib.brik_dequant_q3_f32(self.handle, _addr(lo), _addr(hi), _addr(sc), _addr(mn),
                                                 _addr(out), n))

    def quantize(self, fmt: str, src, planes, n):
        """Encode ``n`` f32 values at ``src`` into the planes of ``fmt`` (the unpackQ* order:
        q8 codes, sc; q4 nib, sc, mn; q3 lo, hi, sc, mn), byte-identical to quantizeQ*."""
        fn = getattr(self.lib, f"brik_quantize_{fmt}")
        self._check(fn(self.handle, _addr(src), *[_addr(p) for p in planes], n))

    def conv2d(self, fmt: str, inp, planes, bias, out, Cin, H, W, Cout, kh, kw, stride=1, pad=0):
        """conv2d_direct_q8 / _q4: ``out[Cout, OH, OW]`` from ``inp[Cin, H, W]`` and a q8 (codes, sc) or
        q4 (nib, sc, mn) OIHW weight; ``bias`` may be None."""
        fn = getattr(self.lib, f"brik_conv2d_{fmt}")
        self._check(fn(self.handle, _addr(inp), *[_addr(p) for p in planes], _addr(bias), _addr(out),
                       Cin, H, W, Cout, kh, kw, stride, pad))

    def matmul_t_f16w(self, x, w, y, M, K, N):
        """y = x . W^T with W [N, K] IEEE f16 bits (MATMUL_T_F16W)."""
        self._check(self.lib.brik_matmul_t_f16w(self.handle, _addr(x), _addr(w), _addr(y), M, K, N))

    def f16_to_f32(self, src, out, n):
        self._check(self.lib.brik_f16_to_f32(self.handle, _addr(src), _addr(out), n))


class Fence:
    """A point on the context stream (``brik_fence``): :meth:`d2h` waits for it, then copies to host;
    safe to call from another thread while the context keeps enqueueing."""

    def __init__(self, ctx: Context, handle):
        self.ctx, self.handle = ctx, handle

    def d2h(self, src, dtype, count: int) -> np.ndarray:
        out = np.empty(count, dtype=dtype)
        rc = self.ctx.lib.brik_fence_d2h(self.handle, _P(out.ctypes.data), _addr(src), out.nbytes)
        if rc != BRIK_OK:
            raise BrikError(rc, self.ctx.lib.brik_fence_error(self.handle).decode())
        return out

    def destroy(self):
        if self.handle:
            self.ctx.lib.brik_fence_destroy(self.handle)
            self.handle = None


class Graph:
    """A recorded launch sequence (``brik_graph``): :meth:`launch` replays it on the context stream."""

    def __init__(self, ctx: Context, handle):
        self.ctx, self.handle = ctx, handle

    def launch(self):
        self.ctx._check(self.ctx.lib.brik_graph_launch(self.ctx.handle, self.handle))

    def destroy(self):
        if self.handle:
            self.ctx.lib.brik_graph_destroy(self.ctx.handle, self.handle)
            self.handle = None


def _job_ex(j) -> GemvJobEx:
    base = GemvJob(_addr(j["x"]), _addr(j["p0"]), _addr(j.get("p1")), _addr(j["sc"]), _addr(j.get("mn")),
                   _addr(j["y"]), j["K"], j["N"])
    flags = (BRIK_JOB_GAIN_ONE_PLUS if j.get("one_plus") else 0) | (BRIK_JOB_ACT_GELU if j.get("gelu") else 0)
    return GemvJobEx(base, _addr(j.get("gate")), _addr(j.get("norm_w")), _addr(j.get("res")),
                     float(j.get("eps", 1e-6)), flags)


class GemvPlan:
    def __init__(self, ctx: Context, handle):
        self.ctx, self.handle = ctx, handle

    def run(self):
        self.ctx._check(self.ctx.lib.brik_gemv_plan_run(self.ctx.handle, self.handle))

    def destroy(self):
        if self.handle:
            self.ctx.lib.brik_gemv_plan_destroy(self.ctx.handle, self.handle)
            self.handle = None
