"""ctypes binding of libltx_b200.so (the C ABI in include/ltx_b200.h).

This is the thin layer a Python caller (the tests, bench.py) uses; it mirrors
the names of the reference crates' entry points it wraps.  The compute path is
entirely in the shared library; when the library cannot be loaded every call
raises (there is no CPU fallback).
"""
from __future__ import annotations

import ctypes
import struct
import weakref
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libltx_b200.so")

LTX_F32, LTX_F16, LTX_BF16, LTX_F8_E4M3, LTX_F8_E5M2 = 0, 1, 2, 3, 4
MAX_DELTAS = 8
COMM_ID_BYTES = 128

STATUS = {
    0: "OK", 1: "INVALID_ARG", 2: "SHAPE", 3: "DTYPE", 4: "MISSING_KEY", 5: "DUPLICATE_KEY",
    6: "LORA_RANK", 7: "NO_LORA_MATCHES", 8: "IO", 9: "FORMAT", 10: "CONFIG", 11: "SIGMA",
    12: "SCHEDULE", 13: "CUDA", 14: "NCCL", 15: "TIMEOUT", 16: "OOM", 17: "UNSUPPORTED",
    18: "MISSING_CONFIG", 19: "NEGATIVE_CONTEXT", 20: "CHUNK_PLAN",
    21: "TARGET_TOKENS", 22: "STRENGTH",
}


class LtxError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"ltx_b200 error {STATUS.get(code, code)}: {msg}")
        self.code = code
        self.kind = STATUS.get(code, str(code))


class LoraDelta(ctypes.Structure):
    _fields_ = [("a_dev", ctypes.c_void_p), ("b_dev", ctypes.c_void_p), ("rank", ctypes.c_int32),
                ("a_dtype", ctypes.c_int32), ("b_dtype", ctypes.c_int32), ("coeff", ctypes.c_float)]


class Chunk(ctypes.Structure):
    """ltx_chunk (plan::Chunk): frames [start, end) and the overlap with the previous chunk."""
    _fields_ = [("start", ctypes.c_uint32), ("end", ctypes.c_uint32), ("real_overlap", ctypes.c_uint32)]

    def as_tuple(self):
        return (self.start, self.end, self.real_overlap)


_lib = None


def lib() -> ctypes.CDLL:
    """Loads the library (raising if it is missing: there is no fallback)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is missing: run `python ltx-rust_b200/build.py` first")
    L = ctypes.CDLL(LIB_PATH)
    V, I, F, P, I64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_void_p, ctypes.c_int64
    sig = {
        "ltx_ctx_create": (I, [I, V, ctypes.POINTER(V)]),
        "ltx_ctx_destroy": (None, [V]),
        "ltx_last_error": (ctypes.c_char_p, [V]),
        "ltx_ctx_stream": (V, [V]),
        "ltx_ctx_synchronize": (I, [V]),
        "ltx_lora_coeff": (F, [F, F, ctypes.c_int32]),
        "ltx_dequant_merge": (I, [V, P, ctypes.c_int32, ctypes.c_int32, F, I64, I64,
                                  ctypes.POINTER(LoraDelta), ctypes.c_int32, P, ctypes.c_int32]),
        "ltx_gemm_bf16": (I, [V, P, I64, P, I64, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                              P, P, I64, P, P, I64]),
        "ltx_gemm_e4m3": (I, [V, P, I64, P, P, I64, F, P, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                              ctypes.c_int32, P, P, I64, P, P, I64, P, I64, P, I64, ctypes.c_int32]),
        "ltx_quantize_rows_e4m3": (I, [V, P, I64, ctypes.c_int32, ctypes.c_int32, P, I64, P]),
        "ltx_attention_fwd": (I, [V, P, I64, P, I64, P, I64, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                                  ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, F, P, I64]),
        "ltx_rope_table": (I, [V, P, ctypes.c_int32, ctypes.c_int32, ctypes.c_double, ctypes.c_double, I64,
                               ctypes.c_double, ctypes.c_double, ctypes.c_double, P, P]),
        "ltx_qk_norm_rope": (I, [V, ctypes.c_char_p]),
        "ltx_gemm_adapters": (I, [V, ctypes.c_char_p]),
        "ltx_attention_packed_fwd": (I, [V, ctypes.c_char_p]),
        "ltx_store_open": (I, [V, ctypes.POINTER(ctypes.c_char_p), ctypes.c_int32, ctypes.c_int32, ctypes.POINTER(V)]),
        "ltx_store_destroy": (None, [V]),
        "ltx_store_merge_lora": (I, [V, ctypes.c_char_p, F, ctypes.POINTER(ctypes.c_int32),
                                     ctypes.POINTER(ctypes.c_int32)]),
        "ltx_store_contains": (I, [V, ctypes.c_char_p]),
        "ltx_store_num_keys": (ctypes.c_int32, [V]),
        "ltx_store_key": (ctypes.c_char_p, [V, ctypes.c_int32]),
        "ltx_store_shape": (I, [V, ctypes.c_char_p, ctypes.POINTER(I64), ctypes.c_int32,
                                ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(ctypes.c_int32)]),
        "ltx_store_metadata": (I, [V, ctypes.c_char_p, ctypes.c_char_p, ctypes.c_size_t,
                                   ctypes.POINTER(ctypes.c_size_t)]),
        "ltx_store_read": (I, [V, ctypes.c_char_p, ctypes.c_int32, P, ctypes.c_size_t]),
        "ltx_model_load": (I, [V, V, ctypes.c_char_p, ctypes.POINTER(V)]),
        "ltx_model_init_random": (I, [V, ctypes.c_char_p, ctypes.c_uint64, ctypes.c_int32, F, ctypes.POINTER(V)]),
        "ltx_model_destroy": (None, [V]),
        "ltx_model_weight_bytes": (I64, [V]),
        "ltx_model_forward": (I, [V, V, P, P, P, P, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, P]),
        "ltx_block_forward": (I, [V, V, ctypes.c_int32, P, P, P, P, P, ctypes.c_int32, ctypes.c_int32,
                                  ctypes.c_int32]),
        "ltx_cfg_euler_step": (I, [V, P, P, P, P, P, ctypes.c_int32, ctypes.c_int32, F, F, F, F]),
        "ltx_denoise_step": (I, [V, V, P, P, P, P, P, P, P, ctypes.c_int32, ctypes.c_int32, F, F, F, F]),
        "ltx_denoise_loop": (I, [V, V, P, P, P, P, P, P, P, ctypes.c_int32, ctypes.c_int32, P, ctypes.c_int32, F, F,
                                 ctypes.c_int32, P]),
        "ltx_apply_noise": (I, [V, P, P, P, P, ctypes.c_int32, ctypes.c_int32, F]),
        "ltx_apply_keyframe": (I, [V, P, P, ctypes.c_int32, ctypes.c_int32, P, ctypes.c_int32, ctypes.c_int32, F]),
        "ltx_seam_cond_plan": (I, [ctypes.c_uint32, ctypes.POINTER(ctypes.c_uint32), ctypes.POINTER(ctypes.c_float),
                                   ctypes.POINTER(ctypes.c_uint32)]),
        "ltx_scheduler_execute": (I, [ctypes.c_int32, ctypes.c_uint64, F, F, ctypes.c_int32, F, P]),
        "ltx_target_positions": (I, [ctypes.c_uint32] * 7 + [F, P]),
        "ltx_reference_positions": (I, [ctypes.c_uint32] * 8 + [F, ctypes.c_uint32, ctypes.c_uint32, P]),
        "ltx_patchify": (I, [V, P] + [ctypes.c_int32] * 5 + [P]),
        "ltx_unpatchify": (I, [V, P] + [ctypes.c_int32] * 5 + [P]),
        "ltx_host_last_error": (ctypes.c_char_p, []),
        "ltx_comm_unique_id": (I, [P, ctypes.c_size_t]),
        "ltx_ctx_init_comm": (I, [V, P, ctypes.c_size_t, ctypes.c_int32, ctypes.c_int32]),
        "ltx_ctx_comm_check": (I, [V]),
        "ltx_ctx_init_cfg_comm": (I, [V, P, ctypes.c_size_t, ctypes.c_int32]),
        "ltx_ctx_tp_exchange": (I, [V]),
        "ltx_ctx_abort_comm": (None, [V]),
        "ltx_wait_flag": (I, [V, P, ctypes.c_int32, ctypes.c_uint32]),
        "ltx_set_flag": (I, [V, P, ctypes.c_int32]),
        "ltx_chunk_plan": (I, [ctypes.c_uint32] * 3 + [ctypes.POINTER(Chunk), ctypes.c_int32,
                                                        ctypes.POINTER(ctypes.c_int32)]),
        "ltx_crossfade_weight": (F, [ctypes.c_uint32, ctypes.c_uint32]),
        "ltx_seam_blend": (I, [V, P, P, ctypes.c_uint32, I64, P]),
        "ltx_chunk_assemble": (I, [V, ctypes.POINTER(P), ctypes.POINTER(Chunk), ctypes.c_int32, I64, P]),
        "ltx_dequant_merge_noalloc": (I, [V, P, ctypes.c_int32, ctypes.c_int32, F, I64, I64,
                                          ctypes.POINTER(LoraDelta), ctypes.c_int32, P, ctypes.c_int32,
                                          ctypes.c_char_p, ctypes.c_size_t]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


class Context:
    """An ltx_ctx bound to a CUDA device and stream (default: torch's current stream)."""

    def __init__(self, device: int = 0, stream: int | None = None):
        if stream is None:
            import torch
            stream = torch.cuda.current_stream(device).cuda_stream
        self.h = ctypes.c_void_p()
        self.device = device
        # stores and models made on this context: closed before it (their
        # destructors synchronise on the context's stream)
        self._owned = weakref.WeakSet()
        rc = lib().ltx_ctx_create(device, ctypes.c_void_p(stream), ctypes.byref(self.h))
        if rc != 0:
            raise LtxError(rc, f"ltx_ctx_create(device={device})")

    def check(self, rc: int, what: str):
        if rc != 0:
            msg = lib().ltx_last_error(self.h)
            raise LtxError(rc, f"{what}: {msg.decode() if msg else ''}")

    def init_comm(self, comm_id: bytes, nranks: int, rank: int):
        """Binds this context to rank `rank` of a tensor-parallel group (collective)."""
        buf = ctypes.create_string_buffer(bytes(comm_id), COMM_ID_BYTES)
        self.check(lib().ltx_ctx_init_comm(self.h, buf, COMM_ID_BYTES, nranks, rank), "ltx_ctx_init_comm")

    def tp_exchange(self) -> str:
        """How tensor-parallel sums run on this context (ltx_ctx_tp_exchange)."""
        return {0: "none", 1: "peer", 2: "nccl"}[lib().ltx_ctx_tp_exchange(self.h)]

    def init_cfg_comm(self, comm_id: bytes, cfg_rank: int):
        """Makes this context half of a CFG-parallel pair (ltx_ctx_init_cfg_comm)."""
        buf = ctypes.create_string_buffer(comm_id, len(comm_id))
        self.check(lib().ltx_ctx_init_cfg_comm(self.h, buf, len(comm_id), cfg_rank), "ltx_ctx_init_cfg_comm")

    def comm_check(self):
        self.check(lib().ltx_ctx_comm_check(self.h), "ltx_ctx_comm_check")

    def abort_comm(self):
        lib().ltx_ctx_abort_comm(self.h)

    def wait_flag(self, flag, expect: int, timeout_ms: int = 2000):
        """Enqueues a bounded device-side wait until flag (int32 device tensor/pointer) == expect."""
        self.check(lib().ltx_wait_flag(self.h, _ptr(flag), expect, timeout_ms), "ltx_wait_flag")

    def set_flag(self, flag, value: int):
        self.check(lib().ltx_set_flag(self.h, _ptr(flag), value), "ltx_set_flag")

    def synchronize(self):
        self.check(lib().ltx_ctx_synchronize(self.h), "synchronize")

    def close(self):
        if self.h:
            for obj in list(self._owned):
                obj.close()
            lib().ltx_ctx_destroy(self.h)
            self.h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ── ltx-weights ──────────────────────────────────────────────────────────
    def dequant_merge(self, w_ptr: int, w_dtype: int, has_scale: bool, scale: float, out_features: int,
                      in_features: int, deltas, dst_ptr: int, dst_dtype: int):
        """WeightStore::read body on device pointers (ltx_dequant_merge)."""
        n = len(deltas)
        arr = (LoraDelta * max(n, 1))(*[LoraDelta(*d) for d in deltas])
        self.check(lib().ltx_dequant_merge(self.h, ctypes.c_void_p(w_ptr), w_dtype, int(has_scale), scale,
                                           out_features, in_features, arr, n, ctypes.c_void_p(dst_ptr),
                                           dst_dtype), "ltx_dequant_merge")


EPI_BF16, EPI_GELU_BF16, EPI_F32, EPI_RESID = 0, 1, 2, 3


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t if isinstance(t, int) else t.data_ptr())


def gemm(ctx: "Context", a, w, out, epilogue=EPI_BF16, bias=None, gate=None, gate_idx=None):
    """out = epilogue(a @ w.T) with torch CUDA tensors (a [M,K] bf16, w [N,K] bf16)."""
    M, K = a.shape
    N = w.shape[0]
    ctx.check(lib().ltx_gemm_bf16(ctx.h, _ptr(a), a.stride(0), _ptr(w), w.stride(0), M, N, K, epilogue,
                                  _ptr(bias), _ptr(out), out.stride(0), _ptr(gate), _ptr(gate_idx),
                                  gate.stride(0) if gate is not None else 0), "ltx_gemm_bf16")


def gemm_e4m3(ctx: "Context", a, a_scale, w, w_scale, out, epilogue=EPI_BF16, bias=None, gate=None, gate_idx=None,
              w_col_scale=None, a2=None, b2=None):
    """out = epilogue(((a @ w.T) + a2 @ b2.T) * a_scale[:, None] * w_scale) with e4m3 operands a [M,K],
    w [N,K] held as uint8 (or float8_e4m3fn) CUDA tensors; a_scale f32 [M] or None; w_col_scale f32 [N]
    overrides w_scale per column; a2 [M,k2] / b2 [N,k2] bf16 append a low-rank block (k2 % 64 == 0)."""
    M, K = a.shape
    N = w.shape[0]
    k2 = 0 if a2 is None else a2.shape[1]
    ctx.check(lib().ltx_gemm_e4m3(ctx.h, _ptr(a), a.stride(0), _ptr(a_scale), _ptr(w), w.stride(0), float(w_scale),
                                  _ptr(w_col_scale), M, N, K, epilogue, _ptr(bias), _ptr(out), out.stride(0), _ptr(gate),
                                  _ptr(gate_idx), gate.stride(0) if gate is not None else 0, _ptr(a2),
                                  a2.stride(0) if a2 is not None else 0, _ptr(b2),
                                  b2.stride(0) if b2 is not None else 0, k2), "ltx_gemm_e4m3")


def quantize_rows_e4m3(ctx: "Context", x, out, scale):
    """Per-row e4m3 of a bf16 [rows, cols] CUDA tensor into uint8 out [rows, cols] and f32 scale [rows]."""
    rows, cols = x.shape
    ctx.check(lib().ltx_quantize_rows_e4m3(ctx.h, _ptr(x), x.stride(0), rows, cols, _ptr(out), out.stride(0),
                                           _ptr(scale)), "ltx_quantize_rows_e4m3")


def attention(ctx: "Context", q, k, v, out, batch, heads, tq, tk, scale, head_dim=128):
    """out = softmax(q k^T * scale) v; q/k/out token-major bf16 CUDA tensors, v bf16 or f16 (row stride = stride(0))."""
    import torch
    vdt = LTX_F16 if v.dtype == torch.float16 else LTX_BF16
    ctx.check(lib().ltx_attention_fwd(ctx.h, _ptr(q), q.stride(0), _ptr(k), k.stride(0), _ptr(v), v.stride(0), vdt,
                                      batch, heads, tq, tk, head_dim, scale, _ptr(out), out.stride(0)),
              "ltx_attention_fwd")


# ── packed batches ─────────────────────────────────────────────────────────────

ROPE_HALF, ROPE_INTERLEAVED = 0, 1

# The arguments of the packed-batch calls as the header's structs lay them out (ltx_norm_rope, ltx_adapter_gemm,
# ltx_packed_attention): packed in one step, a tenth of the time ctypes takes for as many single ones.
_NORM_ROPE = struct.Struct("@9P4q9if")
_ADAPTER_GEMM = struct.Struct("@10P4q7i")
_PACKED_ATTENTION = struct.Struct("@8P4q8i2f")


def _refuse(ctx, what, name, t, dtypes, shape):
    """The reason why `t` is not a tensor of the context's device, one of `dtypes` and `shape`, its rows contiguous."""
    if not t.is_cuda or t.device.index != ctx.device:
        raise LtxError(1, f"{what}: {name} must be on cuda:{ctx.device}, not {t.device}")
    if t.dtype not in dtypes:
        raise LtxError(3, f"{what}: {name} is {t.dtype}, not {' or '.join(str(d) for d in dtypes)}")
    if tuple(t.shape) != tuple(shape):
        raise LtxError(2, f"{what}: {name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    raise LtxError(2, f"{what}: {name} needs contiguous, non-overlapping rows")


def _dense(ctx, what, name, t, dtype, shape):
    """Address of a contiguous CUDA tensor of the context's device; LtxError for any other."""
    if t.get_device() != ctx.device or t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        _refuse(ctx, what, name, t, (dtype,), shape)
    return t.data_ptr()


def _rows(ctx, what, name, t, dtypes, rows, cols):
    """(address, leading dimension) of a CUDA matrix [rows, cols] of the context's device with contiguous rows that do
    not overlap; LtxError for any other.  A single row's stride says nothing, so its length stands for it, and neither
    does the step inside rows of one value."""
    if t.get_device() != ctx.device or t.dtype not in dtypes or t.shape != (rows, cols):
        _refuse(ctx, what, name, t, dtypes, (rows, cols))
    ld, step = t.stride()
    if (step == 1 or cols == 1) and ld >= cols:
        return t.data_ptr(), ld if rows > 1 else cols
    if rows and cols and ((step != 1 and cols > 1) or (ld < cols and rows > 1)):
        _refuse(ctx, what, name, t, dtypes, (rows, cols))
    return t.data_ptr(), cols


def _matrix(what, name, t):
    """Shape of a two-dimensional tensor."""
    if t.dim() != 2:
        raise LtxError(2, f"{what}: {name} has shape {tuple(t.shape)}")
    return t.shape


def rope_table(ctx: "Context", pos, cos, sin, theta=10000.0, factor=1.0, original_len=0, turns_low=1.0, turns_high=32.0,
               amplitude=1.0):
    """cos/sin f32 [rows, rot_dim/2] of int32 positions [rows] (None: 0, 1, 2, ...), stretched by `factor`
    (ltx_rope_table)."""
    import torch
    what, f32 = "rope_table", torch.float32
    shape = rows, half = _matrix(what, "cos", cos)
    c, s = _dense(ctx, what, "cos", cos, f32, shape), _dense(ctx, what, "sin", sin, f32, shape)
    p = None if pos is None else _dense(ctx, what, "pos", pos, torch.int32, (rows,))
    rc = lib().ltx_rope_table(ctx.h, p, rows, 2 * half, theta, factor, original_len, turns_low, turns_high, amplitude, c, s)
    if rc:
        ctx.check(rc, "ltx_rope_table")


def qk_norm_rope(ctx: "Context", q, k, q_out, k_out, heads, kv_heads, cos, sin, pos=None, gamma_q=None, gamma_k=None,
                 norm=True, eps=1e-6, layout=ROPE_HALF):
    """Per-head RMSNorm of q [rows, heads*d] and k [rows, kv_heads*d] (k None with kv_heads 0) and the rotation of
    each head's first values by cos/sin [table_rows, rot_dim/2] (None: no rotation), row r at table row pos[r]
    (ltx_qk_norm_rope).  q_out / k_out may be q / k."""
    import torch
    what, f32, dt = "qk_norm_rope", torch.float32, q.dtype
    rows, cols = _matrix(what, "q", q)
    d = cols // max(heads, 1)
    types = {torch.bfloat16: LTX_BF16, torch.float16: LTX_F16, f32: LTX_F32}
    qp, ldq = _rows(ctx, what, "q", q, types, rows, heads * d)
    qop, ldqo = _rows(ctx, what, "q_out", q_out, (dt,), rows, heads * d)
    kp = kop = gq = gk = cp = sp = pp = ldk = ldko = table = half = 0
    if kv_heads:
        if k is None or k_out is None:
            raise LtxError(1, f"{what}: {kv_heads} key heads without k or k_out")
        kp, ldk = _rows(ctx, what, "k", k, (dt,), rows, kv_heads * d)
        kop, ldko = _rows(ctx, what, "k_out", k_out, (dt,), rows, kv_heads * d)
    if gamma_q is not None:
        gq = _dense(ctx, what, "gamma_q", gamma_q, f32, (d,))
    if gamma_k is not None:
        gk = _dense(ctx, what, "gamma_k", gamma_k, f32, (d,))
    if (cos is None) != (sin is None):
        raise LtxError(1, f"{what}: cos and sin go together")
    if cos is not None:
        shape = table, half = _matrix(what, "cos", cos)
        cp, sp = _dense(ctx, what, "cos", cos, f32, shape), _dense(ctx, what, "sin", sin, f32, shape)
    if pos is not None:
        pp = _dense(ctx, what, "pos", pos, torch.int32, (rows,))
    rc = lib().ltx_qk_norm_rope(ctx.h, _NORM_ROPE.pack(qp, kp, qop, kop, gq, gk, cp, sp, pp, ldq, ldk, ldqo, ldko, types[dt],
                                                       rows, heads, kv_heads, d, 1 if norm else 0, table, 2 * half, layout,
                                                       eps))
    if rc:
        ctx.check(rc, "ltx_qk_norm_rope")


def gemm_adapters(ctx: "Context", x, w, out, adapter_idx, lora_a, lora_b, coeff, epilogue=EPI_BF16, bias=None,
                  gate=None, gate_idx=None):
    """out = epilogue(x @ w.T + coeff[a] (x @ lora_a[a].T) @ lora_b[a].T) with a = adapter_idx[row], -1 for none
    (ltx_gemm_adapters): x [M,K], w [N,K], lora_a [adapters,rank,K], lora_b [adapters,N,rank] bf16, coeff f32,
    adapter_idx int32 [M], out bf16 or (EPI_F32, EPI_RESID) f32 [M,N]."""
    import torch
    what, bf, f32, i32 = "gemm_adapters", torch.bfloat16, torch.float32, torch.int32
    M, K = _matrix(what, "x", x)
    N = _matrix(what, "w", w)[0]
    xp, ldx = _rows(ctx, what, "x", x, (bf,), M, K)
    wp, ldw = _rows(ctx, what, "w", w, (bf,), N, K)
    op, ldo = _rows(ctx, what, "out", out, (f32,) if epilogue in (EPI_F32, EPI_RESID) else (bf,), M, N)
    if lora_a.dim() != 3:
        raise LtxError(2, f"{what}: lora_a has shape {tuple(lora_a.shape)}")
    n, rank = lora_a.shape[:2]
    ip = _dense(ctx, what, "adapter_idx", adapter_idx, i32, (M,))
    ap = _dense(ctx, what, "lora_a", lora_a, bf, (n, rank, K))
    bp = _dense(ctx, what, "lora_b", lora_b, bf, (n, N, rank))
    cp = _dense(ctx, what, "coeff", coeff, f32, (n,))
    bias = 0 if bias is None else _dense(ctx, what, "bias", bias, f32, (N,))
    gp, ldg = (0, 0) if gate is None else _rows(ctx, what, "gate", gate, (f32,), _matrix(what, "gate", gate)[0], N)
    if gate is not None and gate.shape[0] == 0:
        raise LtxError(2, f"{what}: gate has no rows")
    gate_idx = 0 if gate_idx is None else _dense(ctx, what, "gate_idx", gate_idx, i32, (M,))
    rc = lib().ltx_gemm_adapters(ctx.h, _ADAPTER_GEMM.pack(xp, wp, op, bias, gp, gate_idx, ip, ap, bp, cp, ldx, ldw, ldo, ldg, M,
                                                           N, K, epilogue, n, rank, 0 if gate is None else gate.shape[0]))
    if rc:
        ctx.check(rc, "ltx_gemm_adapters")


def attention_packed(ctx: "Context", q, k, v, out, q_offsets, k_offsets, heads, kv_heads, scale, head_dim=128,
                     softcap=0.0, slopes=None, causal=False, prefix=None):
    """out = softmax over the row's own document's keys (ltx_attention_packed_fwd): q/out [rows_q, heads*head_dim] and
    k/v [rows_k, kv_heads*head_dim] bf16 (v bf16 or f16), document i at rows q_offsets[i]:q_offsets[i+1] and
    k_offsets[i]:k_offsets[i+1] (int32 CUDA [docs+1]); slopes f32 [heads], prefix int32 [docs] (with causal)."""
    import torch
    what, bf, i32, qc, kc = "attention_packed", torch.bfloat16, torch.int32, heads * head_dim, kv_heads * head_dim
    docs = q_offsets.shape[0] - 1 if q_offsets.dim() == 1 else -1
    if docs < 0:
        raise LtxError(2, f"{what}: q_offsets needs docs + 1 entries")
    rows_q, rows_k = _matrix(what, "q", q)[0], _matrix(what, "k", k)[0]
    qp, ldq = _rows(ctx, what, "q", q, (bf,), rows_q, qc)
    op, ldo = _rows(ctx, what, "out", out, (bf,), rows_q, qc)
    kp, ldk = _rows(ctx, what, "k", k, (bf,), rows_k, kc)
    vp, ldv = _rows(ctx, what, "v", v, (bf, torch.float16), rows_k, kc)
    qo = _dense(ctx, what, "q_offsets", q_offsets, i32, (docs + 1,))
    ko = _dense(ctx, what, "k_offsets", k_offsets, i32, (docs + 1,))
    slopes = 0 if slopes is None else _dense(ctx, what, "slopes", slopes, torch.float32, (heads,))
    prefix = 0 if prefix is None else _dense(ctx, what, "prefix", prefix, i32, (docs,))
    rc = lib().ltx_attention_packed_fwd(ctx.h, _PACKED_ATTENTION.pack(
        qp, kp, vp, op, qo, ko, prefix, slopes, ldq, ldk, ldv, ldo, LTX_BF16 if v.dtype is bf else LTX_F16, docs, rows_q, rows_k,
        heads, kv_heads, head_dim, 1 if causal else 0, scale, softcap))
    if rc:
        ctx.check(rc, "ltx_attention_packed_fwd")


KEYMAP_IDENTITY, KEYMAP_TRANSFORMER = 0, 1


class WeightStore:
    """ltx-weights WeightStore over the C ABI (ltx_store_*); reads land in device memory."""

    def __init__(self, ctx: Context, paths, keymap=KEYMAP_IDENTITY):
        self.ctx = ctx
        self.h = ctypes.c_void_p()
        arr = (ctypes.c_char_p * len(paths))(*[p.encode() for p in paths])
        ctx.check(lib().ltx_store_open(ctx.h, arr, len(paths), keymap, ctypes.byref(self.h)), "ltx_store_open")
        ctx._owned.add(self)

    def merge_lora(self, path: str, strength: float):
        m, u = ctypes.c_int32(), ctypes.c_int32()
        self.ctx.check(lib().ltx_store_merge_lora(self.h, path.encode(), strength, ctypes.byref(m), ctypes.byref(u)),
                       "ltx_store_merge_lora")
        return m.value, u.value

    def contains(self, key):
        return bool(lib().ltx_store_contains(self.h, key.encode()))

    def keys(self):
        return [lib().ltx_store_key(self.h, i).decode() for i in range(lib().ltx_store_num_keys(self.h))]

    def shape(self, key):
        dims = (ctypes.c_int64 * 8)()
        nd, dt = ctypes.c_int32(), ctypes.c_int32()
        self.ctx.check(lib().ltx_store_shape(self.h, key.encode(), dims, 8, ctypes.byref(nd), ctypes.byref(dt)),
                       "ltx_store_shape")
        return [dims[i] for i in range(nd.value)]

    def metadata(self, key):
        need = ctypes.c_size_t()
        rc = lib().ltx_store_metadata(self.h, key.encode(), None, 0, ctypes.byref(need))
        if rc != 0:
            raise LtxError(rc, f"metadata {key!r}")
        buf = ctypes.create_string_buffer(need.value)
        lib().ltx_store_metadata(self.h, key.encode(), buf, need.value, None)
        return buf.value.decode()

    def read(self, key, dtype=LTX_F32):
        """Returns a torch CUDA tensor (f32 or bf16) with the stored shape."""
        import torch
        shape = self.shape(key)
        t = torch.empty(shape, dtype=torch.float32 if dtype == LTX_F32 else torch.bfloat16, device="cuda")
        self.ctx.check(lib().ltx_store_read(self.h, key.encode(), dtype, _ptr(t), t.numel() * t.element_size()),
                       "ltx_store_read")
        return t

    def close(self):
        if self.h:
            lib().ltx_store_destroy(self.h)
            self.h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class VideoTransformer:
    """ltx-dit VideoTransformer over the C ABI (ltx_model_*)."""

    def __init__(self, ctx: Context, handle):
        self.ctx, self.h = ctx, handle
        ctx._owned.add(self)

    @staticmethod
    def load(ctx: Context, store: WeightStore, config_json: str | None = None):
        h = ctypes.c_void_p()
        ctx.check(lib().ltx_model_load(ctx.h, store.h, config_json.encode() if config_json else None, ctypes.byref(h)),
                  "ltx_model_load")
        return VideoTransformer(ctx, h)

    @staticmethod
    def init_random(ctx: Context, config_json: str, seed=0, lora_rank=64, lora_strength=1.0):
        h = ctypes.c_void_p()
        ctx.check(lib().ltx_model_init_random(ctx.h, config_json.encode(), seed, lora_rank, lora_strength,
                                              ctypes.byref(h)), "ltx_model_init_random")
        return VideoTransformer(ctx, h)

    def weight_bytes(self):
        return lib().ltx_model_weight_bytes(self.h)

    def forward(self, latent, timesteps, positions, context, out):
        """latent [B,T,in], timesteps [B,T], positions [B,3,T,2], context [B,S,Dc] -> out [B,T,out] (f32 CUDA)."""
        B, T, _ = latent.shape
        S = context.shape[1]
        self.ctx.check(lib().ltx_model_forward(self.h, self.ctx.h, _ptr(latent), _ptr(timesteps), _ptr(positions),
                                               _ptr(context), B, T, S, _ptr(out)), "ltx_model_forward")

    def block_forward(self, index, x, context, timestep, pe_cos, pe_sin):
        """TransformerBlock::forward of block `index` in place on x [B,T,D] (ltx_block_forward):
        context [B,S,Dc], timestep [B,T,K*D] (per-token modulation), pe_cos/pe_sin as
        precompute_freqs_cis returns them (split: [B,H,T,d/2]), all f32 CUDA."""
        B, T, _ = x.shape
        S = context.shape[1]
        self.ctx.check(lib().ltx_block_forward(self.h, self.ctx.h, index, _ptr(x), _ptr(context), _ptr(timestep),
                                               _ptr(pe_cos), _ptr(pe_sin), B, T, S), "ltx_block_forward")

    def denoise_step(self, latent, clean, mask, positions, ctx_cond, ctx_uncond, sigma, sigma_next, cfg_scale=1.0,
                     rescale_scale=0.7, mask_host=None):
        """One guided Euler step in place on latent [T, C] (ltx_denoise_step)."""
        T = latent.shape[0]
        S = ctx_cond.shape[0]
        mh = None
        if mask_host is not None:
            mh = mask_host.ctypes.data_as(ctypes.c_void_p)
        self.ctx.check(lib().ltx_denoise_step(self.h, self.ctx.h, _ptr(latent), _ptr(clean), mh, _ptr(mask),
                                              _ptr(positions), _ptr(ctx_cond), _ptr(ctx_uncond), T, S, sigma,
                                              sigma_next, cfg_scale, rescale_scale), "ltx_denoise_step")

    def denoise_loop(self, latent, clean, mask, positions, ctx_cond, ctx_uncond, sigmas, cfg_scale=1.0,
                     rescale_scale=0.7, target_tokens=None, out=None, mask_host=None):
        """euler_denoising_loop + clear_conditioning on the device (ltx_denoise_loop): every
        step in place on latent [T, C]; the first target_tokens tokens are copied to out."""
        import numpy as np
        T = latent.shape[0]
        S = ctx_cond.shape[0]
        sig = np.ascontiguousarray(np.asarray(sigmas, np.float32))
        mh = None if mask_host is None else mask_host.ctypes.data_as(ctypes.c_void_p)
        tt = T if target_tokens is None else target_tokens
        self.ctx.check(lib().ltx_denoise_loop(self.h, self.ctx.h, _ptr(latent), _ptr(clean), mh, _ptr(mask),
                                              _ptr(positions), _ptr(ctx_cond), _ptr(ctx_uncond), T, S,
                                              sig.ctypes.data_as(ctypes.c_void_p), len(sig), cfg_scale,
                                              rescale_scale, tt, _ptr(out)), "ltx_denoise_loop")

    def close(self):
        if self.h:
            lib().ltx_model_destroy(self.h)
            self.h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def cfg_euler_step(ctx: "Context", cond_x0, uncond_x0, latent, clean, mask, sigma, sigma_next, cfg_scale=1.0,
                   rescale_scale=0.7):
    """CFG + rescale + post_process + Euler in place on latent [T, C] from x0 predictions
    (ltx_cfg_euler_step); uncond_x0 may be None when cfg_scale is 1."""
    T, C = latent.shape
    ctx.check(lib().ltx_cfg_euler_step(ctx.h, _ptr(cond_x0), _ptr(uncond_x0), _ptr(latent), _ptr(clean), _ptr(mask),
                                       T, C, sigma, sigma_next, cfg_scale, rescale_scale), "ltx_cfg_euler_step")


def apply_noise(ctx: "Context", latent, noise, clean, mask, noise_scale):
    """GaussianNoiser::apply_with_noise in place on latent [T, C] (ltx_apply_noise)."""
    T, C = latent.shape
    ctx.check(lib().ltx_apply_noise(ctx.h, _ptr(latent), _ptr(noise), _ptr(clean), _ptr(mask), T, C, noise_scale),
              "ltx_apply_noise")


def apply_keyframe(ctx: "Context", clean, mask, image, latent_frame_index, strength):
    """ImageKeyframeCondition::apply_to in place on clean [T, C] and mask [T] (ltx_apply_keyframe):
    image is the one-frame latent [C, 1, H, W] (or [C, H*W]); f32 CUDA tensors."""
    T, C = clean.shape
    tpf = image.numel() // C
    ctx.check(lib().ltx_apply_keyframe(ctx.h, _ptr(clean), _ptr(mask), T, C, _ptr(image), latent_frame_index, tpf,
                                       strength), "ltx_apply_keyframe")


def seam_cond_plan(overlap):
    """seam_cond_plan -> (chunk_local_idx, strength, blend_tail_len) (host, no GPU needed)."""
    idx, st, tail = ctypes.c_uint32(), ctypes.c_float(), ctypes.c_uint32()
    rc = lib().ltx_seam_cond_plan(overlap, ctypes.byref(idx), ctypes.byref(st), ctypes.byref(tail))
    if rc:
        raise LtxError(rc, lib().ltx_host_last_error().decode())
    return idx.value, st.value, tail.value


def scheduler_execute(steps, num_tokens, max_shift=2.05, base_shift=0.95, stretch=True, terminal=0.1):
    """LTX2Scheduler::execute -> list of steps+1 f32 sigmas (host, no GPU needed)."""
    import numpy as np
    out = np.empty(steps + 1, np.float32)
    rc = lib().ltx_scheduler_execute(steps, num_tokens, max_shift, base_shift, int(stretch), terminal,
                                     out.ctypes.data_as(ctypes.c_void_p))
    if rc:
        raise LtxError(rc, "ltx_scheduler_execute")
    return out


def target_positions(frames, height, width, batch=1, scale=(8, 32, 32), fps=24.0):
    """make_target_positions -> np.float32 [batch, 3, F*H*W, 2] (host, no GPU needed)."""
    import numpy as np
    out = np.empty((batch, 3, frames * height * width, 2), np.float32)
    rc = lib().ltx_target_positions(frames, height, width, batch, *scale, fps, out.ctypes.data_as(ctypes.c_void_p))
    if rc:
        raise LtxError(rc, "ltx_target_positions")
    return out


def reference_positions(frames, height, width, batch=1, first_latent_frame=0, scale=(8, 32, 32), fps=24.0,
                        temporal_scale_factor=1, downscale_factor=1):
    """make_reference_positions -> np.float32 [batch, 3, F*H*W, 2] (host, no GPU needed)."""
    import numpy as np
    out = np.empty((batch, 3, frames * height * width, 2), np.float32)
    rc = lib().ltx_reference_positions(frames, height, width, batch, first_latent_frame, *scale, fps,
                                       temporal_scale_factor, downscale_factor, out.ctypes.data_as(ctypes.c_void_p))
    if rc:
        raise LtxError(rc, "ltx_reference_positions")
    return out


def patchify(ctx: "Context", latent5, tokens):
    B, C, F, H, W = latent5.shape
    ctx.check(lib().ltx_patchify(ctx.h, _ptr(latent5), B, C, F, H, W, _ptr(tokens)), "ltx_patchify")


def unpatchify(ctx: "Context", tokens, latent5):
    B, C, F, H, W = latent5.shape
    ctx.check(lib().ltx_unpatchify(ctx.h, _ptr(tokens), B, C, F, H, W, _ptr(latent5)), "ltx_unpatchify")


NOALLOC_SCRATCH_BYTES = 16 << 20


def dequant_merge_noalloc(stream: int, w_ptr: int, w_dtype: int, has_scale: bool, scale: float, out_features: int,
                          in_features: int, deltas, dst_ptr: int, dst_dtype: int):
    """ltx_dequant_merge_noalloc: the same merge without allocating device memory
    (for callers that cannot call cudaMalloc); raises LtxError with the library's message."""
    n = len(deltas)
    arr = (LoraDelta * max(n, 1))(*[LoraDelta(*d) for d in deltas])
    err = ctypes.create_string_buffer(512)
    rc = lib().ltx_dequant_merge_noalloc(ctypes.c_void_p(stream), ctypes.c_void_p(w_ptr), w_dtype, int(has_scale),
                                         scale, out_features, in_features, arr, n, ctypes.c_void_p(dst_ptr),
                                         dst_dtype, err, len(err))
    if rc != 0:
        raise LtxError(rc, err.value.decode())


def lora_coeff(strength: float, alpha: float, rank: int) -> float:
    return lib().ltx_lora_coeff(strength, alpha, rank)


# ── temporal chunks (crates/ltx-chunk) ─────────────────────────────────────────

def chunk_plan(total: int, chunk_len: int, overlap: int):
    """plan::plan -> [(start, end, real_overlap), ...] (host, no GPU needed).
    Raises LtxError(kind "CHUNK_PLAN") naming the ChunkError variant."""
    n = ctypes.c_int32(0)
    cap = max(1, total // max(1, chunk_len - overlap) + 2)
    arr = (Chunk * cap)()
    rc = lib().ltx_chunk_plan(total, chunk_len, overlap, arr, cap, ctypes.byref(n))
    if rc:
        raise LtxError(rc, lib().ltx_host_last_error().decode())
    return [arr[i].as_tuple() for i in range(n.value)]


def crossfade_weight(offset: int, overlap_len: int) -> float:
    """blend::crossfade_weight (host)."""
    return lib().ltx_crossfade_weight(offset, overlap_len)


def seam_blend(ctx: "Context", outgoing, incoming, dst):
    """Blends overlap frames on the device: tensors [frames, ...] f32 (dst may be incoming)."""
    frames = outgoing.shape[0]
    fv = outgoing.numel() // max(frames, 1)
    ctx.check(lib().ltx_seam_blend(ctx.h, _ptr(outgoing), _ptr(incoming), frames, fv, _ptr(dst)), "ltx_seam_blend")


def chunk_assemble(ctx: "Context", chunk_tensors, chunks, dst):
    """The clip the reference's Blender emits, from per-chunk device tensors [len_n, ...] f32."""
    n = len(chunks)
    ptrs = (ctypes.c_void_p * n)(*[_ptr(t) for t in chunk_tensors])
    arr = (Chunk * n)(*[Chunk(*c) for c in chunks])
    fv = dst.numel() // max(dst.shape[0], 1)
    ctx.check(lib().ltx_chunk_assemble(ctx.h, ptrs, arr, n, fv, _ptr(dst)), "ltx_chunk_assemble")


# ── tensor parallelism ─────────────────────────────────────────────────────────

def comm_unique_id() -> bytes:
    """A fresh communicator id (host only; rank 0 makes it and shares it)."""
    buf = ctypes.create_string_buffer(COMM_ID_BYTES)
    rc = lib().ltx_comm_unique_id(buf, COMM_ID_BYTES)
    if rc:
        raise LtxError(rc, lib().ltx_host_last_error().decode())
    return buf.raw


def share_comm_id(group=None) -> bytes:
    """Rank 0's fresh communicator id, broadcast to every rank of a torch.distributed group."""
    import torch.distributed as dist
    obj = [comm_unique_id() if dist.get_rank(group) == 0 else None]
    dist.broadcast_object_list(obj, src=0, group=group)
    return obj[0]


def init_tensor_parallel(ctx: "Context", group=None):
    """Binds ctx to this process's rank of a torch.distributed group (collective)."""
    import torch.distributed as dist
    rank, ws = dist.get_rank(group), dist.get_world_size(group)
    if ws > 1:
        ctx.init_comm(share_comm_id(group), ws, rank)


def cfg_tp_layout(world_size: int, rank: int):
    """CFG-parallel x tensor-parallel placement of `rank` among `world_size` (even)
    GPUs: ranks [0, n/2) run the conditional pass, [n/2, n) the unconditional one,
    each half one tensor-parallel group; rank r pairs with r + n/2.
    Returns (cfg_rank, tp_size, tp_rank, tp_group_ranks, pair_ranks)."""
    if world_size < 2 or world_size % 2:
        raise ValueError(f"CFG-parallel needs an even number of ranks, not {world_size}")
    half = world_size // 2
    cfg_rank, tp_rank = divmod(rank, half)
    return (cfg_rank, half, tp_rank, list(range(cfg_rank * half, cfg_rank * half + half)),
            [tp_rank, tp_rank + half])


def init_cfg_tensor_parallel(ctx: "Context"):
    """Binds ctx to its CFG pair and (for more than 2 ranks) its tensor-parallel group,
    over the default torch.distributed group; the ids travel over torch.distributed.
    Every rank creates every subgroup in the same order (new_group is collective)."""
    import torch.distributed as dist
    ws, rank = dist.get_world_size(), dist.get_rank()
    cfg_rank, half, tp_rank, tp_ranks, pair = cfg_tp_layout(ws, rank)
    tp_groups = [dist.new_group(list(range(g * half, g * half + half))) for g in range(2)]
    pair_groups = [dist.new_group([r, r + half]) for r in range(half)]
    if half > 1:
        g = tp_groups[cfg_rank]
        obj = [comm_unique_id() if rank == tp_ranks[0] else None]
        dist.broadcast_object_list(obj, src=tp_ranks[0], group=g)
        ctx.init_comm(obj[0], half, tp_rank)
    g = pair_groups[tp_rank]
    obj = [comm_unique_id() if rank == pair[0] else None]
    dist.broadcast_object_list(obj, src=pair[0], group=g)
    ctx.init_cfg_comm(obj[0], cfg_rank)
    return cfg_rank, half, tp_rank
