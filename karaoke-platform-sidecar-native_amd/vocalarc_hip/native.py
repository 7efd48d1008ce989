"""ctypes binding of lib/libvocalarc_hip.so (include/vocalarc_hip.h and
include/native_gpu.h).

Device buffers are passed as raw pointers; the tests and the benchmark use
torch tensors on cuda:0 for device memory and streams.  There is no fallback:
if the library is missing the import of `lib()` raises.
"""

from __future__ import annotations

import ctypes
import os
import weakref
from pathlib import Path

from .dims import CDims, ModelDims, to_c

PKG = Path(__file__).resolve().parent.parent
# VOCALARC_HIP_LIB names another build of the library (e.g. to compare two)
LIB_PATH = Path(os.environ.get("VOCALARC_HIP_LIB", PKG / "lib" / "libvocalarc_hip.so"))

EPI_STORE, EPI_GELU, EPI_TANH, EPI_RESIDUAL, EPI_GEGLU = range(5)
PRECISION_FP32, PRECISION_BF16, PRECISION_FP32_MFMA = 0, 1, 2
BF16_A, BF16_C, BF16_STAGED = 1, 2, 4  # vh_gemm_bf16 operand flags; STAGED forces the register-staged kernel
ATT_OUT_BF16, ATT_BF16, ATT_SPLIT, ATT_H2, ATT_OUT_H2 = 1, 2, 4, 8, 16  # vh_attention flags
NOALLOC_MAX_LENGTH = 4096  # VH_NOALLOC_MAX_LENGTH
TYPE_FP32, TYPE_BF16 = 0, 1  # VH_TYPE_*
CACHE_BF16, CACHE_INT8, CACHE_BLOCK = 0, 1, 16  # VH_CACHE_*
SPEC_REFERENCE, SPEC_FRAME_MAJOR = 0, 1  # spectrum layouts: [F][C][T][2] / [C][T][F][2]

_P = ctypes.c_void_p
_I = ctypes.c_int
_I64 = ctypes.c_int64
_lib = None


class CCross(ctypes.Structure):
    """vh_cross"""
    _fields_ = ([(n, _I) for n in ("type", "sequences", "heads", "kv_heads", "query_length", "key_length", "causal")] +
                [("scale", ctypes.c_float)] +
                [(n, _I64 * 3) for n in ("q_strides", "k_strides", "v_strides", "out_strides")] +
                [(n, _P) for n in ("query_lengths", "key_lengths", "query_start", "bias_table")] +
                [(n, _I) for n in ("buckets", "max_distance", "bidirectional")])


class CRotaryAngles(ctypes.Structure):
    """vh_rotary_angles"""
    _fields_ = [("base", ctypes.c_double), ("factor", ctypes.c_double), ("original", _I), ("low", ctypes.c_double),
                ("high", ctypes.c_double), ("magnitude", ctypes.c_double)]


class CRotary(ctypes.Structure):
    """vh_rotary"""
    _fields_ = [("dim", _I), ("interleaved", _I), ("positions", _I), ("table", _P)]


class CRotaryRows(ctypes.Structure):
    """vh_rotary_rows"""
    _fields_ = ([(n, _I) for n in ("type", "sequences", "length", "heads", "head_dim")] +
                [("x_strides", _I64 * 3), ("y_strides", _I64 * 3), ("start", _P)])


class CCache(ctypes.Structure):
    """vh_cache"""
    _fields_ = ([(n, _I) for n in ("type", "kv_heads", "head_dim", "page_tokens", "pages", "sequences", "table_pages")] +
                [("pool", _P), ("table", _P)])


class CCacheRows(ctypes.Structure):
    """vh_cache_rows"""
    _fields_ = [("type", _I), ("length", _I), ("k_strides", _I64 * 3), ("v_strides", _I64 * 3), ("start", _P), ("lengths", _P)]


class CCacheQueries(ctypes.Structure):
    """vh_cache_queries"""
    _fields_ = ([(n, _I) for n in ("type", "heads", "length", "causal", "most_keys")] + [("scale", ctypes.c_float)] +
                [("q_strides", _I64 * 3), ("out_strides", _I64 * 3)] +
                [(n, _P) for n in ("query_lengths", "key_lengths", "start")])


class CBeam(ctypes.Structure):
    """vh_beam"""
    _fields_ = ([(n, _I) for n in ("type", "sequences", "beams", "vocab", "picks", "end_token")] + [("strides", _I64 * 2)])


# Signatures (result, arguments) of every entry point declared in
# include/vocalarc_hip.h (vh_*) and include/native_gpu.h (native_gpu_*).
SIGNATURES = {
    "vh_create": (_P, []), "vh_destroy": (None, [_P]), "vh_set_stream": (_I, [_P, _P]),
    "vh_synchronize": (_I, [_P]), "vh_last_error": (ctypes.c_char_p, []), "vh_device_name": (ctypes.c_char_p, [_P]),
    "vh_rmsnorm": (_I, [_P, _I64, _I, _P, _P, _P]), "vh_rmsnorm_bf16": (_I, [_P, _I64, _I, _P, _P, _P]),
    "vh_rmsnorm_h2": (_I, [_P, _I64, _I, _P, _P, _P, _P]),
    "vh_softmax_rows": (_I, [_P, _I64, _I, _P, _P]),
    "vh_rope_bhld": (_I, [_P, _I64, _I, _I, _P]),
    "vh_geglu": (_I, [_P, _I64, _I, _P, _P]),
    "vh_residual_add": (_I, [_P, _I64, _P, _P]),
    "vh_gemm": (_I, [_P, _I64, _I, _I, _P, _I, _P, _I, _P, _P, _I, _I]),
    "vh_gemm_bf16": (_I, [_P, _I64, _I, _I, _P, _I, _P, _I, _P, _P, _I, _I, _I]),
    "vh_gemm_split": (_I, [_P, _I64, _I, _I, _P, _I, _P, _P, _P, _I, _I]),
    "vh_split_bytes": (ctypes.c_size_t, [_I, _I]),
    "vh_split_weights": (_I, [_P, _I, _I, _P, _I, _P]),
    "vh_gemm_h2": (_I, [_P, _I64, _I, _I, _P, _I, ctypes.c_float, _P, _P, _P, _I, _I, _I]),
    "vh_gemm_h2_ex": (_I, [_P, _I64, _I, _I, _P, _I, _P, _P, _P, _P, _I, _I, _I, _P, _P]),
    "vh_h2_bytes": (ctypes.c_size_t, [_I, _I]),
    "vh_split_weights_h2": (_I, [_P, _I, _I, _P, _I, _P]),
    "vh_operand_bounds": (_I, [_P, _P, _I, _P, _I, _P, _I, _P]),
    "vh_to_bf16": (_I, [_P, _I64, _I, _P, _P, _I]),
    "vh_attention": (_I, [_P, _I, _I, _I, _P, _P, _I, _I]),
    "vh_attention_noalloc": (_I, [_P, _I, _I, _I, _P, _P, _I, _I]),
    "vh_layernorm": (_I, [_P, _I, _I64, _I, _P, _I64, _P, _P, ctypes.c_float, _P, _I64, _P]),
    "vh_layernorm_backward": (_I, [_P, _I, _I64, _I, _P, _I64, _P, _I64, _P, _P, _P, _I64, _P, _P, _P]),
    "vh_layernorm_workspace_bytes": (ctypes.c_size_t, [_I64, _I]),
    "vh_cross_attention": (_I, [_P, ctypes.POINTER(CCross), _P, _P, _P, _P, _P, _P]),
    "vh_cross_attention_backward": (_I, [_P, ctypes.POINTER(CCross)] + [_P] * 11),
    "vh_cross_saved_bytes": (ctypes.c_size_t, [ctypes.POINTER(CCross)]),
    "vh_cross_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(CCross), _I]),
    "vh_relative_bucket": (_I, [_I, _I, _I, _I]),
    "vh_rotary_table": (_I, [_P, ctypes.POINTER(CRotaryAngles), _I, _I, _P]),
    "vh_rotary_apply": (_I, [_P, ctypes.POINTER(CRotary), ctypes.POINTER(CRotaryRows), _P, _P, _I]),
    "vh_cache_bytes": (ctypes.c_size_t, [ctypes.POINTER(CCache)]),
    "vh_cache_append": (_I, [_P, ctypes.POINTER(CCache), ctypes.POINTER(CCacheRows), ctypes.POINTER(CRotary), _P, _P]),
    "vh_cache_read": (_I, [_P, ctypes.POINTER(CCache), ctypes.POINTER(CCacheRows), _P, _P]),
    "vh_cache_attention": (_I, [_P, ctypes.POINTER(CCache), ctypes.POINTER(CCacheQueries), ctypes.POINTER(CRotary), _P, _P, _P]),
    "vh_cache_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(CCache), ctypes.POINTER(CCacheQueries)]),
    "vh_cache_reorder": (_I, [_P, ctypes.POINTER(CCache), _I] + [_P] * 5),
    "vh_beam_select": (_I, [_P, ctypes.POINTER(CBeam)] + [_P] * 8),
    "vh_beam_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(CBeam)]),
    "vh_model_load": (_P, [_P, ctypes.POINTER(CDims), _P, ctypes.c_size_t]),
    "vh_model_free": (None, [_P]), "vh_model_set_precision": (_I, [_P, _I]),
    "vh_transformer": (_I, [_P, _P, _I, _I, _P, _I, _I]),
    "vh_stft": (_I, [_P, _P, _P, _I, _P, _I]),
    "vh_istft": (_I, [_P, _P, _P, _P, _I, _P, _I]),
    "vh_band_split": (_I, [_P, _P, _P, _I, _P, _I]),
    "vh_mask_estimate": (_I, [_P, _P, _P, _I, _P, _I]),
    "vh_forward": (_I, [_P, _P, _P, _I, _P, _P]),
    "vh_separate": (_I, [_P, _P, _P, _I, _I, _I, _I, _P, _P]),
    "vh_timing_enable": (_I, [_P, ctypes.c_char_p]), "vh_timing_reset": (_I, [_P]),
    "vh_timing_get": (_I, [_P, ctypes.c_char_p, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(_I64)]),
    "native_gpu_create": (_P, []), "native_gpu_destroy": (None, [_P]),
    "native_gpu_matmul": (_I, [_P, _I64, _I, _I, _P, _P, _P, _P]),
    "native_gpu_backend": (ctypes.c_char_p, [_P]), "native_gpu_device": (ctypes.c_char_p, [_P]),
    "native_gpu_uses_full_batches": (_I, [_P]), "native_gpu_can_use_full_batches": (_I, [_P, _I]),
    "native_gpu_transformer": (_I, [_P, _I, _I, _P, _P, _P, _P, _P, _P]),
    "native_gpu_resident_begin": (_I, [_P, _I, _I, _P]),
    "native_gpu_resident_transformer": (_I, [_P, _I, _I, _P]),
    "native_gpu_resident_transpose": (_I, [_P, _I, _I]),
    "native_gpu_resident_end": (_I, [_P, _P]),
    "native_gpu_resident_mask": (_I, [_P, _I, _P, _P, _P, _I]),
}
HARNESS_SYMBOLS = [n for n in SIGNATURES if n.startswith("vh_")]
ABI_SYMBOLS = [n for n in SIGNATURES if n.startswith("native_gpu_")]


class NativeError(RuntimeError):
    pass


def lib():
    """Load the HIP library (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise NativeError(f"{LIB_PATH} is missing: build it with `make -C {PKG}`")
    L = ctypes.CDLL(str(LIB_PATH))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def last_error() -> str:
    e = lib().vh_last_error()
    return e.decode() if e else ""


def _ok(rc: int, what: str) -> None:
    if not rc:
        raise NativeError(f"{what} failed: {last_error()}")


def ptr(t) -> int:
    """Device (or host) address of a torch tensor / numpy array."""
    if hasattr(t, "data_ptr"):
        return t.data_ptr()
    return t.ctypes.data


def _opt(t):
    """ptr(t), or a null pointer for None."""
    return ptr(t) if t is not None else None


def _out_cols(N: int, epilogue: int) -> int:
    """Output columns of a linear with N weight rows (GELU-GLU halves them)."""
    return N // 2 if epilogue == EPI_GEGLU else N


def _att_flags(out_bf16: bool, bf16: bool, split: bool, h2: bool) -> int:
    return ((ATT_OUT_BF16 if out_bf16 else 0) | (ATT_BF16 if bf16 else 0) | (ATT_SPLIT if split else 0) |
            (ATT_H2 if h2 else 0))


class Context:
    """vh_context bound to a HIP stream (default: torch's current stream)."""

    def __init__(self, stream: int | None = None):
        self.models = weakref.WeakSet()  # vh_destroy frees them with the context
        self.h = lib().vh_create()
        if not self.h:
            raise NativeError(f"vh_create failed: {last_error()}")
        if stream is None:
            try:
                import torch
                stream = torch.cuda.current_stream().cuda_stream
            except Exception:  # noqa: BLE001 - no torch: the null stream
                stream = 0
        _ok(lib().vh_set_stream(self.h, stream), "vh_set_stream")

    def close(self):
        if self.h:
            for m in list(self.models):  # freed by vh_destroy below
                m.h = None
            lib().vh_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001
            pass

    @property
    def device_name(self) -> str:
        return lib().vh_device_name(self.h).decode()

    def sync(self):
        _ok(lib().vh_synchronize(self.h), "vh_synchronize")

    def set_stream(self, stream: int):
        """Issue the context's work on the HIP stream handle `stream` (0: the null stream)."""
        _ok(lib().vh_set_stream(self.h, stream), "vh_set_stream")

    # -- isolated kernels (device pointers) --
    def rmsnorm(self, x, gamma, y, rows: int, dim: int):
        _ok(lib().vh_rmsnorm(self.h, rows, dim, ptr(x), ptr(gamma), ptr(y)), "vh_rmsnorm")

    def rmsnorm_bf16(self, x, gamma, y, rows: int, dim: int):
        _ok(lib().vh_rmsnorm_bf16(self.h, rows, dim, ptr(x), ptr(gamma), ptr(y)), "vh_rmsnorm_bf16")

    def rmsnorm_h2(self, x, gamma, bound, y, rows: int, dim: int):
        """y as h2 rows (fp16 pieces of y * 2^e, e from the device float bound[0]) for gemm_h2(a_rows=True)."""
        _ok(lib().vh_rmsnorm_h2(self.h, rows, dim, ptr(x), ptr(gamma), ptr(bound), ptr(y)), "vh_rmsnorm_h2")

    def softmax_rows(self, x, y, rows: int, length: int):
        _ok(lib().vh_softmax_rows(self.h, rows, length, ptr(x), ptr(y)), "vh_softmax_rows")

    def rope_bhld(self, x, bh: int, length: int, dim_head: int = 64):
        _ok(lib().vh_rope_bhld(self.h, bh, length, dim_head, ptr(x)), "vh_rope_bhld")

    def geglu(self, x, y, rows: int, width: int):
        _ok(lib().vh_geglu(self.h, rows, width, ptr(x), ptr(y)), "vh_geglu")

    def residual_add(self, x, r, n: int):
        _ok(lib().vh_residual_add(self.h, n, ptr(x), ptr(r)), "vh_residual_add")

    def gemm(self, A, W, C, M: int, N: int, K: int, bias=None, epilogue: int = EPI_STORE,
             lda: int | None = None, ldw: int | None = None, ldc: int | None = None):
        _ok(lib().vh_gemm(self.h, M, N, K, ptr(A), lda or K, ptr(W), ldw or K,
                          _opt(bias), ptr(C),
                          ldc or _out_cols(N, epilogue), epilogue), "vh_gemm")

    def gemm_bf16(self, A, Wh, C, M: int, N: int, K: int, ldw: int, bias=None, epilogue: int = EPI_STORE,
                  lda: int | None = None, ldc: int | None = None, flags: int = 0):
        """Wh: bf16 weight copy [N][ldw] (see to_bf16); flags: BF16_A / BF16_C operand types, BF16_STAGED."""
        _ok(lib().vh_gemm_bf16(self.h, M, N, K, ptr(A), lda or K, ptr(Wh), ldw,
                               _opt(bias), ptr(C),
                               ldc or _out_cols(N, epilogue), epilogue, flags), "vh_gemm_bf16")

    @staticmethod
    def split_bytes(N: int, K: int) -> int:
        """Bytes of the bf16 pieces of an N x K weight (see split_weights)."""
        return int(lib().vh_split_bytes(N, K))

    def split_weights(self, W, Ws, N: int, K: int, ldw_in: int | None = None):
        """fp32 W [N][ldw_in] -> its tile-major bf16 pieces Ws (split_bytes(N, K) bytes)."""
        _ok(lib().vh_split_weights(self.h, N, K, ptr(W), ldw_in or K, ptr(Ws)), "vh_split_weights")

    def gemm_split(self, A, Ws, C, M: int, N: int, K: int, bias=None, epilogue: int = EPI_STORE,
                   lda: int | None = None, ldc: int | None = None):
        """fp32-accurate linear on bf16 matrix cores; Ws from split_weights."""
        _ok(lib().vh_gemm_split(self.h, M, N, K, ptr(A), lda or K, ptr(Ws),
                                _opt(bias), ptr(C),
                                ldc or _out_cols(N, epilogue), epilogue), "vh_gemm_split")

    @staticmethod
    def h2_bytes(N: int, K: int) -> int:
        """Bytes of the fp16 pieces of an N x K weight (see split_weights_h2)."""
        return int(lib().vh_h2_bytes(N, K))

    def split_weights_h2(self, W, Wp, N: int, K: int, ldw_in: int | None = None):
        """fp32 W [N][ldw_in] -> max|W| and the tile-major fp16 pieces Wp (h2_bytes(N, K) bytes)."""
        _ok(lib().vh_split_weights_h2(self.h, N, K, ptr(W), ldw_in or K, ptr(Wp)), "vh_split_weights_h2")

    def gemm_h2(self, A, Wp, C, M: int, N: int, K: int, bias=None, epilogue: int = EPI_STORE,
                lda: int | None = None, ldc: int | None = None, a_bound: float = 0.0, a_rows: bool = False):
        """fp32-accurate linear on fp16 matrix cores; Wp from split_weights_h2; a_bound bounds |A| (0: max|A|);
        a_rows: A is given as h2 rows split with a_bound (rmsnorm_h2)."""
        _ok(lib().vh_gemm_h2(self.h, M, N, K, ptr(A), lda or K, float(a_bound), ptr(Wp),
                             _opt(bias), ptr(C),
                             ldc or _out_cols(N, epilogue), epilogue, 1 if a_rows else 0),
            "vh_gemm_h2")

    def gemm_h2_ex(self, A, Wp, C, M: int, N: int, K: int, a_bound, bias=None, epilogue: int = EPI_STORE,
                   lda: int | None = None, ldc: int | None = None, row_norm: bool = False, zero_slot=None,
                   amax=None):
        """gemm_h2 with a device bound a_bound; row_norm: C = op(rms(A) (A Wp^T) + bias) with the RMSNorm gain folded
        into Wp; zero_slot set to 0; amax (residual epilogue) raised to max|C| (see vh_gemm_h2_ex)."""
        _ok(lib().vh_gemm_h2_ex(self.h, M, N, K, ptr(A), lda or K, ptr(a_bound), ptr(Wp), _opt(bias), ptr(C),
                                ldc or _out_cols(N, epilogue), epilogue, 2 if row_norm else 0, _opt(zero_slot),
                                _opt(amax)),
            "vh_gemm_h2_ex")

    def operand_bounds(self, gamma, D: int, out, W=None, N: int = 0, bias=None, square: bool = False):
        """Device bounds out[0..1] of the A operands after an RMSNorm with gain gamma (see vh_operand_bounds)."""
        _ok(lib().vh_operand_bounds(self.h, ptr(gamma), D, _opt(W), N,
                                    _opt(bias), 1 if square else 0, ptr(out)),
            "vh_operand_bounds")

    def to_bf16(self, src, dst, rows: int, cols: int, ld: int):
        _ok(lib().vh_to_bf16(self.h, rows, cols, ptr(src), ptr(dst), ld), "vh_to_bf16")

    def attention(self, qkv, out, sequences: int, length: int, heads: int, rotary: bool = True, out_bf16: bool = False,
                  bf16: bool = False, split: bool = False, h2: bool = False, out_h2: bool = False):
        """bf16: qkv is bf16 and the bf16-MFMA kernel runs; out_bf16: out is bf16; split: fp32 accuracy on the
        bf16 matrix cores (three-piece splits, length > 64); h2: fp32 accuracy on the fp16 matrix cores (two-piece
        splits, scales from max|qkv|, any length); out_h2 (with h2): out as h2 rows scaled from max|qkv|."""
        _ok(lib().vh_attention(self.h, sequences, length, heads, ptr(qkv), ptr(out), int(rotary),
                               _att_flags(out_bf16, bf16, split, h2) | (ATT_OUT_H2 if out_h2 else 0)), "vh_attention")

    def attention_noalloc(self, qkv, out, sequences: int, length: int, heads: int, rotary: bool = True,
                          out_bf16: bool = False, bf16: bool = False, split: bool = False, h2: bool = False) -> int:
        """vh_attention_noalloc (no device allocation; length <= NOALLOC_MAX_LENGTH); returns its status."""
        return lib().vh_attention_noalloc(self.h, sequences, length, heads, ptr(qkv), ptr(out), int(rotary),
                                          _att_flags(out_bf16, bf16, split, h2))

    def layernorm(self, x, gamma, beta, y, rows: int, dim: int, eps: float = 1e-5, stats=None, ldx: int | None = None,
                  ldy: int | None = None, bf16: bool = False):
        """Layer norm rows; bf16: x and y are bf16; stats [rows][2] receives (mean, rstd) for the backward pass."""
        _ok(lib().vh_layernorm(self.h, int(bf16), rows, dim, ptr(x), ldx or dim, ptr(gamma), _opt(beta), eps, ptr(y),
                               ldy or dim, _opt(stats)), "vh_layernorm")

    @staticmethod
    def layernorm_workspace_bytes(rows: int, dim: int) -> int:
        """Bytes of layernorm_backward's workspace."""
        n = int(lib().vh_layernorm_workspace_bytes(rows, dim))
        _ok(n, "vh_layernorm_workspace_bytes")
        return n

    def layernorm_backward(self, dy, x, gamma, stats, dx, rows: int, dim: int, dgamma=None, dbeta=None, workspace=None,
                           lddy: int | None = None, ldx: int | None = None, lddx: int | None = None,
                           bf16: bool = False):
        """dx, and dgamma and dbeta where given (then with the workspace, layernorm_workspace_bytes(rows, dim))."""
        _ok(lib().vh_layernorm_backward(self.h, int(bf16), rows, dim, ptr(dy), lddy or dim, ptr(x), ldx or dim,
                                        ptr(gamma), ptr(stats), ptr(dx), lddx or dim, _opt(dgamma), _opt(dbeta),
                                        _opt(workspace)), "vh_layernorm_backward")

    # -- timing --
    def timing(self, classes: str | None = "*"):
        """Time the named kernel classes (comma list, "*" = all, None = off)."""
        _ok(lib().vh_timing_enable(self.h, classes.encode() if classes else None), "vh_timing_enable")

    def timing_reset(self):
        _ok(lib().vh_timing_reset(self.h), "vh_timing_reset")

    def timing_get(self, name: str) -> tuple[float, int]:
        ms = ctypes.c_double(0.0)
        n = _I64(0)
        if not lib().vh_timing_get(self.h, name.encode(), ctypes.byref(ms), ctypes.byref(n)):
            return 0.0, 0
        return ms.value, n.value


def _reshapes(shape, like) -> bool:
    """Whether a contiguous tensor of `shape` has the elements of a contiguous one of `like` in the same places for a
    reader of either: each dimension joins or splits neighbours of the other's, in their order (dimensions of 1 aside)."""
    a, b = [n for n in shape if n != 1], [n for n in like if n != 1]
    if 0 in a or 0 in b:
        return 0 in a and 0 in b
    while a and b:
        n, m = a.pop(0), b.pop(0)
        many = b if n > m else a  # whose dimensions are joined to the wider one
        wide, joined = max(n, m), min(n, m)
        while joined < wide and many:
            joined *= many.pop(0)
        if joined != wide:
            return False
    return not a and not b


class CrossAttention:
    """The layout of an attention over another sequence's states (vh_cross), for tensors q [S][Lq][H][64], k and v
    [S][Lk][KV heads][64] and out as q, of any strides that vh_cross takes.  Later calls may pass other tensors of the
    same layout (dq, dk, dv as q, k, v and dout as out); contiguous ones also in a shape that joins or splits neighbouring
    dimensions ([S * Lq][H * 64]).  query_lengths, key_lengths, query_start: int32 device tensors [S]; bias_table: fp32
    [buckets][H].  Shapes, types, devices and the buffers' sizes are checked here; what the library takes of strides and
    sizes by it."""

    def __init__(self, ctx: Context, q, k, v, out, *, causal: bool = False, scale: float = 0.125, query_lengths=None,
                 key_lengths=None, query_start=None, bias_table=None, max_distance: int = 128,
                 bidirectional: bool = True):
        import torch
        S, Lq, H, D = q.shape
        if q.dtype not in (torch.float32, torch.bfloat16) or D != 64 or k.dim() != 4 or k.shape[0] != S or \
                k.shape[3] != 64 or tuple(v.shape) != tuple(k.shape) or tuple(out.shape) != tuple(q.shape) or \
                len({t.dtype for t in (q, k, v, out)}) != 1:
            raise NativeError("CrossAttention: q and out [S][Lq][H][64], k and v [S][Lk][KV][64], all fp32 or all bf16")
        if any(t.stride(3) != 1 for t in (q, k, v, out)):
            raise NativeError("CrossAttention: a head's 64 elements are consecutive")
        if any(t is not None and t.device != q.device
               for t in (k, v, out, query_lengths, key_lengths, query_start, bias_table)):
            raise NativeError("CrossAttention: tensors on different devices")
        for t in (query_lengths, key_lengths, query_start):
            if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (S,) or not t.is_contiguous()):
                raise NativeError("CrossAttention: lengths and starts are contiguous int32 [S]")
        if bias_table is not None and (bias_table.dtype != torch.float32 or bias_table.dim() != 2 or
                                       bias_table.shape[1] != H or not bias_table.is_contiguous()):
            raise NativeError("CrossAttention: the bias table is contiguous fp32 [buckets][H]")
        self.ctx = ctx
        self._kept = (query_lengths, key_lengths, query_start, bias_table)
        self.c = CCross(int(q.dtype == torch.bfloat16), S, H, k.shape[2], Lq, k.shape[1], int(causal), scale)
        for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
            setattr(self.c, name + "_strides", (_I64 * 3)(*t.stride()[:3]))
        for name, t in zip(("query_lengths", "key_lengths", "query_start", "bias_table"), self._kept):
            setattr(self.c, name, _opt(t))
        if bias_table is not None:
            self.c.buckets, self.c.max_distance = bias_table.shape[0], max_distance
            self.c.bidirectional = int(bidirectional)
        self._ref = ctypes.byref(self.c)
        self._like = {n: (t.dtype, t.shape, t.stride(), t.device)
                      for n, t in (("q", q), ("k", k), ("v", v), ("out", out))}
        self._elsewhere = None if q.device == torch.device("cuda:0") else q.device  # every context's GPU is the first
        self._packed = {"q": q.is_contiguous(), "k": k.is_contiguous(), "v": v.is_contiguous(), "out": out.is_contiguous()}
        self._bytes = {}

    def _tensor(self, name, like, t):
        """t's address; laid out as `like` was, or (of contiguous ones) a shape that joins or splits its dimensions."""
        dtype, shape, stride, device = self._like[like]
        if t.shape == shape:
            same = t.stride() == stride or not t.numel() or \
                all(n == 1 or a == b for n, a, b in zip(shape, t.stride(), stride))
        else:
            same = t.is_contiguous() and self._packed[like] and _reshapes(t.shape, shape)
        if not same or t.dtype != dtype or t.device != device:
            raise NativeError(f"CrossAttention: {name} is not laid out as {like} was")
        return t.data_ptr()

    def _buffer(self, name, t, size, *key):
        if t is None:
            return None
        if key not in self._bytes:
            self._bytes[key] = size(*key[1:])
        if t.numel() * t.element_size() < self._bytes[key] or not t.is_contiguous() or t.device != self._like["q"][3]:
            raise NativeError(f"CrossAttention: {name} has fewer than {self._bytes[key]} bytes in a row, or is on another "
                              "device")
        return t.data_ptr()

    def _on_gpu(self):
        if self._elsewhere is not None:
            raise NativeError(f"CrossAttention: the tensors are on {self._elsewhere}, the context's work runs on cuda:0")

    def saved_bytes(self) -> int:
        n = int(lib().vh_cross_saved_bytes(self._ref))
        _ok(n, "vh_cross_saved_bytes")
        return n

    def workspace_bytes(self, backward: bool = False) -> int:
        n = int(lib().vh_cross_workspace_bytes(self._ref, int(backward)))
        _ok(n, "vh_cross_workspace_bytes")
        return n

    def forward(self, q, k, v, out, saved=None, workspace=None):
        f = self._tensor
        args = (f("q", "q", q), f("k", "k", k), f("v", "v", v), f("out", "out", out),
                self._buffer("saved", saved, self.saved_bytes, "saved"),
                self._buffer("workspace", workspace, self.workspace_bytes, "workspace", False))
        self._on_gpu()
        _ok(lib().vh_cross_attention(self.ctx.h, self._ref, *args), "vh_cross_attention")

    def backward(self, q, k, v, out, saved, dout, dq, dk=None, dv=None, dbias=None, workspace=None):
        f = self._tensor
        table = self._kept[3]
        if dbias is not None and table is not None and \
                ((dbias.dtype, dbias.shape, dbias.device) != (table.dtype, table.shape, table.device) or
                 not dbias.is_contiguous()):
            raise NativeError("CrossAttention: dbias is not laid out as the bias table")
        args = (f("q", "q", q), f("k", "k", k), f("v", "v", v), f("out", "out", out),
                self._buffer("saved", saved, self.saved_bytes, "saved"), f("dout", "out", dout), f("dq", "q", dq),
                f("dk", "k", dk) if dk is not None else None, f("dv", "v", dv) if dv is not None else None, _opt(dbias),
                self._buffer("workspace", workspace, self.workspace_bytes, "workspace", True))
        self._on_gpu()
        _ok(lib().vh_cross_attention_backward(self.ctx.h, self._ref, *args), "vh_cross_attention_backward")


class _Plan:
    """What the bindings below share: later calls' tensors and buffers are checked against the ones that a layout was made
    of, before the library sees them."""

    what = ""

    def _keep(self, **tensors):
        self._like = {n: (t.dtype, t.shape, t.stride(), t.device) for n, t in tensors.items()}

    def _refuse(self, text):
        raise NativeError(f"{self.what}: {text}")

    def _same_device(self, tensors):
        devices = {t.device for t in tensors if t is not None}
        if len(devices) > 1:
            self._refuse("tensors on different devices")

    def _ints(self, name, t, *shape):
        import torch
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous()):
            self._refuse(f"{name} is a contiguous int32 tensor {list(shape)}")

    def _activations(self, **tensors):
        import torch
        if any(t.dtype not in (torch.float32, torch.bfloat16) for t in tensors.values()) or \
                len({t.dtype for t in tensors.values()}) != 1:
            self._refuse(f"{', '.join(tensors)}: all fp32 or all bf16")
        if any(t.shape[-1] > 1 and t.stride(-1) != 1 for t in tensors.values()):
            self._refuse("a row's elements are consecutive")

    def _whole(self, name, t, dtype, shape, device):
        """t's address, where it is a contiguous tensor of that type and shape on that device."""
        if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
            self._refuse(f"{name} is a contiguous {dtype} tensor {list(shape)} on {device}")
        return t.data_ptr()

    def _tensor(self, name, like, t):
        """t's address, where it is laid out as `like` was."""
        if (t.dtype, t.shape, t.stride(), t.device) == self._like[like]:
            return t.data_ptr()
        dtype, shape, stride, device = self._like[like]
        if t.dtype != dtype or t.shape != shape or t.device != device or \
                (t.stride() != stride and t.numel() and any(n > 1 and a != b for n, a, b in zip(shape, t.stride(), stride))):
            self._refuse(f"{name} is not laid out as {like} was")
        return t.data_ptr()

    def _buffer(self, name, t, nbytes, device):
        if t is None:
            return None
        if t.numel() * t.element_size() < nbytes or not t.is_contiguous() or t.device != device:
            self._refuse(f"{name} has fewer than {nbytes} bytes in a row, or is on another device")
        return t.data_ptr()

    def _on_gpu(self, device):
        if device.type != "cuda" or device.index:  # every context's GPU is the first
            self._refuse(f"the tensors are on {device}, the context's work runs on cuda:0")


_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch
        _torch_module = torch
    return _torch_module


def _rotary_ref(r):
    return r._ref if r is not None else None


class Rotary(_Plan):
    """A rotation (vh_rotary) with its table of `positions` rows, on the context's GPU.  dim: the head's leading dims that
    turn; interleaved: pairs of neighbours, else of the halves; with a factor over 1 the angles are scaled (see
    vh_rotary_angles)."""

    what = "Rotary"

    def __init__(self, ctx: Context, positions: int, dim: int, *, interleaved: bool = False, base: float = 10000.0,
                 factor: float = 1.0, original: int = 0, low: float = 1.0, high: float = 32.0, magnitude: float = 1.0):
        import torch
        if positions < 1 or dim < 2 or dim > 256 or dim % 2:
            self._refuse(f"{positions} positions (from 1) of {dim} dims (even, 2 to 256)")
        self.ctx = ctx
        self.table = torch.empty(positions, dim // 2, 2, device="cuda:0")
        self.c = CRotary(dim, int(interleaved), positions, ptr(self.table))
        self._ref = ctypes.byref(self.c)
        angles = CRotaryAngles(base, factor, original, low, high, magnitude)
        _ok(lib().vh_rotary_table(ctx.h, ctypes.byref(angles), dim, positions, ptr(self.table)), "vh_rotary_table")
        self._rows = {}

    def apply(self, x, y, start=None, backward: bool = False):
        """y [S][L][H][D] = x turned from position start[s] (int32 device tensor [S], None: 0) on; y may be x.  backward:
        by the transpose, which takes y's gradient to x's."""
        key = (x.dtype, x.shape, x.stride(), y.dtype, y.shape, y.stride())
        rows = self._rows.get(key)
        if rows is None:
            if x.dim() != 4 or x.shape[3] < self.c.dim or y.shape != x.shape:
                self._refuse(f"x and y are [S][L][H][D] with D from {self.c.dim}")
            self._activations(x=x, y=y)
            S, L, H, D = x.shape
            c = CRotaryRows(int(x.element_size() == 2), S, L, H, D, (_I64 * 3)(*x.stride()[:3]), (_I64 * 3)(*y.stride()[:3]))
            rows = c, ctypes.byref(c), (S,)
            self._rows = {**(self._rows if len(self._rows) < 64 else {}), key: rows}
        c, ref, sequences = rows
        device = x.device
        if y.device != device:
            self._refuse("tensors on different devices")
        c.start = self._whole("start", start, _torch().int32, sequences, device) if start is not None else None
        self._on_gpu(device)
        _ok(lib().vh_rotary_apply(self.ctx.h, self._ref, ref, x.data_ptr(), y.data_ptr(), int(backward)), "vh_rotary_apply")


class PagedCache(_Plan):
    """A pool of pages of keys and values (vh_cache): kind "bf16", or "int8" with a scale for every 16 tokens and head.
    Tables [sequences][pages of one], int32, say which pages a sequence has, and are the caller's."""

    what = "PagedCache"

    def __init__(self, ctx: Context, kind: str, *, kv_heads: int, head_dim: int, page_tokens: int, pages: int,
                 device: str = "cuda:0"):
        import torch
        if kind not in ("bf16", "int8"):
            self._refuse(f"a cache of {kind!r}: bf16 or int8")
        self.ctx = ctx
        self.c = CCache(CACHE_INT8 if kind == "int8" else CACHE_BF16, kv_heads, head_dim, page_tokens, pages)
        n = int(lib().vh_cache_bytes(ctypes.byref(self.c)))
        _ok(n, "vh_cache_bytes")
        self.pool = torch.empty(n, dtype=torch.uint8, device=device)
        self.c.pool = ptr(self.pool)
        self._view = CCache.from_buffer_copy(self.c)  # reorder's, filled at each call
        self._view_ref = ctypes.byref(self._view)

    def _with(self, table):
        """The cache seen through a table."""
        import torch
        if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous():
            self._refuse("the table is a contiguous int32 tensor [sequences][pages]")
        self._same_device((self.pool, table))
        c = CCache.from_buffer_copy(self.c)
        c.sequences, c.table_pages, c.table = table.shape[0], table.shape[1], ptr(table)
        return c

    def tokens(self, table, k, v, *, start=None, lengths=None, rotary: Rotary | None = None) -> "CacheTokens":
        """Rows k and v [sequences][length][kv_heads][head_dim] to append, or to read into."""
        return CacheTokens(self, table, k, v, start, lengths, rotary)

    def queries(self, table, q, out, *, most_keys: int, causal: bool = False, scale: float = 0.125, query_lengths=None,
                key_lengths=None, query_start=None, rotary: Rotary | None = None) -> "CacheQueries":
        """Queries q and out [sequences][length][heads][head_dim] over the cache."""
        return CacheQueries(self, table, q, out, most_keys, causal, scale, query_lengths, key_lengths, query_start, rotary)

    def reorder(self, table, parents, lengths, spare, table_out, spare_out, *, beams: int):
        """The table's rows in the order of their parents (see vh_cache_reorder)."""
        if table.dim() != 2:
            self._refuse("the table is [sequences][pages]")
        shape, device, int32, v = table.shape, self.pool.device, _torch().int32, self._view
        S = shape[0]
        if beams < 1 or S % beams:
            self._refuse(f"{S} sequences in groups of {beams} beams")
        f = self._whole
        v.sequences, v.table_pages, v.table = S, shape[1], f("table", table, int32, shape, device)
        args = (f("parents", parents, int32, (S,), device), f("lengths", lengths, int32, (S // beams,), device),
                f("spare", spare, int32, (S,), device), f("table_out", table_out, int32, shape, device),
                f("spare_out", spare_out, int32, (S,), device))
        self._on_gpu(device)
        _ok(lib().vh_cache_reorder(self.ctx.h, self._view_ref, beams, *args), "vh_cache_reorder")


class CacheTokens(_Plan):
    """The layout of rows of keys and values and where they are in a paged cache.  Later calls may pass other tensors of the
    same layout; table, start and lengths are read when a call's work runs."""

    what = "CacheTokens"

    def __init__(self, cache: PagedCache, table, k, v, start, lengths, rotary):
        self.ctx, self.c = cache.ctx, cache._with(table)
        if k.dim() != 4 or k.shape[0] != table.shape[0] or tuple(k.shape[2:]) != (self.c.kv_heads, self.c.head_dim) or \
                v.shape != k.shape:
            self._refuse("k and v are [sequences][length][kv_heads][head_dim]")
        self._activations(k=k, v=v)
        self._ints("start", start, k.shape[0])
        self._ints("lengths", lengths, k.shape[0])
        self._same_device((cache.pool, k, v, start, lengths))
        self._kept = (cache, table, start, lengths, rotary)
        self._keep(k=k, v=v)
        self.rows = CCacheRows(int(k.element_size() == 2), k.shape[1], (_I64 * 3)(*k.stride()[:3]), (_I64 * 3)(*v.stride()[:3]),
                               _opt(start), _opt(lengths))
        self._refs = (ctypes.byref(self.c), ctypes.byref(self.rows))
        self._rotary = _rotary_ref(rotary)
        self._device = k.device

    def append(self, k, v):
        """Puts the rows into the cache, keys turned."""
        args = self._tensor("k", "k", k), self._tensor("v", "v", v)
        self._on_gpu(self._device)
        _ok(lib().vh_cache_append(self.ctx.h, *self._refs, self._rotary, *args), "vh_cache_append")

    def read(self, k=None, v=None):
        """What the cache holds at the rows' positions, as it is there, into k and v (either may be None)."""
        args = [self._tensor(n, n, t) if t is not None else None for n, t in (("k", k), ("v", v))]
        self._on_gpu(self._device)
        _ok(lib().vh_cache_read(self.ctx.h, *self._refs, *args), "vh_cache_read")


class CacheQueries(_Plan):
    """The layout of an attention over a paged cache (vh_cache_queries).  Later calls may pass other tensors of the same
    layout; table, lengths and starts are read when a call's work runs, so a captured call follows them."""

    what = "CacheQueries"

    def __init__(self, cache: PagedCache, table, q, out, most_keys, causal, scale, query_lengths, key_lengths, query_start, rotary):
        self.ctx, self.c = cache.ctx, cache._with(table)
        if q.dim() != 4 or q.shape[0] != table.shape[0] or q.shape[3] != self.c.head_dim or out.shape != q.shape:
            self._refuse("q and out are [sequences][length][heads][head_dim]")
        self._activations(q=q, out=out)
        for name, t in (("query_lengths", query_lengths), ("key_lengths", key_lengths), ("query_start", query_start)):
            self._ints(name, t, q.shape[0])
        self._same_device((cache.pool, q, out, query_lengths, key_lengths, query_start))
        self._kept = (cache, table, query_lengths, key_lengths, query_start, rotary)
        self._keep(q=q, out=out)
        self.q = CCacheQueries(int(q.element_size() == 2), q.shape[2], q.shape[1], int(causal), most_keys, scale,
                               (_I64 * 3)(*q.stride()[:3]), (_I64 * 3)(*out.stride()[:3]), _opt(query_lengths),
                               _opt(key_lengths), _opt(query_start))
        self._refs = (ctypes.byref(self.c), ctypes.byref(self.q))
        self._rotary = _rotary_ref(rotary)
        self._device, self._bytes = q.device, None

    def workspace_bytes(self) -> int:
        if self._bytes is None:
            n = int(lib().vh_cache_workspace_bytes(*self._refs))
            _ok(n, "vh_cache_workspace_bytes")
            self._bytes = n
        return self._bytes

    def forward(self, q, out, workspace=None):
        args = (self._tensor("q", "q", q), self._tensor("out", "out", out),
                self._buffer("workspace", workspace, self.workspace_bytes(), self._device))
        self._on_gpu(self._device)
        _ok(lib().vh_cache_attention(self.ctx.h, *self._refs, self._rotary, *args), "vh_cache_attention")


class BeamSearch(_Plan):
    """One step of beam search (vh_beam) for logits [sequences][beams][vocab], fp32 or bf16."""

    what = "BeamSearch"

    def __init__(self, ctx: Context, logits, *, picks: int | None = None, end_token: int = -1):
        if logits.dim() != 3:
            self._refuse("logits are [sequences][beams][vocab]")
        self._activations(logits=logits)
        S, B, V = logits.shape
        self.ctx, self.picks = ctx, B if picks is None else picks
        self._keep(logits=logits)
        self.c = CBeam(int(logits.element_size() == 2), S, B, V, self.picks, end_token, (_I64 * 2)(*logits.stride()[:2]))
        self._ref = ctypes.byref(self.c)
        self._beams, self._picks = (S, B), (S, self.picks)
        self._device, self._bytes = logits.device, None

    def workspace_bytes(self) -> int:
        if self._bytes is None:
            n = int(lib().vh_beam_workspace_bytes(self._ref))
            _ok(n, "vh_beam_workspace_bytes")
            self._bytes = n
        return self._bytes

    def select(self, logits, scores, tokens, parents, new_scores, *, ended=None, new_ended=None, workspace):
        """The best `picks` of each sequence: tokens and parents (int32), new_scores (fp32) and new_ended (int32), all
        [sequences][picks]; scores (fp32) and ended (int32) are the beams' [sequences][beams]."""
        f, device, torch = self._whole, self._device, _torch()
        beams, picks = self._beams, self._picks
        args = (self._tensor("logits", "logits", logits), f("scores", scores, torch.float32, beams, device),
                f("ended", ended, torch.int32, beams, device) if ended is not None else None,
                f("tokens", tokens, torch.int32, picks, device), f("parents", parents, torch.int32, picks, device),
                f("new_scores", new_scores, torch.float32, picks, device),
                f("new_ended", new_ended, torch.int32, picks, device) if new_ended is not None else None,
                self._buffer("workspace", workspace, self.workspace_bytes(), device))
        self._on_gpu(device)
        _ok(lib().vh_beam_select(self.ctx.h, self._ref, *args), "vh_beam_select")


class Model:
    """A VSCNAT01 pack uploaded to the device."""

    def __init__(self, ctx: Context, dims: ModelDims, pack) -> None:
        self.ctx = ctx
        self.dims = dims
        self._cd = to_c(dims)
        self.h = lib().vh_model_load(ctx.h, ctypes.byref(self._cd), ptr(pack), pack.nbytes)
        if not self.h:
            raise NativeError(f"vh_model_load failed: {last_error()}")
        ctx.models.add(self)

    def close(self):
        if self.h:
            lib().vh_model_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001
            pass

    def set_precision(self, precision: int):
        _ok(lib().vh_model_set_precision(self.h, precision), "vh_model_set_precision")

    def transformer(self, layer: int, axis: int, x, sequences: int, length: int):
        _ok(lib().vh_transformer(self.ctx.h, self.h, layer, axis, ptr(x), sequences, length), "vh_transformer")

    def stft(self, audio, length: int, source, layout: int = SPEC_REFERENCE):
        _ok(lib().vh_stft(self.ctx.h, self.h, ptr(audio), length, ptr(source), layout), "vh_stft")

    def istft(self, source, mask, length: int, audio, layout: int = SPEC_REFERENCE):
        _ok(lib().vh_istft(self.ctx.h, self.h, ptr(source), ptr(mask), length, ptr(audio), layout), "vh_istft")

    def band_split(self, source, frames: int, out, layout: int = SPEC_REFERENCE):
        _ok(lib().vh_band_split(self.ctx.h, self.h, ptr(source), frames, ptr(out), layout), "vh_band_split")

    def mask_estimate(self, features, frames: int, mask, layout: int = SPEC_REFERENCE):
        _ok(lib().vh_mask_estimate(self.ctx.h, self.h, ptr(features), frames, ptr(mask), layout), "vh_mask_estimate")

    def forward(self, audio, length: int, vocals, instrumental=None):
        _ok(lib().vh_forward(self.ctx.h, self.h, ptr(audio), length, ptr(vocals),
                             _opt(instrumental)), "vh_forward")

    def separate(self, audio, length: int, chunk: int, step: int, batch: int, vocals, instrumental=None):
        _ok(lib().vh_separate(self.ctx.h, self.h, ptr(audio), length, chunk, step, batch, ptr(vocals),
                              _opt(instrumental)), "vh_separate")
