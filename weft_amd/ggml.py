"""GGML operator boundary of libweft_hip from Python: MUL_MAT / MUL_MAT_ID and,
between them in a decoder layer, the residual norm, the norm and rotation of
heads, the paged key / value cache and the attention over it; the product of
8-bit floats; log probabilities.

``Tensor`` is the part of ``struct ggml_tensor`` (ggml/include/ggml.h:667-692)
that MUL_MAT reads: type id, ``ne``, byte strides ``nb`` and a device data
pointer.  ``mul_mat`` runs GGML_OP_MUL_MAT with the semantics of
ggml_compute_forward_mul_mat (ggml-cpu/ggml-cpu.c:1245-1443) on the quantized
kernels; where GGML asserts, it raises ``HipError`` (the library launches
nothing).
"""
from __future__ import annotations

import ctypes
from collections.abc import Sequence

from . import _lib

# enum ggml_type (ggml/include/ggml.h:389-431), the types of this path
F32, Q4_0, Q8_0, Q4_K, Q5_K, Q6_K, Q8_K, IQ2_XXS, I32, MXFP4, NVFP4 = 0, 2, 8, 12, 13, 14, 15, 16, 26, 39, 40
Q4_1, Q8_1, IQ2_XS = 3, 9, 17
F16 = 1  # activations and cache rows; no MUL_MAT type
F8_E4M3 = 4096  # 8-bit floats with scales beside them: mul_mat_f8; no GGML type


# bytes of the types that are no records and that MUL_MAT does not know
_PLAIN = {I32: 4, F16: 2, F8_E4M3: 1}


class Tensor(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int32), ("ne", ctypes.c_int64 * 4),
                ("nb", ctypes.c_size_t * 4), ("data", ctypes.c_void_p)]


def type_size(t: int) -> int:
    return _lib.load().weft_ggml_type_size(t)


def blck_size(t: int) -> int:
    return _lib.load().weft_ggml_blck_size(t)


def row_size(t: int, ne: int) -> int:
    return _lib.load().weft_ggml_row_size(t, ne)


def vec_dot_type(t: int) -> int:
    return _lib.load().weft_ggml_vec_dot_type(t)


def tensor(t: int, ne: Sequence[int], data: int = 0, nb: Sequence[int] | None = None) -> Tensor:
    """A descriptor with GGML's default strides (ggml_new_tensor_impl:
    nb0 = type size, nb1 = nb0 * ne0 / block size, nb_i = nb_{i-1} * ne_{i-1})
    unless ``nb`` is given."""
    ne = list(ne) + [1] * (4 - len(ne))
    if nb is None:
        size = _PLAIN.get(t) or type_size(t)
        nb = [size, size * ne[0] if t in _PLAIN else row_size(t, ne[0])]
        nb += [nb[1] * ne[1], nb[1] * ne[1] * ne[2]]
    return Tensor(t, (ctypes.c_int64 * 4)(*ne), (ctypes.c_size_t * 4)(*nb), data)


def mul_mat_work_size(src0: Tensor, src1: Tensor) -> int:
    return _lib.load().weft_ggml_mul_mat_work_size(ctypes.byref(src0), ctypes.byref(src1))


def mul_mat(src0: Tensor, src1: Tensor, dst: Tensor, wdata: int = 0, wsize: int = 0) -> None:
    """Enqueue dst = MUL_MAT(src0, src1) on the current stream."""
    lib = _lib.load()
    code = lib.weft_ggml_mul_mat(ctypes.byref(src0), ctypes.byref(src1), ctypes.byref(dst),
                                 ctypes.c_void_p(wdata), wsize)
    if code != 0:
        lib.weft_hip_get_last_error()  # the same error, recorded: clear it
        raise _lib.HipError(code, "weft_ggml_mul_mat")


def mul_mat_id_work_size(src0: Tensor, src1: Tensor, ids: Tensor) -> int:
    return _lib.load().weft_ggml_mul_mat_id_work_size(ctypes.byref(src0), ctypes.byref(src1),
                                                      ctypes.byref(ids))


def mul_mat_id(src0: Tensor, src1: Tensor, ids: Tensor, dst: Tensor, wdata: int = 0,
               wsize: int = 0) -> None:
    """Enqueue dst = MUL_MAT_ID(src0 experts, src1, ids) on the current stream."""
    lib = _lib.load()
    code = lib.weft_ggml_mul_mat_id(ctypes.byref(src0), ctypes.byref(src1), ctypes.byref(ids),
                                    ctypes.byref(dst), ctypes.c_void_p(wdata), wsize)
    if code != 0:
        lib.weft_hip_get_last_error()
        raise _lib.HipError(code, "weft_ggml_mul_mat_id")


# the library's per-device work buffer of mul_mat_id_noalloc (weft_hip.h)
NOALLOC_SCRATCH_BYTES = 32 << 20


def mul_mat_id_noalloc(src0: Tensor, src1: Tensor, ids: Tensor, dst: Tensor) -> None:
    """MUL_MAT_ID without a caller work buffer: the library's per-device
    scratch stands in for it (calls that overlap on one device race)."""
    lib = _lib.load()
    code = lib.weft_ggml_mul_mat_id_noalloc(ctypes.byref(src0), ctypes.byref(src1), ctypes.byref(ids),
                                            ctypes.byref(dst))
    if code != 0:
        lib.weft_hip_get_last_error()
        raise _lib.HipError(code, "weft_ggml_mul_mat_id_noalloc")


class KvBatch(ctypes.Structure):
    """A batch of sequences over a paged cache (weft_ggml_kv_batch): I32 tensors
    ``pages`` (pages a sequence, sequences), ``starts`` (sequences + 1, where
    each sequence's new tokens begin among the call's rows) and ``lengths``
    (sequences, with the new tokens).  All three are read on the device."""
    _fields_ = [("pages", Tensor), ("starts", Tensor), ("lengths", Tensor)]


def kv_batch(pages: Tensor, starts: Tensor, lengths: Tensor) -> KvBatch:
    return KvBatch(pages, starts, lengths)


def _done(lib: ctypes.CDLL, code: int, where: str) -> None:
    if code != 0:
        lib.weft_hip_get_last_error()  # the same error, recorded: clear it
        raise _lib.HipError(code, where)


def _ref(t: ctypes.Structure | None):
    return None if t is None else ctypes.byref(t)


def add_rms_norm(x: Tensor, residual: Tensor | None, weight: Tensor | None, total: Tensor | None, dst: Tensor,
                 eps: float) -> None:
    """Enqueue dst = norm(x + residual) * weight, the mean square over a row;
    ``total`` (which may be x's own memory) keeps the sum.  dst is F32, F16, or the Q8_0 /
    Q8_1 / Q8_K records that mul_mat takes as a quantized src1."""
    lib = _lib.load()
    _done(lib, lib.weft_ggml_add_rms_norm(_ref(x), _ref(residual), _ref(weight), _ref(total), _ref(dst), eps),
          "weft_ggml_add_rms_norm")


def kv_write(k: Tensor, v: Tensor, batch: KvBatch, k_cache: Tensor, v_cache: Tensor) -> None:
    """Enqueue the quantization of new rows k, v (D, kv heads, tokens) into
    their sequences' pages; caches are (D, page size, kv heads, pages) of F16,
    Q8_0 or Q4_0."""
    lib = _lib.load()
    _done(lib, lib.weft_ggml_kv_write(_ref(k), _ref(v), _ref(batch), _ref(k_cache), _ref(v_cache)),
          "weft_ggml_kv_write")


def kv_read(k_cache: Tensor, v_cache: Tensor, batch: KvBatch, k: Tensor, v: Tensor) -> None:
    """Enqueue the read of every sequence's first n positions into k, v
    (D, kv heads, n, sequences), zeros past its length."""
    lib = _lib.load()
    _done(lib, lib.weft_ggml_kv_read(_ref(k_cache), _ref(v_cache), _ref(batch), _ref(k), _ref(v)),
          "weft_ggml_kv_read")


def attention_work_size(q: Tensor, k_cache: Tensor, v_cache: Tensor, batch: KvBatch) -> int:
    return _lib.load().weft_ggml_attention_work_size(_ref(q), _ref(k_cache), _ref(v_cache), _ref(batch))


def attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, batch: KvBatch, dst: Tensor, scale: float,
              window: int = 0, sinks: int = 0, wdata: int = 0, wsize: int = 0) -> None:
    """Enqueue dst = causal attention of the new tokens' queries (D, heads,
    tokens) over their sequences' cache; with a window, a query sees the last
    ``window`` positions and the first ``sinks``."""
    lib = _lib.load()
    _done(lib, lib.weft_ggml_attention(_ref(q), _ref(k_cache), _ref(v_cache), _ref(batch), _ref(dst), scale, window,
                                       sinks, wdata, wsize),
          "weft_ggml_attention")


def quantize_f8(x: Tensor, codes: Tensor, scales: Tensor) -> None:
    """Enqueue the quantization of rows x (K, rows; F32 or F16) to 8-bit floats:
    ``scales`` of (ceil(K / 128), rows) is one for each 128 values of a row, of
    (ceil(K / 128), ceil(rows / 128)) one for each block of 128 x 128 (weights)."""
    lib = _lib.load()
    _done(lib, lib.weft_ggml_quantize_f8(x, codes, scales), "weft_ggml_quantize_f8")


def mul_mat_f8_work_size(w: Tensor, x: Tensor) -> int:
    return _lib.load().weft_ggml_mul_mat_f8_work_size(w, x)


def mul_mat_f8(w: Tensor, w_scales: Tensor, x: Tensor, x_scales: Tensor | None, dst: Tensor, wdata: int = 0,
               wsize: int = 0) -> None:
    """Enqueue dst (N, M) = the product of weights w (K, N; 8-bit floats, scales by
    blocks) with rows x (K, M): F32 or F16, quantized on the way, or 8-bit floats
    with their x_scales."""
    lib = _lib.load()
    _done(lib, lib.weft_ggml_mul_mat_f8(w, w_scales, x, x_scales, dst, wdata, wsize),
          "weft_ggml_mul_mat_f8")


class HeadRope(ctypes.Structure):
    """How heads are turned (weft_ggml_head_rope)."""
    _fields_ = [("n_rot", ctypes.c_int32), ("neighbours", ctypes.c_int32), ("base", ctypes.c_double),
                ("scale", ctypes.c_double), ("magnitude", ctypes.c_double)]


def head_rope(n_rot: int, neighbours: bool = False, base: float = 10000.0, scale: float = 1.0,
              magnitude: float = 1.0) -> HeadRope:
    """The rotation of a head's first n_rot values: pairs (i, i + n_rot / 2), or
    neighbours (2i, 2i + 1), by position * scale * base^(-2i / n_rot)."""
    return HeadRope(n_rot, neighbours, base, scale, magnitude)


def head_norm_rope(q: Tensor, k: Tensor | None, q_dst: Tensor, k_dst: Tensor | None, positions: Tensor | None,
                   rope: HeadRope, eps: float | None = None, q_weight: Tensor | None = None,
                   k_weight: Tensor | None = None, factors: Tensor | None = None) -> None:
    """Enqueue the norm (unless eps is None) of every head of q and k (D, heads,
    tokens) and its rotation by the tokens' positions (I32); a destination may be its
    source.  factors (n_rot / 2) divide the pairs' frequencies."""
    lib = _lib.load()
    _done(lib, lib.weft_ggml_head_norm_rope(q, k, q_dst, k_dst, positions, rope, eps is not None, eps or 0.0, q_weight,
                                            k_weight, factors),
          "weft_ggml_head_norm_rope")


MOST_ALTERNATIVES = 64


def log_probs_work_size(logits: Tensor, n_top: int) -> int:
    return _lib.load().weft_ggml_log_probs_work_size(logits, n_top)


def log_probs(logits: Tensor, tokens: Tensor | None, token_lp: Tensor | None, entropy: Tensor | None,
              top_ids: Tensor | None, top_lp: Tensor | None, scale: float = 1.0, wdata: int = 0, wsize: int = 0) -> None:
    """Enqueue, for rows of logits (V, rows) times scale: the log probabilities of
    tokens (n, rows), the rows' entropy and their largest logits' ids and log
    probabilities (A, rows), largest first, of equal ones the lowest id."""
    lib = _lib.load()
    _done(lib, lib.weft_ggml_log_probs(logits, tokens, token_lp, entropy, top_ids, top_lp, scale, wdata, wsize),
          "weft_ggml_log_probs")
