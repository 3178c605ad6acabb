"""Thin object layer over the C ABI: a device context and a resident flat index.

Host arrays are numpy; device arrays are anything exposing ``data_ptr()`` (torch
tensors).  PyTorch is plumbing here (device memory and streams for callers that
already hold their data on the GPU); all compute is inside libneedle_hip.so.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

from . import _lib
from .distance import DistanceFunction

PRECISION = {"fp32": _lib.PRECISION_FP32, "bf16": _lib.PRECISION_BF16, "exact": _lib.PRECISION_EXACT_SCAN}


def _f32(a) -> np.ndarray:
    return np.ascontiguousarray(a, dtype=np.float32)


def pack_bitmask(bits) -> np.ndarray:
    """bool[n] -> uint32[ceil(n/32)]; bit i lives in word i>>5 at position i&31."""
    b = np.asarray(bits, dtype=np.bool_).reshape(-1)
    pad = (-b.size) % 32
    if pad:
        b = np.concatenate([b, np.zeros(pad, dtype=np.bool_)])
    return np.packbits(b.reshape(-1, 32), axis=1, bitorder="little").view(np.uint32).reshape(-1).copy()


def _mask_words(mask, n):
    if mask is None:
        return None
    m = np.asarray(mask)
    if m.dtype == np.bool_:
        if m.size != n:
            raise ValueError(f"mask has {m.size} entries for {n} rows")
        m = pack_bitmask(m)
    m = np.ascontiguousarray(m, dtype=np.uint32)
    if m.size < (n + 31) // 32:
        raise ValueError("bitmask too short")
    return m


def _wait_for_producer(t) -> None:
    """The library works on its own stream: whatever the caller's stream still has in flight for a device tensor must
    have finished before the library reads it."""
    if getattr(t, "is_cuda", False):
        import torch

        torch.cuda.current_stream(t.device).synchronize()


_VALUES = {"torch.float32": _lib.VALUE_F32, "torch.float16": _lib.VALUE_F16, "torch.bfloat16": _lib.VALUE_BF16}
_NAMES: dict = {}  # torch dtypes by the object: a name costs more than the rest of a check


def _dtype(t) -> str:
    name = _NAMES.get(t.dtype)
    if name is None:
        name = _NAMES[t.dtype] = str(t.dtype)
    return name


def _value(t, what: str) -> int:
    v = _VALUES.get(_dtype(t))
    if v is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, not {t.dtype}")
    return v


_U32 = 2 ** 32 - 1


def _check_u32(**sizes) -> None:
    """Sizes that the library takes in 32 bits: ctypes would cut a longer number to its lowest 32."""
    for name, value in sizes.items():
        if value > _U32:
            raise _lib.NeedleHipError(_lib.ERR_UNSUPPORTED, f"{name} = {value} does not fit 32 bits")


def _check_end_token(end_token: int, vocab: int, rows: int, k: int) -> None:
    if rows and k and not 0 <= end_token < vocab:  # (its lowest 32 bits could be)
        raise _lib.NeedleHipError(_lib.ERR_INVALID_ARGUMENT, f"end_token {end_token} is not below vocab {vocab}")


_torch_module = None


def _torch():
    """torch, for callers that hold its tensors; imported once, and only then."""
    global _torch_module
    if _torch_module is None:
        import torch

        _torch_module = torch
    return _torch_module


_stream_of = None  # (current device, current stream of a device, wait for a stream) where torch has the raw handles


def _wait_for_stream(device: int) -> None:
    """torch's current stream on `device` has finished: what its synchronize() does, in a third of the time where torch tells
    the handle.  Stream 0 names no device, so this holds on the current device only."""
    global _stream_of
    if _stream_of is None:
        inner = _torch()._C
        names = [getattr(inner, name, None) for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream")]
        wait = C.CFUNCTYPE(C.c_int, C.c_void_p)(("hipStreamSynchronize", _lib.lib()))
        _stream_of = (*names, wait) if all(names) else ()
    if not _stream_of or _stream_of[0]() != device or _stream_of[2](_stream_of[1](device)):
        _torch().cuda.current_stream(device).synchronize()  # (raises what the runtime reports)


def _rows_of(t, name: str, dtype=None, cols=None, rows=None):
    """(rows, columns, elements from row to row) of a matrix whose rows are contiguous, any distance apart."""
    shape = t.shape
    if len(shape) != 2 or (dtype is not None and _dtype(t) not in dtype) or (cols is not None and shape[1] != cols) or \
            (rows is not None and shape[0] != rows):
        raise ValueError(f"{name} must be [{'n' if rows is None else rows}, {'dim' if cols is None else cols}]"
                         f"{'' if dtype is None else ' of ' + ' or '.join(dtype)}, not {list(shape)} of {t.dtype}")
    n, dim = shape
    apart, next_to = t.stride()
    if n <= 1:
        apart = dim
    if (dim > 1 and next_to != 1) or apart < dim:
        raise ValueError(f"{name} must have contiguous rows that do not overlap")
    return n, dim, apart


_F32, _I8, _WORDS, _FLAGS = ("torch.float32",), ("torch.int8",), ("torch.int32", "torch.uint32"), ("torch.bool", "torch.uint8")


def _flat(t, name: str, dtype, size: int) -> None:
    if _dtype(t) not in dtype or t.numel() != size or not t.is_contiguous():
        raise ValueError(f"{name} must be {size} contiguous values of {' or '.join(dtype)}, not {list(t.shape)} of {t.dtype}")


def _codes_i8(codes, scales, what: str):
    """Host int8 codes [rows, dim] and their f32 scales, contiguous.  Values are not converted: a wider type would wrap."""
    _check_u32(**{f"{name} of {what}": d for name, d in zip(("rows", "dim"), np.shape(codes))})
    c, s = np.ascontiguousarray(codes), _f32(scales).reshape(-1)
    if c.dtype != np.int8 or c.ndim != 2 or s.size != c.shape[0]:
        raise ValueError(f"{what} must be int8 [rows, dim] with one scale per row")
    return c, s


def _state_layout(src, dst, axis: int):
    """(outer, inner, bytes, strides of src, strides of dst) in bytes of two tensors whose dimension `axis` numbers the
    rows: dimensions before it must fold into one, those behind it into runs of neighbouring elements that lie one stride
    apart."""
    shape, a, b, size = tuple(src.shape), src.stride(), dst.stride(), src.element_size()
    run, i = 1, len(shape) - 1
    while i > axis and (shape[i] == 1 or a[i] == b[i] == run):  # dimensions that continue the run in both tensors
        run *= shape[i]
        i -= 1
    parts = []
    for first, last in ((i, axis), (axis - 1, -1)):  # behind the rows, then before them
        n, sa, sb = 1, 0, 0
        for d in range(first, last, -1):
            if shape[d] == 1:
                continue
            if n == 1:
                n, sa, sb = shape[d], a[d], b[d]
            elif a[d] == n * sa and b[d] == n * sb:
                n *= shape[d]
            else:
                raise ValueError("a state's dimensions must fold into one before its rows and, behind them, into runs one stride apart")
        parts.append((n, sa * size, sb * size))
    (inner, ia, ib), (outer, oa, ob) = parts
    return outer, inner, run * size, (oa, a[axis] * size, ia), (ob, b[axis] * size, ib)


def _destroy_handle(owner, destroy_name: str = "needle_hip_index_destroy") -> None:
    """Destroys owner._h unless the context it is bound to has been closed: closing a context frees everything bound to
    it, and a wrapper that outlives its context (garbage collected later) must not hand the dead handle to the library
    again."""
    h, ctx = getattr(owner, "_h", None), getattr(owner, "ctx", None)
    ctx_alive = ctx is not None and getattr(ctx, "_h", None) is not None and bool(ctx._h.value)
    if h is not None and h.value and ctx_alive and not _lib.shutting_down():
        getattr(_lib.lib(), destroy_name)(h)
    owner._h = C.c_void_p()


class Context:
    """One HIP device (needle_hip_ctx)."""

    _close_order = 1  # at interpreter exit contexts close after the indexes bound to them

    def __init__(self, device: int = 0):
        self._h = C.c_void_p()
        _lib.check(_lib.lib().needle_hip_init(device, C.byref(self._h)))
        self.device = device
        _lib.register_live(self)

    def close(self) -> None:
        if getattr(self, "_h", None) and self._h.value and not _lib.shutting_down():
            _lib.lib().needle_hip_shutdown(self._h)
        self._h = C.c_void_p()

    def __del__(self):  # pragma: no cover - best effort
        try:
            self.close()
        except Exception:
            pass

    def set_profiling(self, on: bool) -> None:
        _lib.check(_lib.lib().needle_hip_set_profiling(self._h, int(on)))

    def metrics(self) -> dict:
        m = _lib.Metrics()
        _lib.check(_lib.lib().needle_hip_get_metrics(self._h, C.byref(m)))
        return {name: getattr(m, name) for name, _ in _lib.Metrics._fields_}

    def reset_metrics(self) -> None:
        _lib.check(_lib.lib().needle_hip_reset_metrics(self._h))

    def set_tuning(self, **overrides) -> None:
        """Planning overrides (needle_hip_set_tuning): tests force a code path with them, the A/B tools sweep them.
        `stages=(10, 25)` sets the staged-launch schedule; `reset=1` restores the built-in choices."""
        for key, value in overrides.items():
            if key == "stages":
                vals = list(value) + [0] * (4 - len(value))
                for i, pc in enumerate(vals[:4]):
                    _lib.check(_lib.lib().needle_hip_set_tuning(self._h, f"stage{i}".encode(), float(pc)))
            else:
                _lib.check(_lib.lib().needle_hip_set_tuning(self._h, key.encode(), float(value)))

    def apply_tuning_spec(self, spec: str | None) -> None:
        """`key=value,key=value` as the bench tools take it (stages as `stages=10:25`)."""
        for item in filter(None, (spec or "").split(",")):
            key, _, val = item.partition("=")
            if key == "stages":
                self.set_tuning(stages=[float(x) for x in val.split(":") if x])
            else:
                self.set_tuning(**{key: float(val)})

    # ---- operator-level calls ------------------------------------------
    def batch_distance(self, metric: DistanceFunction, query, base, arith: int = _lib.ARITH_ACCEL_CHUNK4) -> np.ndarray:
        q, b = _f32(query), _f32(base)
        if b.size == 0:
            return np.empty(0, dtype=np.float32)
        if b.ndim != 2 or b.shape[1] != q.size:
            raise _lib.DimensionMismatch(_lib.ERR_DIMENSION_MISMATCH, "Dimension mismatch")
        out = np.empty(b.shape[0], dtype=np.float32)
        _lib.check(_lib.lib().needle_hip_batch_distance(self._h, int(metric), arith, q.ctypes.data, b.ctypes.data,
                                                        b.shape[0], q.size, out.ctypes.data))
        return out

    def kmeans_assign(self, vectors, centroids, arith: int = _lib.ARITH_ACCEL_CHUNK4) -> np.ndarray:
        v, c = _f32(vectors), _f32(centroids)
        out = np.zeros(v.shape[0], dtype=np.uint32)
        if v.shape[0]:
            _lib.check(_lib.lib().needle_hip_kmeans_assign(self._h, arith, v.ctypes.data, v.shape[0], c.ctypes.data,
                                                           c.shape[0], v.shape[1], out.ctypes.data))
        return out

    def normalize(self, vectors, arith: int = _lib.ARITH_DISTANCE_RS) -> np.ndarray:
        """Rows of `vectors` normalised on the device (a copy is returned): distance.rs's `normalize` recipe, or
        the accelerator's `batch_normalize` with arith ACCEL_CHUNK4."""
        v = np.array(vectors, dtype=np.float32, order="C", copy=True)
        flat = v.reshape(1, -1) if v.ndim == 1 else v
        if flat.size:
            _lib.check(_lib.lib().needle_hip_normalize(self._h, arith, flat.ctypes.data, flat.shape[0], flat.shape[1]))
        return v

    def normalize_device(self, d_vectors, arith: int = _lib.ARITH_DISTANCE_RS) -> None:
        """In place, on a contiguous float32 [n, dim] device tensor."""
        _wait_for_producer(d_vectors)
        _lib.check(_lib.lib().needle_hip_normalize_device(self._h, arith, d_vectors.data_ptr(), int(d_vectors.shape[0]),
                                                          int(d_vectors.shape[1])))

    def batch_top_k(self, scores, k: int):
        """(idx[rows,k] uint64, scores[rows,k] f32, counts[rows] uint32): the k smallest of every row by (score, index)."""
        s = _f32(scores)
        if s.ndim == 1:
            s = s.reshape(1, -1)
        rows, n = s.shape
        kk = max(k, 1)
        idx = np.full((rows, kk), np.iinfo(np.uint64).max, dtype=np.uint64)
        val = np.full((rows, kk), np.inf, dtype=np.float32)
        cnt = np.zeros(rows, dtype=np.uint32)
        _lib.check(_lib.lib().needle_hip_batch_top_k(self._h, s.ctypes.data if s.size else None, rows, n, k, idx.ctypes.data,
                                                     val.ctypes.data, cnt.ctypes.data))
        return idx[:, :k], val[:, :k], cnt

    def merge_topk(self, dists, ids, counts, k: int):
        """Host form of the shard merge: dists/ids [lists, q, per], counts [lists, q] -> (ids[q,k], dists[q,k], counts[q])."""
        d, i = _f32(dists), np.ascontiguousarray(ids, dtype=np.uint64)
        c = np.ascontiguousarray(counts, dtype=np.uint32)
        lists, q, per = d.shape
        kk = max(k, 1)
        oi = np.full((q, kk), np.iinfo(np.uint64).max, dtype=np.uint64)
        od = np.full((q, kk), np.inf, dtype=np.float32)
        oc = np.zeros(q, dtype=np.uint32)
        _lib.check(_lib.lib().needle_hip_merge_topk(self._h, d.ctypes.data, i.ctypes.data, c.ctypes.data, lists, q, per, k,
                                                    oi.ctypes.data, od.ctypes.data, oc.ctypes.data))
        return oi[:, :k], od[:, :k], oc

    def distance_matrix(self, metric: DistanceFunction, queries, base, arith: int = _lib.ARITH_SERVICE) -> np.ndarray:
        """[queries][vectors] distances (the dot product negated), every value in the chosen arithmetic:
        distance_matrix_cosine / _euclidean of src/services/compute/gpu_kernels.rs:223-265 with ARITH_SERVICE."""
        q, b = _f32(queries), _f32(base)
        if q.ndim != 2 or b.ndim != 2 or (q.shape[0] and b.shape[0] and q.shape[1] != b.shape[1]):
            raise _lib.DimensionMismatch(_lib.ERR_DIMENSION_MISMATCH, "Dimension mismatch")
        out = np.empty((q.shape[0], b.shape[0]), dtype=np.float32)
        if out.size:
            _lib.check(_lib.lib().needle_hip_distance_matrix(self._h, int(metric), arith, q.ctypes.data, q.shape[0],
                                                             b.ctypes.data, b.shape[0], q.shape[1], out.ctypes.data))
        return out

    def distance_matrix_device(self, metric: DistanceFunction, d_queries, d_base, d_out, arith: int = _lib.ARITH_SERVICE) -> None:
        for t in (d_queries, d_base):
            _wait_for_producer(t)
        _lib.check(_lib.lib().needle_hip_distance_matrix_device(self._h, int(metric), arith, d_queries.data_ptr(),
                                                                int(d_queries.shape[0]), d_base.data_ptr(),
                                                                int(d_base.shape[0]), int(d_queries.shape[1]), d_out.data_ptr()))

    def multi_query_search(self, metric: DistanceFunction, queries, base, k: int, arith: int = _lib.ARITH_SERVICE):
        """(idx[q,k] uint64, dists[q,k] f32, counts[q] uint32): per query the k nearest vectors by (distance, index),
        formed on the device from the distance matrix (multi_query_search, gpu_kernels.rs:267-300)."""
        q, b = _f32(queries), _f32(base)
        if q.ndim != 2 or b.ndim != 2 or (q.shape[0] and b.shape[0] and q.shape[1] != b.shape[1]):
            raise _lib.DimensionMismatch(_lib.ERR_DIMENSION_MISMATCH, "Dimension mismatch")
        nq, kk = q.shape[0], max(k, 1)
        idx = np.full((nq, kk), np.iinfo(np.uint64).max, dtype=np.uint64)
        val = np.full((nq, kk), np.inf, dtype=np.float32)
        cnt = np.zeros(nq, dtype=np.uint32)
        if nq:
            _lib.check(_lib.lib().needle_hip_multi_query_search(self._h, int(metric), arith, q.ctypes.data, nq,
                                                                b.ctypes.data if b.size else None, b.shape[0], q.shape[1], k,
                                                                idx.ctypes.data, val.ctypes.data, cnt.ctypes.data))
        return idx[:, :k], val[:, :k], cnt

    def merge_topk_device(self, d_dists, d_ids, d_counts, lists: int, q: int, per: int, k: int, d_out_ids, d_out_dists,
                          d_out_counts) -> None:
        _lib.check(_lib.lib().needle_hip_merge_topk_device(self._h, d_dists.data_ptr(), d_ids.data_ptr(),
                                                           d_counts.data_ptr(), lists, q, per, k, d_out_ids.data_ptr(),
                                                           d_out_dists.data_ptr(), d_out_counts.data_ptr()))

    # ---- rows in 8-bit integers, their products, the best continuations ---------------------------------------------
    def _check_device(self, *tensors) -> None:
        """Every given tensor lies on the context's device; the caller's stream there has finished."""
        for t in tensors:
            if t is not None and t.get_device() != self.device:  # -1 on the host
                raise ValueError(f"a tensor lies on {t.device}, the context on device {self.device}")
        _wait_for_stream(self.device)

    def quantize_rows(self, rows):
        """(codes int8 [n, dim], scales f32 [n]) of float32 or float16 host rows: symmetric, scale = max |x| * (1 / 127) per row in f32,
        codes the whole numbers nearest to x / scale (needle_hip_quantize_rows_i8).  NaN / Inf raise InvalidVector."""
        r = np.asarray(rows)
        if r.ndim == 2:
            _check_u32(dim=r.shape[1])
        r = np.ascontiguousarray(r, dtype=np.float16 if r.dtype == np.float16 else np.float32)
        if r.ndim != 2:
            raise ValueError("rows must be [n, dim]")
        codes, scales = np.zeros(r.shape, dtype=np.int8), np.zeros(r.shape[0], dtype=np.float32)
        _lib.check(_lib.lib().needle_hip_quantize_rows_i8(self._h, r.ctypes.data, _lib.VALUE_F16 if r.dtype == np.float16 else _lib.VALUE_F32,
                                                          r.shape[0], r.shape[1], codes.ctypes.data, scales.ctypes.data))
        return codes, scales

    def quantize_rows_device(self, d_rows, d_codes, d_scales) -> None:
        """The same for a float32 / float16 / bfloat16 device matrix, into int8 [n, dim] codes and float32 [n] scales; rows may
        lie apart.  A row with a NaN or an infinity gets scale NaN and codes 0."""
        n, dim, apart = _rows_of(d_rows, "d_rows")
        if dim > _U32:
            _check_u32(dim=dim)
        value = _value(d_rows, "d_rows")
        _, _, codes_apart = _rows_of(d_codes, "d_codes", _I8, dim, n)
        _flat(d_scales, "d_scales", _F32, n)
        self._check_device(d_rows, d_codes, d_scales)
        _lib.check(_lib.lib().needle_hip_quantize_rows_i8_device(self._h, d_rows.data_ptr(), value, n, dim, apart, d_codes.data_ptr(),
                                                                 codes_apart, d_scales.data_ptr()))

    def matmul_i8(self, a, a_scales, b, b_scales, bias=None) -> np.ndarray:
        """f32 [m, n] of (a[i] . b[j]) * a_scales[i] * b_scales[j] (+ bias[j]) for int8 host codes [m, k] and [n, k]
        (needle_hip_matmul_i8)."""
        a, sa = _codes_i8(a, a_scales, "a")
        b, sb = _codes_i8(b, b_scales, "b")
        if a.shape[1] != b.shape[1]:
            raise _lib.DimensionMismatch(_lib.ERR_DIMENSION_MISMATCH, f"Dimension mismatch: {a.shape[1]} and {b.shape[1]}")
        t = None if bias is None else _f32(bias).reshape(-1)
        if t is not None and t.size != b.shape[0]:
            raise ValueError("bias must have one value per row of b")
        out = np.empty((a.shape[0], b.shape[0]), dtype=np.float32)
        _lib.check(_lib.lib().needle_hip_matmul_i8(self._h, a.ctypes.data, sa.ctypes.data, a.shape[0], b.ctypes.data, sb.ctypes.data,
                                                   b.shape[0], a.shape[1], None if t is None else t.ctypes.data, out.ctypes.data))
        return out

    def matmul_i8_device(self, d_a, d_a_scales, d_b, d_b_scales, d_out, d_bias=None) -> None:
        """The same on the device, into a float32 / float16 / bfloat16 [m, n] matrix.  Rows of every matrix may lie apart: the
        first k codes of longer rows (a Matryoshka prefix) are a view like any other."""
        self._product(d_a, d_a_scales, d_b, d_b_scales, d_out, d_bias)

    def linear_i8_device(self, d_x, d_b, d_b_scales, d_out, d_bias=None) -> None:
        """matmul_i8_device for rows that are still in floating point: they are quantized as quantize_rows_device does and
        multiplied in one call."""
        self._product(d_x, None, d_b, d_b_scales, d_out, d_bias)

    def _product(self, d_a, d_a_scales, d_b, d_b_scales, d_out, d_bias) -> None:
        m, k, a_apart = _rows_of(d_a, "the rows", None if d_a_scales is None else _I8)
        if (m | k) >> 32:
            _check_u32(m=m, k=k)
        n, b_k, b_apart = _rows_of(d_b, "d_b", _I8)
        if b_k != k:
            raise _lib.DimensionMismatch(_lib.ERR_DIMENSION_MISMATCH, f"Dimension mismatch: {k} and {b_k}")
        _, _, out_apart = _rows_of(d_out, "d_out", None, n, m)
        out_value = _value(d_out, "d_out")
        _flat(d_b_scales, "d_b_scales", _F32, n)
        if d_bias is not None:
            _flat(d_bias, "d_bias", _F32, n)
        if d_a_scales is None:
            x_value = _value(d_a, "d_x")
        else:
            _flat(d_a_scales, "d_a_scales", _F32, m)
        self._check_device(d_a, d_a_scales, d_b, d_b_scales, d_out, d_bias)
        right = (m, d_b.data_ptr(), b_apart, d_b_scales.data_ptr(), n, k, None if d_bias is None else d_bias.data_ptr(), out_value,
                 d_out.data_ptr(), out_apart)
        if d_a_scales is None:
            _lib.check(_lib.lib().needle_hip_linear_i8_device(self._h, d_a.data_ptr(), x_value, a_apart, *right))
        else:
            _lib.check(_lib.lib().needle_hip_matmul_i8_device(self._h, d_a.data_ptr(), a_apart, d_a_scales.data_ptr(), *right))

    def beam_select(self, logits, scores, k: int, *, beams: int, normalize: bool = True, mask=None, finished=None, end_token: int = 0):
        """(parents, tokens uint32, scores f32, all [groups, k], counts uint32 [groups]): the k best continuations of every group
        of `beams` rows of host logits [groups * beams, vocab], by total (normalize: scores + log-softmax; else scores +
        logits), then beam, then token (needle_hip_beam_select).  mask: bool [vocab] or [rows, vocab], True = admitted."""
        x = np.asarray(logits)
        _check_u32(beams=beams, k=k, **dict(zip(("rows", "vocab"), x.shape)))
        x = np.ascontiguousarray(x, dtype=np.float16 if x.dtype == np.float16 else np.float32)
        if x.ndim != 2 or beams < 1 or x.shape[0] % beams:
            raise ValueError("logits must be [groups * beams, vocab]")
        rows, vocab = x.shape
        s = None if scores is None else _f32(scores).reshape(-1)
        f = None if finished is None else np.ascontiguousarray(np.asarray(finished).reshape(-1) != 0, dtype=np.uint8)
        if (s is not None and s.size != rows) or (f is not None and f.size != rows):
            raise ValueError("scores and finished need one value per row of logits")
        if f is not None:
            _check_end_token(end_token, vocab, rows, k)
        words, stride = None, 0
        if mask is not None:
            b = np.asarray(mask, dtype=np.bool_)
            if b.shape not in ((vocab,), (rows, vocab)):
                raise ValueError("mask must be bool [vocab] or [rows, vocab]")
            stride = (vocab + 31) // 32 if b.ndim == 2 else 0
            words = np.ascontiguousarray(np.concatenate([pack_bitmask(r) for r in b.reshape(-1, vocab)]) if b.size else np.zeros(0, np.uint32))
        groups = rows // beams
        p = _lib.BeamParams(groups=groups, beams=beams, vocab=vocab, k=k, value=_lib.VALUE_F16 if x.dtype == np.float16 else _lib.VALUE_F32,
                            normalize=int(bool(normalize)), row_stride=vocab, scores=None if s is None else s.ctypes.data,
                            finished=None if f is None else f.ctypes.data, mask=None if words is None else words.ctypes.data,
                            mask_stride=stride, end_token=end_token, reserved=0)
        parents, tokens = np.empty((groups, k), dtype=np.uint32), np.empty((groups, k), dtype=np.uint32)
        out, counts = np.empty((groups, k), dtype=np.float32), np.zeros(groups, dtype=np.uint32)
        _lib.check(_lib.lib().needle_hip_beam_select(self._h, C.byref(p), x.ctypes.data, parents.ctypes.data, tokens.ctypes.data,
                                                     out.ctypes.data, counts.ctypes.data))
        return parents, tokens, out, counts

    def beam_select_device(self, d_logits, d_scores, k: int, d_parents, d_tokens, d_out_scores, d_counts, *, beams: int,
                           normalize: bool = True, d_mask=None, d_finished=None, end_token: int = 0, states=()) -> None:
        """beam_select on device tensors, and the move of what the beams carry.  d_logits: float32 / float16 / bfloat16
        [groups * beams, vocab], rows may lie apart; d_mask: int32 / uint32 words [rows, ceil(vocab / 32)] or one row of them;
        d_finished: bool / uint8 [rows]; outputs [groups, k] (int32 / uint32, int32 / uint32, float32) and int32 / uint32
        [groups], unused places -1 / -1 / -inf.  states: (src, dst) or (src, dst, axis) pairs of tensors whose dimension
        `axis` (default 0) holds groups * beams rows in src and groups * k in dst; dst's rows become copies of their
        parents' (rows of unused places stay as they were)."""
        rows, vocab, apart = _rows_of(d_logits, "d_logits")
        if (rows | vocab | beams | k) >> 32:
            _check_u32(rows=rows, vocab=vocab, beams=beams, k=k)
        if beams < 1 or rows % beams:
            raise ValueError("d_logits must be [groups * beams, vocab]")
        groups, value = rows // beams, _value(d_logits, "d_logits")
        if d_scores is not None:
            _flat(d_scores, "d_scores", _F32, rows)
        if d_finished is not None:
            _flat(d_finished, "d_finished", _FLAGS, rows)
            _check_end_token(end_token, vocab, rows, k)
        _flat(d_parents, "d_parents", _WORDS, groups * k)
        _flat(d_tokens, "d_tokens", _WORDS, groups * k)
        _flat(d_counts, "d_counts", _WORDS, groups)
        _flat(d_out_scores, "d_out_scores", _F32, groups * k)
        stride = 0
        if d_mask is not None:
            n, _, words_apart = _rows_of(d_mask.reshape(1, -1) if d_mask.dim() == 1 else d_mask, "d_mask", _WORDS, (vocab + 31) // 32)
            if n not in (1, rows):
                raise ValueError("d_mask must have one row, or one for every row of d_logits")
            stride = words_apart if n == rows and rows > 1 else 0
        arr, n_states = self._states(states, groups, beams, k) if states else (None, 0)
        self._check_device(d_logits, d_scores, d_mask, d_finished, d_parents, d_tokens, d_out_scores, d_counts)
        p = _lib.BeamParams(groups, beams, vocab, k, value, 1 if normalize else 0, apart, None if d_scores is None else d_scores.data_ptr(),
                            None if d_finished is None else d_finished.data_ptr(), None if d_mask is None else d_mask.data_ptr(), stride,
                            end_token, 0)
        _lib.check(_lib.lib().needle_hip_beam_select_device(self._h, C.byref(p), d_logits.data_ptr(), arr, n_states, d_parents.data_ptr(),
                                                            d_tokens.data_ptr(), d_out_scores.data_ptr(), d_counts.data_ptr()))

    def beam_reorder_device(self, d_parents, states, *, beams: int) -> None:
        """The move of the states alone (needle_hip_beam_reorder_device), for parents [groups, k] picked elsewhere: int32 /
        uint32 numbers below `beams`; any other number leaves its row of dst as it was."""
        if d_parents.dim() != 2 or beams < 1:
            raise ValueError("d_parents must be [groups, k]")
        groups, k = int(d_parents.shape[0]), int(d_parents.shape[1])
        _check_u32(groups=groups, beams=beams, k=k)
        _flat(d_parents, "d_parents", _WORDS, groups * k)
        arr, n_states = self._states(states, groups, beams, k)
        self._check_device(d_parents)
        _lib.check(_lib.lib().needle_hip_beam_reorder_device(self._h, d_parents.data_ptr(), groups, beams, k, arr, n_states))

    def _states(self, states, groups: int, beams: int, k: int):
        out = []
        for s in states:
            src, dst = s[0], s[1]
            axis = s[2] if len(s) > 2 else 0
            here, there = list(src.shape), list(dst.shape)
            if not 0 <= axis < len(here) or here[axis] != groups * beams or len(there) != len(here) or there[axis] != groups * k:
                raise ValueError(f"a state must have {groups * beams} rows in src and {groups * k} in dst")
            here[axis] = there[axis] = 0
            if here != there or src.dtype != dst.dtype:
                raise ValueError("a state's src and dst must differ in nothing but their rows")
            if src.get_device() != self.device or dst.get_device() != self.device:
                raise ValueError(f"states must be tensors on device {self.device}")
            if src.numel() == 0 or dst.numel() == 0:
                continue
            outer, inner, run, a, b = _state_layout(src, dst, axis)
            out.append(_lib.BeamState(src.data_ptr(), dst.data_ptr(), outer, inner, run, *a, *b))
        return ((_lib.BeamState * len(out))(*out) if out else None), len(out)


class FlatIndex:
    """Resident exact flat index (needle_hip_index, kind flat)."""

    def __init__(self, ctx: Context, base, metric: DistanceFunction, *, arith: int = _lib.ARITH_DISTANCE_RS,
                 valid=None, dim: int | None = None):
        self.ctx = ctx
        self.metric = DistanceFunction(metric)
        self._h = C.c_void_p()
        L = _lib.lib()
        if hasattr(base, "data_ptr"):  # device tensor
            if base.dim() != 2 or str(base.dtype) != "torch.float32" or not base.is_contiguous():
                raise ValueError("device base must be a contiguous float32 [n, dim] tensor")
            n, d = int(base.shape[0]), int(base.shape[1])
            vm = _mask_words(valid, n)
            _wait_for_producer(base)
            _lib.check(L.needle_hip_flat_build_device(ctx._h, base.data_ptr(), n, d, int(self.metric), arith,
                                                      vm.ctypes.data if vm is not None else None, C.byref(self._h)))
        else:
            b = _f32(base)
            if b.ndim != 2:
                if dim is None:
                    raise ValueError("an empty base needs an explicit dim")
                b = b.reshape(0, dim)
            n, d = b.shape
            if n == 0 and dim is not None:
                d = dim
            vm = _mask_words(valid, n)
            _lib.check(L.needle_hip_flat_build(ctx._h, b.ctypes.data if n else None, n, d, int(self.metric), arith,
                                               vm.ctypes.data if vm is not None else None, C.byref(self._h)))
        self.n, self.dim = n, d

    @classmethod
    def from_rows(cls, ctx: Context, rows, metric: DistanceFunction, *, arith: int = _lib.ARITH_DISTANCE_RS, valid=None):
        """Build from separately allocated rows (the reference's Vec<Vec<f32>>)."""
        keep = [_f32(r) for r in rows]
        n = len(keep)
        d = keep[0].size if n else 0
        ptrs = (C.c_void_p * max(n, 1))(*[r.ctypes.data for r in keep])
        self = cls.__new__(cls)
        self.ctx, self.metric, self._h = ctx, DistanceFunction(metric), C.c_void_p()
        vm = _mask_words(valid, n)
        _lib.check(_lib.lib().needle_hip_flat_build_rows(ctx._h, ptrs, n, d, int(metric), arith,
                                                         vm.ctypes.data if vm is not None else None, C.byref(self._h)))
        self.n, self.dim = n, d
        return self

    def close(self) -> None:
        _destroy_handle(self)

    def __del__(self):  # pragma: no cover
        try:
            self.close()
        except Exception:
            pass

    def __len__(self) -> int:
        return int(_lib.lib().needle_hip_index_len(self._h))

    def set_valid_mask(self, valid) -> None:
        vm = _mask_words(valid, self.n)
        _lib.check(_lib.lib().needle_hip_index_set_valid_mask(self._h, vm.ctypes.data if vm is not None else None))

    def append(self, rows, valid=None) -> None:
        """Rows appended behind the resident ones (needle_hip_index_append): row j of the batch becomes internal id
        len + j; only the new rows are uploaded.  `rows` is a host array or a contiguous float32 device tensor."""
        if hasattr(rows, "data_ptr"):
            if rows.dim() != 2 or str(rows.dtype) != "torch.float32" or not rows.is_contiguous() or int(rows.shape[1]) != self.dim:
                raise ValueError("device rows must be a contiguous float32 [n, dim] tensor")
            m = int(rows.shape[0])
            vm = _mask_words(valid, m)
            _wait_for_producer(rows)
            _lib.check(_lib.lib().needle_hip_index_append_device(self._h, rows.data_ptr(), m,
                                                                  vm.ctypes.data if vm is not None else None))
        else:
            r = _f32(rows)
            if r.ndim == 1:
                r = r.reshape(1, -1)
            if r.ndim != 2 or r.shape[1] != self.dim:
                raise _lib.DimensionMismatch(_lib.ERR_DIMENSION_MISMATCH,
                                             f"Dimension mismatch: expected {self.dim}, got {r.shape[-1]}")
            m = int(r.shape[0])
            vm = _mask_words(valid, m)
            _lib.check(_lib.lib().needle_hip_index_append(self._h, r.ctypes.data, m, vm.ctypes.data if vm is not None else None))
        self.n += m

    def swap_remove(self, pos: int) -> None:
        """The last row takes internal id `pos`; the index shrinks by one (Vec::swap_remove, needle_hip_index_swap_remove)."""
        _lib.check(_lib.lib().needle_hip_index_swap_remove(self._h, int(pos)))
        self.n -= 1

    def search(self, queries, k: int, *, precision: str = "fp32", filter_mask=None):
        """Host arrays in, host arrays out: (ids[q,k] uint64, dists[q,k] float32, counts[q] uint32)."""
        q = _f32(queries)
        if q.ndim == 1:
            q = q.reshape(1, -1)
        if q.ndim != 2:
            raise ValueError("queries must be [q, dim]")
        nq, qd = q.shape
        kk = max(k, 1)
        ids = np.full((nq, kk), np.iinfo(np.uint64).max, dtype=np.uint64)
        dists = np.full((nq, kk), np.inf, dtype=np.float32)
        counts = np.zeros(nq, dtype=np.uint32)
        fm = _mask_words(filter_mask, self.n)
        sp = _lib.SearchParams(k=k, nprobe=0, precision=PRECISION[precision], reserved=0,
                               filter_bitmask=fm.ctypes.data if fm is not None else None)
        _lib.check(_lib.lib().needle_hip_batch_search(self._h, q.ctypes.data if nq else None, nq, qd, C.byref(sp),
                                                      ids.ctypes.data, dists.ctypes.data, counts.ctypes.data))
        return ids[:, :k], dists[:, :k], counts

    def search_device(self, d_queries, k: int, d_out_ids, d_out_dists, d_out_counts, *, precision: str = "fp32",
                      d_filter=None) -> None:
        """Device tensors in and out (float32 [q,dim]; int64/uint64 [q,k]; float32 [q,k]; int32/uint32 [q])."""
        nq = int(d_queries.shape[0])
        _wait_for_producer(d_queries)
        if int(d_queries.shape[1]) != self.dim:
            raise _lib.DimensionMismatch(_lib.ERR_DIMENSION_MISMATCH,
                                         f"Dimension mismatch: expected {self.dim}, got {int(d_queries.shape[1])}")
        sp = _lib.SearchParams(k=k, nprobe=0, precision=PRECISION[precision], reserved=0,
                               filter_bitmask=d_filter.data_ptr() if d_filter is not None else None)
        _lib.check(_lib.lib().needle_hip_batch_search_device(self._h, d_queries.data_ptr(), nq, C.byref(sp),
                                                             d_out_ids.data_ptr(), d_out_dists.data_ptr(),
                                                             d_out_counts.data_ptr()))
