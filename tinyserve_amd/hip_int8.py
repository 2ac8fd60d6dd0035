"""The 8-bit integer path of a step's projections on MI355X (``csrc/int8_rows.hip``,
``csrc/int8_linear.hip``): activations quantised per token, weights per output channel, their
products on the int8 matrix cores.

A decoder layer's projections (src/tinyserve/model.py:137-179) with 8-bit weights:

    h    = rms_norm(x)                  rms_norm_rows_int8(x, w, eps)
    qkv  = F.linear(h, W_qkv)           int8_linear(h, W_qkv, dtype)
    x    = x + F.linear(attn, W_o)      y = int8_linear(quantize_rows(attn), W_o, dtype)
    h    = rms_norm(x)                  add_rms_norm_rows_int8(x, y, w, eps)   (x updated)
    act  = silu(gate) * up              silu_mul_int8(int8_linear(h, W_gate_up, dtype))
    x    = x + F.linear(act, W_down)    int8_linear(act, W_down, dtype), added by the next norm

``Int8Rows`` holds such a matrix: codes ``q`` (int8 ``[M, K]``) and one float32 ``scale`` per
row; it stands for ``q * scale[:, None]``. Weights ``[N, K]`` are quantised once by
``quantize_rows(w)``. The reference keeps every weight in one float type, so no function of it
corresponds. These are for inference: no gradient flows through them.

Every launch goes on torch's current stream of the inputs' device, never synchronises, and
allocates only its results, by torch's caching allocator, so a HIP graph can capture them.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from tinyserve_amd import _lib

PLAIN, NORM, ADD_NORM, SILU = 0, 1, 2, 3
MAX_K = 131071  # products of longer rows could pass an int32
MAX_DIM = 1 << 30  # rows or columns of one call
MAX_STRIDE = 1 << 23  # bytes between rows that ts_int8_linear reads in tiles


class Int8Rows(NamedTuple):
    """An 8-bit matrix with one scale per row: ``q`` int8 ``[M, K]``, unit column stride,
    ``scale`` float32 ``[M]``. A row with a NaN scale stands for NaN."""

    q: torch.Tensor
    scale: torch.Tensor


_current_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream
_empty = torch.empty
_INT8, _FLOAT = torch.int8, torch.float32


# The compiled host path of the calls (csrc/fastint8.cpp), bound by the first call that goes
# through Python; None where it is not built, and then every call does.
_fast = None
_bound = False


def _bind_fast() -> None:
    global _fast, _bound
    _bound = True
    try:
        from tinyserve_amd import _fastint8
    except ImportError:
        return
    lib = _lib.load()
    names = ("ts_int8_quantize_rows", "ts_int8_embedding", "ts_int8_linear", "ts_int8_linear_workspace", "ts_int8_pad_rows")
    _fastint8.bind(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names), Int8Rows, _stream)
    _fast = _fastint8


def _readable(q: torch.Tensor) -> bool:
    """Whether every row may be read up to a whole 16 columns."""
    m, k = q.shape
    need = (k + 15) // 16 * 16
    return q.stride(0) >= need and q.storage_offset() + (m - 1) * q.stride(0) + need <= q.untyped_storage().nbytes()


def _fits(q: torch.Tensor) -> bool:
    """Whether tiles can read ``q``: rows 16-byte aligned, readable to a whole 16 columns and at
    most ``MAX_STRIDE`` apart."""
    stride = q.stride(0)
    return q.data_ptr() % 16 == 0 and stride % 16 == 0 and stride <= MAX_STRIDE and (q.shape[1] % 16 == 0 or _readable(q))


def _padded(x: torch.Tensor, w: torch.Tensor, dev: int) -> tuple[torch.Tensor, torch.Tensor]:
    """``x`` and ``w``, copied to 16-byte aligned rows padded with zeros where tiles cannot read
    them; both in one launch."""
    k = x.shape[1]
    stride = (k + 15) & ~15
    args: list[int | None] = []
    got = []
    for q in (x, w):
        if _fits(q):
            args += [None, 0, None, 0]
            got.append(q)
        else:
            out = _empty((q.shape[0], stride), dtype=_INT8, device=q.device)
            args += [q.data_ptr(), q.stride(0), out.data_ptr(), q.shape[0]]
            got.append(out)
    _lib.call("ts_int8_pad_rows", *args, stride, k, _stream(dev))
    return got[0], got[1]


def _matrix(x: torch.Tensor, what: str) -> tuple[int, int, int]:
    """Rows, columns and dtype code of a float matrix ``[T, N]``."""
    code = _lib.DTYPES.get(x.dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {x.dtype}: float32, float16 or bfloat16")
    if x.dim() != 2:
        raise ValueError(f"{what} must be a [T, N] tensor, got {tuple(x.shape)}")
    t, n = x.shape
    if x.stride(1) != 1 and n > 1:
        raise ValueError(f"{what} must be row-contiguous, got {tuple(x.shape)} with strides {x.stride()}")
    if t > MAX_DIM or n > MAX_DIM:
        raise ValueError(f"{what}: at most {MAX_DIM} rows and columns, got {(t, n)}")
    return t, n, code


def _norm_args(weight: torch.Tensor, x: torch.Tensor, n: int, eps: float) -> None:
    if weight.dtype is not x.dtype or weight.shape != (n,) or not weight.is_contiguous():
        raise ValueError(f"the weight must be a contiguous {x.dtype} vector of {n}, got {weight.dtype} {tuple(weight.shape)}")
    if not eps > 0:
        raise ValueError(f"eps must be positive, got {eps}")


def _codes(r: Int8Rows, what: str) -> tuple[int, int]:
    """Rows and columns of an ``Int8Rows``."""
    q, scale = r
    if q.dtype is not _INT8 or q.dim() != 2:
        raise ValueError(f"{what}: codes must be int8 [M, K], got {q.dtype} {tuple(q.shape)}")
    m, k = q.shape
    if q.stride(1) != 1 and k > 1:
        raise ValueError(f"{what}: codes must be row-contiguous, got {(m, k)} with strides {q.stride()}")
    if scale.dtype is not _FLOAT or scale.shape != (m,) or not scale.is_contiguous():
        raise ValueError(f"{what}: scales must be contiguous float32 [{m}], got {scale.dtype} {tuple(scale.shape)}")
    if m > MAX_DIM or k > MAX_DIM:
        raise ValueError(f"{what}: at most {MAX_DIM} rows and columns, got {(m, k)}")
    return m, k


def _quantize(form: int, x: torch.Tensor, y: torch.Tensor | None, weight: torch.Tensor | None, eps: float, dev: int,
              t: int, n: int, code: int) -> Int8Rows:  # fmt: skip
    """One launch of ``ts_int8_quantize_rows``. Codes' rows start at multiples of 16 bytes."""
    if not _bound:
        _bind_fast()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return _quantize(form, x, y, weight, eps, dev, t, n, code)
    stride = (n + 15) & ~15
    q = _empty((t, stride), dtype=_INT8, device=x.device)
    scale = _empty(t, dtype=_FLOAT, device=x.device)
    if t and n:
        _lib.call("ts_int8_quantize_rows", x.data_ptr(), y if y is None else y.data_ptr(),
                  weight if weight is None else weight.data_ptr(), q.data_ptr(), scale.data_ptr(), t, n, x.stride(0),
                  0 if y is None else y.stride(0), stride, eps, form, code, _stream(dev))  # fmt: skip
    elif t:
        scale.zero_()  # rows of no columns
    return Int8Rows(q if stride == n else q[:, :n], scale)


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """Rows of ``x [T, N]`` in 8 bits: ``a = max|x[t]|``, ``q = rint(x * (127 / a))``,
    ``scale = a / 127``. A row of zeros (or below 2^-100) gets scale 0, one that holds a NaN or
    an infinity scale NaN; both get zero codes."""
    if _fast is not None and (got := _fast.quantize(PLAIN, x, None, None, 0.0)) is not None:
        return got
    t, n, code = _matrix(x, "x")
    return _quantize(PLAIN, x, None, None, 0.0, _lib.require_device(x), t, n, code)


def rms_norm_rows_int8(x: torch.Tensor, weight: torch.Tensor, eps: float) -> Int8Rows:
    """``quantize_rows`` of RMSNorm of each row of ``x``, in one launch. The norm is not rounded
    to x's dtype before it is quantised (``rms_norm_rows`` rounds twice). ``eps`` is positive."""
    if _fast is not None and (got := _fast.quantize(NORM, x, None, weight, eps)) is not None:
        return got
    t, n, code = _matrix(x, "x")
    _norm_args(weight, x, n, eps)
    return _quantize(NORM, x, None, weight, eps, _lib.require_device(x, weight), t, n, code)


def add_rms_norm_rows_int8(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, eps: float) -> Int8Rows:
    """``x.add_(y)``, rounded to its dtype, then ``rms_norm_rows_int8(x, weight, eps)``, in one
    launch. ``x`` is updated in place; its rows must not overlap each other's, nor ``y``'s unless
    ``y`` is ``x``."""
    if _fast is not None and (got := _fast.quantize(ADD_NORM, x, y, weight, eps)) is not None:
        return got
    t, n, code = _matrix(x, "x")
    _norm_args(weight, x, n, eps)
    if y.dtype is not x.dtype or y.shape != x.shape or (y.stride(1) != 1 and n > 1):
        raise ValueError(f"y must be row-contiguous {tuple(x.shape)} {x.dtype}, got {tuple(y.shape)} {y.dtype}")
    return _quantize(ADD_NORM, x, y, weight, eps, _lib.require_device(x, y, weight), t, n, code)


def silu_mul_int8(gate_up: torch.Tensor) -> Int8Rows:
    """``quantize_rows(F.silu(gate) * up)`` of ``[gate | up]`` rows ``[T, 2N]``, in one launch,
    in float32 up to the 8 bits (``silu_mul`` rounds each factor to the dtype)."""
    if _fast is not None and (got := _fast.quantize(SILU, gate_up, None, None, 0.0)) is not None:
        return got
    t, n, code = _matrix(gate_up, "gate_up")
    if n % 2:
        raise ValueError(f"need [gate | up] rows of an even width, got {(t, n)}")
    return _quantize(SILU, gate_up, None, None, 0.0, _lib.require_device(gate_up), t, n // 2, code)


def int8_linear(x: Int8Rows, w: Int8Rows, dtype: torch.dtype, out: torch.Tensor | None = None) -> torch.Tensor:
    """``F.linear`` of 8-bit rows: ``(q_x . q_w^T) * scale_x[:, None] * scale_w``, ``[M, N]`` in
    ``dtype``. The integer sums are exact and rounded to float32 once.

    Args:
        x: ``[M, K]`` tokens. w: ``[N, K]`` weights, a scale per output channel. K up to 131071;
            rows that do not start at multiples of 16 bytes (the functions here make them so)
            are copied first where the product runs in tiles.
        out: ``[M, N]`` in ``dtype``, unit column stride (default: a new tensor).
    """
    if _fast is not None and (got := _fast.linear(x, w, dtype, out)) is not None:
        return got
    m, k = _codes(x, "x")
    n, kw = _codes(w, "w")
    xq, xs = x
    wq, ws = w
    if kw != k:
        raise ValueError(f"x has {k} columns but w is {(n, kw)}")
    if k > MAX_K:
        raise ValueError(f"K is at most {MAX_K} (the sums are int32), got {k}")
    code = _lib.DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {dtype}: float32, float16 or bfloat16")
    dev = _lib.require_device(xq, xs, wq, ws)
    if not _bound:
        _bind_fast()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return int8_linear(x, w, dtype, out)
    if out is None:
        out = _empty((m, n), dtype=dtype, device=xq.device)
        stride = n
    else:
        if out.shape != (m, n) or out.dtype != dtype or (out.stride(1) != 1 and n > 1) or (m > 1 and out.stride(0) < n):
            raise ValueError(f"out must be {dtype} [{m}, {n}] with unit column stride, got {out.dtype} {tuple(out.shape)}")
        if _lib.require_device(out) != dev:
            raise ValueError("out is on another device")
        stride = out.stride(0)
    if m and n:
        padded = k % 16 == 0 or (_readable(xq) and _readable(wq))
        need = _lib.load().ts_int8_linear_workspace(m, n, k)
        workspace = _empty(need, dtype=torch.uint8, device=xq.device) if need else None  # kept until both launches
        sums = None if workspace is None else workspace.data_ptr()
        rc = _lib.call_status("ts_int8_linear", xq.data_ptr(), xq.stride(0), xs.data_ptr(), wq.data_ptr(), wq.stride(0),
                              ws.data_ptr(), out.data_ptr(), stride, m, n, k, padded, code, sums, need, _stream(dev))  # fmt: skip
        if rc == _lib.TS_EUNSUPPORTED:  # it runs in tiles, which need aligned rows
            xq, wq = _padded(xq, wq, dev)
            _lib.call("ts_int8_linear", xq.data_ptr(), xq.stride(0), xs.data_ptr(), wq.data_ptr(), wq.stride(0),
                      ws.data_ptr(), out.data_ptr(), stride, m, n, k, 1, code, sums, need, _stream(dev))  # fmt: skip
        elif rc:
            raise ValueError(f"ts_int8_linear: {_lib.load().ts_strerror(rc).decode()}")
    return out


def int8_embedding(table: Int8Rows, ids: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Rows ``ids`` of an 8-bit table as ``dtype``: ``table.q[ids] * table.scale[ids][:, None]``,
    ``[T, N]``, rounded once. ids: int64 ``[T]`` (int32 is accepted and widened); an id outside
    the table gives a row of NaN."""
    if _fast is not None and (got := _fast.embedding(table, ids, dtype)) is not None:
        return got
    if ids.dim() != 1 or ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"ids must be a [T] int64 or int32 tensor, got {ids.dtype} {tuple(ids.shape)}")
    return _rows_of(table, ids, dtype)


def dequantize_rows(rows: Int8Rows, dtype: torch.dtype) -> torch.Tensor:
    """The values that ``rows`` stands for, ``q * scale[:, None]``, in ``dtype``, rounded once."""
    if _fast is not None and (got := _fast.embedding(rows, None, dtype)) is not None:
        return got
    return _rows_of(rows, None, dtype)


def _rows_of(table: Int8Rows, ids: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor:
    v, n = _codes(table, "table")
    q, scale = table
    code = _lib.DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {dtype}: float32, float16 or bfloat16")
    t = v
    if ids is None:
        dev = _lib.require_device(q, scale)
    else:
        t = ids.shape[0]
        if t and not v:
            raise ValueError("the table has no rows")
        if t > MAX_DIM:
            raise ValueError(f"at most {MAX_DIM} ids, got {t}")
        dev = _lib.require_device(q, scale, ids)
    if not _bound:
        _bind_fast()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return _rows_of(table, ids, dtype)
    out = _empty((t, n), dtype=dtype, device=q.device)
    if t and n:
        if ids is not None and (ids.dtype is not torch.int64 or not ids.is_contiguous()):
            ids = ids.to(torch.int64).contiguous()
        _lib.call("ts_int8_embedding", q.data_ptr(), q.stride(0), scale.data_ptr(), v,
                  ids if ids is None else ids.data_ptr(), out.data_ptr(), n, t, n, code, _stream(dev))  # fmt: skip
    return out
