"""Microscaled formats: quantise, read back, multiply, and the norm that quantises its output.

A quantised matrix is (codes, scales).  "mxfp4" codes are uint8, two elements to a byte (the even one in the
low half); "mxfp8" codes are float8_e4m3fn.  Every 32 elements of the last dimension share a power of two,
2^(scale - 127), held as uint8 in "rows" layout ((..., K / 32)) or in the order the tensor cores read ("tc",
one flat buffer; include/s24.h gives both).  The product takes "tc"; "rows" is what checkpoints hold.

Like the rest of the library these are inference calls: results carry no gradient.

A decoding step's calls are a few microseconds long on the GPU, so the way to the launch is kept short: plain
integers for pointers and devices, the stream's handle without a Stream object, outputs allocated from an empty
tensor of their type (1.4 us instead of 2.3 for a new one by type and device).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib as L
from .ops import _NVTX, _after_gemm, _on_device, _require_cuda, _tile_cfg

_DT = {torch.float16: L.FP16, torch.bfloat16: L.BF16, torch.float32: L.FP32}
_FMT = {"mxfp4": L.MXFP4, "mxfp8": L.MXFP8}
_CODES = {torch.uint8: L.MXFP4, torch.float8_e4m3fn: L.MXFP8}
_SCALES = {"rows": L.SCALES_ROWS, "tc": L.SCALES_TC}
_SCALE_TYPES = (torch.uint8, torch.float8_e8m0fnu)
_EMPTY = {}   # (device index, type) -> a tensor without elements


def _new(device: int, dtype: torch.dtype, *shape: int) -> torch.Tensor:
    e = _EMPTY.get((device, dtype))
    if e is None:
        e = torch.empty(0, dtype=dtype, device=torch.device("cuda", device))
        if type(e) is torch.Tensor:   # not one that a dispatch mode put in its place
            _EMPTY[(device, dtype)] = e
    return e.new_empty(*shape)


def _device_of(*ts: Optional[torch.Tensor]) -> int:
    d = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != d or d < 0:
            _require_cuda(*ts)   # says which and why
    return d


def _call(name: str, t: torch.Tensor, device: int, *args) -> None:
    """library call `name` on t's device and its current stream"""
    fn = getattr(L.lib(), name)
    if torch._C._cuda_getDevice() == device and not _NVTX:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with _on_device(t, name[4:]):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc != L.OK:
        L.check(rc)


def mx_scales_numel(R: int, K: int) -> int:
    """bytes of a tensor-core-order scale buffer for an (R, K) matrix"""
    return -(-R // 128) * -(-K // 128) * 512 if R > 0 and K > 0 else 0


def _rows_of(t: torch.Tensor) -> Tuple[int, int]:
    shape = t.shape
    if len(shape) == 2:
        return shape
    if not shape:
        raise RuntimeError("expected a tensor of at least one dimension")
    r = 1
    for n in shape[:-1]:
        r *= n
    return r, shape[-1]


def _matrix(t: torch.Tensor, R: int, width: int, step: int) -> Tuple[torch.Tensor, int]:
    """t as (R, width) rows with unit column stride, whose pointer and row stride are multiples of `step` bytes
    (copied if they are not), and the row stride in elements"""
    if t.dim() != 2:
        t = t.reshape(R, width)
    stride, inner = t.stride()
    if R == 1:
        stride = width
    if inner != 1 and width > 1 or stride < width or stride * t.element_size() % step or t.data_ptr() % step:
        return t.clone(memory_format=torch.contiguous_format), width
    return t, stride


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _check_dense(x: torch.Tensor, fmt: str) -> Tuple[int, int, int]:
    """(format, R, K) of a quantisation of x"""
    f = _FMT.get(fmt)
    if f is None:
        raise ValueError(f"unknown format {fmt!r} (have 'mxfp4' and 'mxfp8')")
    R, K = _rows_of(x)
    if K % 32 != 0:
        raise RuntimeError(f"the last dimension must be divisible by 32, the size of a block (got {K})")
    return f, R, K


def _new_quantized(x: torch.Tensor, d: int, R: int, K: int, fmt: int, want_rows: bool, want_tc: bool):
    if not want_rows and not want_tc:
        raise RuntimeError("ask for at least one layout of the scales (want_rows, want_tc)")
    lead = (R,) if x.dim() == 2 else x.shape[:-1]
    codes = _new(d, torch.uint8, *lead, K // 2) if fmt == L.MXFP4 else _new(d, torch.float8_e4m3fn, *lead, K)
    return codes, _new(d, torch.uint8, *lead, K // 32) if want_rows else None, _new(d, torch.uint8, mx_scales_numel(R, K)) if want_tc else None


def _codes_of(codes: torch.Tensor) -> Tuple[int, int, int]:
    """(format, R, K) of a codes tensor"""
    fmt = _CODES.get(codes.dtype)
    if fmt is None:
        raise RuntimeError(f"Invalid datatype {codes.dtype} of codes (uint8 for mxfp4, float8_e4m3fn for mxfp8)")
    R, K = _rows_of(codes)
    if fmt == L.MXFP4:
        K *= 2
    if K % 32 != 0:
        raise RuntimeError(f"the last dimension must be divisible by 32, the size of a block (got {K})")
    return fmt, R, K


def _check_scales(scales: torch.Tensor, layout: str, R: int, K: int) -> None:
    """the kernels read whole records, and every row: a short buffer would be read past its end"""
    if layout not in _SCALES:
        raise ValueError(f"unknown scale layout {layout!r} (have 'rows' and 'tc')")
    need = R * (K // 32) if layout == "rows" else mx_scales_numel(R, K)
    if scales.numel() != need or scales.dtype not in _SCALE_TYPES or not scales.is_contiguous():
        raise RuntimeError(f"{layout!r} scales of a ({R}, {K}) matrix are {need} contiguous bytes (uint8), got {scales.numel()} of "
                           f"{scales.dtype}")


def mx_quantize(x: torch.Tensor, fmt: str = "mxfp4", want_rows: bool = True, want_tc: bool = False):
    """Quantise x (..., K), float16 / bfloat16 / float32, along its last dimension in one pass.

    Returns (codes, scales (..., K / 32) or None, tensor-core-order scales or None).
    """
    dt = _DT.get(x.dtype)
    if dt is None:
        raise RuntimeError(f"Invalid datatype {x.dtype} of dense matrix")
    f, R, K = _check_dense(x, fmt)
    d = _device_of(x)
    codes, scales, tc = _new_quantized(x, d, R, K, f, want_rows, want_tc)
    if R * K:
        m, ld = _matrix(x, R, K, 32)
        _call("s24_mx_quantize", x, d, m.data_ptr(), R, K, ld, dt, f, codes.data_ptr(), _ptr(scales), _ptr(tc))
    return codes, scales, tc


def mx_dequantize(codes: torch.Tensor, scales: torch.Tensor, layout: str = "rows", dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Read (codes, scales) back as a (..., K) tensor of `dtype` (float16, bfloat16 or float32), rounded once."""
    f, R, K = _codes_of(codes)
    dt = _DT.get(dtype)
    if dt is None:
        raise RuntimeError(f"Invalid datatype {dtype} of dense matrix")
    _check_scales(scales, layout, R, K)
    d = _device_of(codes, scales)
    out = _new(d, dtype, R, K) if codes.dim() == 2 else _new(d, dtype, *codes.shape[:-1], K)
    if R * K:
        c = codes if codes.is_contiguous() and codes.data_ptr() % 32 == 0 else codes.clone(memory_format=torch.contiguous_format)
        _call("s24_mx_dequantize", codes, d, c.data_ptr(), scales.data_ptr(), _SCALES[layout], out.data_ptr(), R, K, f, dt)
    return out


def mx_scales_convert(scales: torch.Tensor, from_layout: str, to_layout: str, R: int, K: int) -> torch.Tensor:
    """Re-lay the scales of an (R, K) matrix between "rows" ((R, K / 32)) and "tc"."""
    if R < 0 or K < 0 or K % 32 != 0:
        raise RuntimeError(f"the last dimension must be divisible by 32, the size of a block (got {K})")
    _check_scales(scales, from_layout, R, K)
    if to_layout not in _SCALES or to_layout == from_layout:
        raise ValueError(f"cannot convert scales from {from_layout!r} to {to_layout!r}")
    d = _device_of(scales)
    out = _new(d, torch.uint8, R, K // 32) if to_layout == "rows" else _new(d, torch.uint8, mx_scales_numel(R, K))
    if R * K:
        _call("s24_mx_scales_convert", scales, d, scales.data_ptr(), _SCALES[from_layout], out.data_ptr(), _SCALES[to_layout], R, K)
    return out


def mx_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None, fmt: str = "mxfp8",
                want_rows: bool = True, want_tc: bool = False):
    """Root-mean-square norm over the last dimension with the residual's addition, quantised as it is computed:
    h = x + residual (rounded to x's type; x itself without a residual), y = h * weight / sqrt(mean(h^2) + eps).

    x and residual (..., K) and weight (K) share a type, float16 or bfloat16; K is at most 65536.  y is not rounded
    before it is quantised.  Returns (codes, scales or None, tensor-core-order scales or None, h).
    """
    dtype = x.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise RuntimeError(f"Invalid datatype {dtype} of dense matrix")
    f, R, K = _check_dense(x, fmt)
    if weight.dtype is not dtype or weight.dim() != 1 or weight.shape[0] != K:
        raise RuntimeError(f"`weight` must be a ({K},) {dtype} tensor, got {tuple(weight.shape)} {weight.dtype}")
    if residual is not None and (residual.dtype is not dtype or residual.shape != x.shape):
        raise RuntimeError(f"`residual` must be a {tuple(x.shape)} {dtype} tensor, got {tuple(residual.shape)} {residual.dtype}")
    if K > L.MX_NORM_MAX_K:
        raise RuntimeError(f"rows of at most {L.MX_NORM_MAX_K} elements (got {K})")
    d = _device_of(x, weight, residual)
    codes, scales, tc = _new_quantized(x, d, R, K, f, want_rows, want_tc)
    h = x if residual is None else torch.empty_like(x, memory_format=torch.contiguous_format)
    if R * K:
        m, ldx = _matrix(x, R, K, 32)
        r, ldr = (None, 0) if residual is None else _matrix(residual, R, K, 32)
        w = weight if weight.stride(0) == 1 and weight.data_ptr() % 32 == 0 else weight.clone(memory_format=torch.contiguous_format)
        _call("s24_mx_rms_norm", x, d, m.data_ptr(), _ptr(r), w.data_ptr(), None if residual is None else h.data_ptr(), R, K, ldx, ldr, eps,
              _DT[dtype], f, codes.data_ptr(), _ptr(scales), _ptr(tc))
    return codes, scales, tc, h


def mx_matmul(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
              out: Optional[torch.Tensor] = None, manual_config: Optional[dict] = None) -> torch.Tensor:
    """C (..., N) = deq(a) (..., K) @ deq(b) (N, K)^T with fp32 accumulation, rounded once to `out_dtype`.

    a and b are codes of either format, their scales in tensor-core order (`want_tc=True`, or mx_scales_convert);
    K must be a multiple of 128 where the formats differ.  `out` (2-dimensional, of `out_dtype`) must not
    overlap the operands.  `manual_config` has a tile ("BM" and "BN": 256 x 256, 256 x 128 or 128 x 128) or "SPLIT", the
    number of CTAs that share K (1, 2, 4 or 8; 1 where K has fewer steps than that).  As with every product of the library, make the first call on a device before a stream
    capture.
    """
    fa, M, K = _codes_of(a)
    fb, N, Kb = _codes_of(b)
    if b.dim() != 2:
        raise RuntimeError(f"b must be 2-dimensional (N, K), got {b.dim()} dimensions")
    if K != Kb or K == 0:
        raise RuntimeError(f"a has {K} elements a row and b {Kb}: they must be equal and not 0")
    step_a = step_b = 16
    if fa != fb:
        if K % 128 != 0:
            raise RuntimeError(f"operands of different formats need K % 128 == 0 (got {K})")
        step_a, step_b = (32, 16) if fa == L.MXFP4 else (16, 32)
    dt = _DT.get(out_dtype)
    if dt is None:
        raise RuntimeError(f"Invalid datatype {out_dtype} of the product")
    _check_scales(a_scales, "tc", M, K)
    _check_scales(b_scales, "tc", N, K)
    d = _device_of(a, a_scales, b, b_scales, out)
    if out is None:
        c = _new(d, out_dtype, M, N) if a.dim() == 2 else _new(d, out_dtype, *a.shape[:-1], N)
        ldc = N
    else:
        c = out
        ldc = c.stride(0) if c.dim() == 2 and M > 1 else N
        if tuple(c.shape) != (M, N) or c.dtype != out_dtype or (N > 1 and c.stride(1) != 1) or ldc < N:
            raise RuntimeError(f"`out` must be a ({M}, {N}) {out_dtype} tensor with unit column stride and rows that do not overlap")
    if M * N:
        width = K // 2 if fa == L.MXFP4 else K
        ma, lda = _matrix(a, M, width, step_a)
        mb, ldb = _matrix(b, N, K // 2 if fb == L.MXFP4 else K, step_b)
        _call("s24_mx_matmul", a, d, ma.data_ptr(), a_scales.data_ptr(), mb.data_ptr(), b_scales.data_ptr(), c.data_ptr(), M, N, K, lda, ldb,
              ldc, fa, fb, dt, None if manual_config is None else _tile_cfg(manual_config))
        _after_gemm(a)
    return c
