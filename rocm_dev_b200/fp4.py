"""Host side of microscaled 4-bit floating point: quantisers and products.

Two formats, named by a string: ``"mxfp4"`` (blocks of 32 share a power of two) and ``"nvfp4"`` (blocks of 16 share an
e4m3 scale, the tensor one fp32 scale).  ``include/rocm_dev_b200.h`` states the arithmetic and the held form.  The
reference project has no counterpart: its lowest precision is fp8.

Serving: quantise the weights once, a step's activations with ``quantize_fp4``, and multiply with ``skinny_gemm_fp4`` (up
to 32 rows) or ``dense_gemm_fp4``.  Training: ``quantize_fp4_both`` reads x, w and dy once each; then with ``r`` the form
along the rows and ``c`` the one along the columns

    y  = dense_gemm_fp4(x_r, w_r)        dx = dense_gemm_fp4(dy_r, w_c)        dw = dense_gemm_fp4(dy_c, x_c)
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import check, lib

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
WORKSPACE_FLOATS = 1024


class Fp4Tensor(NamedTuple):
    """A held tensor [rows, K]: ``codes`` uint8 [rows, ceil(K / 32) * 16], ``scales`` uint8 in tiles (flat),
    ``tensor_scale`` fp32[1] (``nvfp4``) or None."""
    codes: torch.Tensor
    scales: torch.Tensor
    tensor_scale: Optional[torch.Tensor]
    format: str
    rows: int
    K: int


def _format(name: str) -> int:
    try:
        return FORMATS[name]
    except (KeyError, TypeError):
        raise ValueError(f"format must be one of {sorted(FORMATS)}, got {name!r}") from None


def _type(dtype: torch.dtype) -> int:
    try:
        return _TYPES[dtype]
    except KeyError:
        raise TypeError(f"bfloat16, float16 or float32 expected, got {dtype}") from None


def scale_bytes(format: str, rows: int, K: int) -> int:
    """Size of the tiled scales of a [rows, K] tensor."""
    return (rows + 127) // 128 * ((K + 255) // 256) * (256 // BLOCK[format]) * 128


def row_bytes(K: int) -> int:
    return (K + 31) // 32 * 16


class _on:
    """``with torch.cuda.device(dev)``, at no cost where it is the current device already."""
    __slots__ = ("dev", "prev")

    def __init__(self, dev):
        self.dev = dev.index

    def __enter__(self):
        self.prev = torch.cuda.current_device()
        if self.prev != self.dev:
            torch.cuda.set_device(self.dev)

    def __exit__(self, *exc):
        if self.prev != self.dev:
            torch.cuda.set_device(self.prev)


def _empty(format: str, rows: int, K: int, tensor_scale, dev) -> Fp4Tensor:
    return Fp4Tensor(torch.empty((rows, row_bytes(K)), dtype=torch.uint8, device=dev),
                     torch.empty(scale_bytes(format, rows, K), dtype=torch.uint8, device=dev), tensor_scale, format, rows, K)


def _quantize(x: torch.Tensor, format: str, tensor_scale, along_rows: bool, along_columns: bool):
    fmt, typ = _format(format), _type(x.dtype)
    assert x.is_cuda and x.dim() == 2, "a 2-D device tensor is required (there is no CPU path)"
    rows, K = x.shape
    if rows < 1 or K < 1:
        raise ValueError(f"an empty tensor cannot be quantised: {tuple(x.shape)}")
    if x.stride(1) != 1 and K > 1 or x.stride(0) < K and rows > 1:
        x = x.contiguous()                        # transposed or overlapping views
    ldx = x.stride(0) if rows > 1 else K
    dev = x.device
    given = tensor_scale is not None
    work = None
    if fmt == 0:
        assert not given, "mxfp4 has no tensor scale"
    elif given:
        assert tensor_scale.device == dev and tensor_scale.dtype == torch.float32 and tensor_scale.numel() == 1
    else:
        tensor_scale = torch.empty(1, dtype=torch.float32, device=dev)
        work = torch.empty(WORKSPACE_FLOATS, dtype=torch.float32, device=dev)
    r = _empty(format, rows, K, tensor_scale, dev) if along_rows else None
    c = _empty(format, K, rows, tensor_scale, dev) if along_columns else None
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    with _on(dev):
        check(lib().rdb_quantize_fp4(x.data_ptr(), typ, ldx, rows, K, fmt, p(tensor_scale), given, p(r and r.codes),
                                     p(r and r.scales), p(c and c.codes), p(c and c.scales), p(work),
                                     torch.cuda.current_stream(dev).cuda_stream), "rdb_quantize_fp4")
    return r, c


def quantize_fp4(x: torch.Tensor, format: str = "nvfp4", tensor_scale: torch.Tensor | None = None) -> Fp4Tensor:
    """x [rows, K] (bf16, fp16 or fp32; rows may be a pitch apart) -> held form, blocks along the rows.
    ``tensor_scale`` (``nvfp4``): a positive fp32[1] to use in place of max|x| / 2688 - a calibrated one, for which x is
    read once instead of twice."""
    return _quantize(x, format, tensor_scale, True, False)[0]


def quantize_fp4_both(x: torch.Tensor, format: str = "nvfp4", tensor_scale: torch.Tensor | None = None):
    """(held form of x, held form of its transpose [K, rows] with blocks along x's columns), one tensor scale for both."""
    return _quantize(x, format, tensor_scale, True, True)


def _checked(t: Fp4Tensor) -> int:
    fmt = _format(t.format)
    codes, scales, ts = t.codes, t.scales, t.tensor_scale
    assert codes.is_cuda and codes.dtype == torch.uint8 and codes.shape == (t.rows, row_bytes(t.K)) and codes.is_contiguous()
    assert scales.device == codes.device and scales.dtype == torch.uint8 and scales.is_contiguous() and \
        scales.numel() == scale_bytes(t.format, t.rows, t.K)
    if fmt == 0:
        assert ts is None, "mxfp4 has no tensor scale"
    else:
        assert ts is not None and ts.device == codes.device and ts.dtype == torch.float32 and ts.numel() == 1
    return fmt


def dequantize_fp4(t: Fp4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that codes and scales stand for, [rows, K] of ``dtype``."""
    fmt, typ = _checked(t), _type(dtype)
    dev = t.codes.device
    out = torch.empty((t.rows, t.K), dtype=dtype, device=dev)
    with _on(dev):
        check(lib().rdb_dequantize_fp4(t.codes.data_ptr(), t.scales.data_ptr(), t.tensor_scale.data_ptr() if fmt else None, fmt,
                                       t.rows, t.K, out.data_ptr(), typ, torch.cuda.current_stream(dev).cuda_stream),
              "rdb_dequantize_fp4")
    return out


def _product(A: Fp4Tensor, B: Fp4Tensor, out, out_dtype):
    fmt = _checked(A)
    if B.format != A.format or B.K != A.K:
        raise ValueError(f"operands of one format and depth are required: {A.format} K={A.K}, {B.format} K={B.K}")
    _checked(B)
    dev = A.codes.device
    assert B.codes.device == dev
    if out is None:
        typ = _type(out_dtype)
        out = torch.empty((A.rows, B.rows), dtype=out_dtype, device=dev)
    else:
        typ = _type(out.dtype)
        assert out.device == dev and out.is_contiguous() and out.shape == (A.rows, B.rows)
    return (A.codes.data_ptr(), A.scales.data_ptr(), A.tensor_scale.data_ptr() if fmt else None, B.codes.data_ptr(),
            B.scales.data_ptr(), B.tensor_scale.data_ptr() if fmt else None, out.data_ptr(), typ, A.rows, B.rows, A.K, fmt), out, dev


def dense_gemm_fp4(A: Fp4Tensor, B: Fp4Tensor, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype = torch.bfloat16, tiling: int = 0, max_ctas: int = 0) -> torch.Tensor:
    """D[M,N] = A . B^T over the values of A [M,K] and B [N,K], any sizes; fp32 accumulation, rounded once to
    ``out_dtype`` (``out``'s type where it is given).  ``tiling``, ``max_ctas``: the tuner's knobs, 0 = automatic."""
    args, out, dev = _product(A, B, out, out_dtype)
    with _on(dev):
        check(lib().rdb_dense_gemm_fp4_tuned(*args, tiling, max_ctas, torch.cuda.current_stream(dev).cuda_stream),
              "rdb_dense_gemm_fp4")
    return out


def skinny_gemm_fp4(A: Fp4Tensor, B: Fp4Tensor, out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
                    flags: int = 0) -> torch.Tensor:
    """The same product for at most 32 rows of A (decode): a stream over B.  ``flags``: 0 or ``OVERLAP_PRIOR_KERNEL`` (the
    launch may request B while the preceding kernel of the stream drains; that kernel must not write B)."""
    args, out, dev = _product(A, B, out, out_dtype)
    with _on(dev):
        check(lib().rdb_skinny_gemm_fp4(*args, flags, torch.cuda.current_stream(dev).cuda_stream), "rdb_skinny_gemm_fp4")
    return out


def pack_fp4_scales(scales: torch.Tensor, format: str, K: int) -> torch.Tensor:
    """Plain scale bytes [rows, ceil(K / block)] (as checkpoints hold them) -> the tiles that the kernels read."""
    b = BLOCK[format]
    rows, blocks = scales.shape
    assert scales.dtype == torch.uint8 and blocks == (K + b - 1) // b
    full = torch.zeros(((rows + 127) // 128 * 128, (K + 255) // 256 * (256 // b)), dtype=torch.uint8, device=scales.device)
    full[:rows, :blocks] = scales
    return full.reshape(full.shape[0] // 128, 4, 32, -1, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def unpack_fp4_scales(t: Fp4Tensor) -> torch.Tensor:
    """The plain scale bytes [rows, ceil(K / block)] of a held tensor."""
    b = BLOCK[t.format]
    full = t.scales.reshape((t.rows + 127) // 128, -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape((t.rows + 127) // 128 * 128, -1)
    return full[:t.rows, :(t.K + b - 1) // b].contiguous()
