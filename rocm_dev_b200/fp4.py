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

import ctypes as C

import torch

from ._lib import check, lib

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
WORKSPACE_FLOATS = 1024
_BYTE = torch.uint8

# A step's calls are short: what a call costs on the host shows.  These two are the cheap forms of
# torch.cuda.current_device() and torch.cuda.current_stream(dev).cuda_stream (0.1 us each instead of 0.2 and 2.2).
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def scale_bytes(format: str, rows: int, K: int) -> int:
    """Size of the tiled scales of a [rows, K] tensor."""
    return (rows + 127) // 128 * ((K + 255) // 256) * (256 // BLOCK[format]) * 128


def row_bytes(K: int) -> int:
    """Bytes of a row of codes."""
    return (K + 31) // 32 * 16


def _format(name: str) -> int:
    fmt = FORMATS.get(name) if isinstance(name, str) else None
    if fmt is None:
        raise ValueError(f"format must be one of {sorted(FORMATS)}, got {name!r}")
    return fmt


def _type(dtype: torch.dtype) -> int:
    typ = _TYPES.get(dtype)
    if typ is None:
        raise TypeError(f"bfloat16, float16 or float32 expected, got {dtype}")
    return typ


class Fp4Tensor:
    """A held tensor [rows, K]: ``codes`` uint8 [rows, row_bytes(K)], ``scales`` uint8 in tiles (flat, scale_bytes(format,
    rows, K)), ``tensor_scale`` fp32[1] (``nvfp4``) or None, all on ``device``."""
    __slots__ = ("format", "rows", "K", "device", "_fmt", "_args", "_parts", "_buffer")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, tensor_scale, format: str, rows: int, K: int):
        fmt = _format(format)
        index = codes.get_device()
        if (codes.dtype is not _BYTE or codes.shape != (rows, (K + 31) // 32 * 16) or not codes.is_contiguous()
                or scales.dtype is not _BYTE or scales.numel() != (rows + 127) // 128 * ((K + 255) // 256) * (2048 if fmt else 1024)
                or not scales.is_contiguous() or scales.get_device() != index):
            raise ValueError(f"codes must be contiguous uint8 [{rows}, {row_bytes(K)}] and scales {scale_bytes(format, rows, K)} "
                             "contiguous bytes on one device")
        if fmt == 0:
            if tensor_scale is not None:
                raise ValueError("mxfp4 has no tensor scale")
            scale_ptr = None
        elif (tensor_scale is None or tensor_scale.dtype is not torch.float32 or tensor_scale.numel() != 1
              or tensor_scale.get_device() != index):
            raise ValueError("nvfp4 needs a tensor scale: one fp32 on the device of the codes")
        else:
            scale_ptr = tensor_scale.data_ptr()
        self._args = (codes.data_ptr(), scales.data_ptr(), scale_ptr)
        self._parts = (codes, scales, tensor_scale)
        self.format, self.rows, self.K, self.device, self._fmt = format, rows, K, codes.device, fmt

    def _views(self):
        # a quantiser's result is one allocation (codes, scales, tensor scale at the addresses in _args); its tensors are
        # made when they are asked for
        if self._parts is None:
            buf, given = self._buffer
            base = buf.data_ptr()
            codes, scales, ts = self._args
            rb, sb = row_bytes(self.K), scale_bytes(self.format, self.rows, self.K)
            part = lambda at, n: buf[at - base:at - base + n]  # noqa: E731
            self._parts = (part(codes, self.rows * rb).view(self.rows, rb), part(scales, sb),
                           given if ts is None or given is not None else part(ts, 4).view(torch.float32))
        return self._parts

    @property
    def codes(self) -> torch.Tensor:
        return self._views()[0]

    @property
    def scales(self) -> torch.Tensor:
        return self._views()[1]

    @property
    def tensor_scale(self):
        return self._views()[2]

    def to(self, device) -> "Fp4Tensor":
        """The same tensor on another device (or on the host, to be stored)."""
        move = lambda t: None if t is None else t.to(device)  # noqa: E731
        return Fp4Tensor(move(self.codes), move(self.scales), move(self.tensor_scale), self.format, self.rows, self.K)

    def __repr__(self) -> str:
        return f"Fp4Tensor({self.format}, [{self.rows}, {self.K}], {self.device})"


def _device(dev: torch.device) -> int:
    if dev.type != "cuda":
        raise ValueError(f"device tensors required, got one on {dev} (there is no CPU path)")
    return dev.index


class _Entries:
    """The library's functions, through csrc/fastcall.c where it was built, else through ctypes."""

    def __init__(self):
        L = lib()
        names = ("rdb_quantize_fp4", "rdb_dequantize_fp4", "rdb_dense_gemm_fp4_tuned", "rdb_skinny_gemm_fp4")
        try:
            from . import _fastcall as fast
            fast.bind(*(C.cast(getattr(L, n), C.c_void_p).value for n in names))
            found = (fast.quantize, fast.dequantize, fast.dense, fast.skinny)
        except ImportError:
            found = tuple(getattr(L, n) for n in names)
        self.quantize, self.dequantize, self.dense, self.skinny = found


_entries = None


def _call(name: str, dev: int, *args) -> None:
    """The entry `name` with args and the current stream of device dev, dev being made the current device."""
    global _entries
    if _entries is None:
        _entries = _Entries()
    fn = getattr(_entries, name)
    if _current_device() == dev:
        code = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            code = fn(*args, _raw_stream(dev))
    if code:
        check(code, f"{name} (4-bit)")


def _held(form: str, fmt: int, rows: int, K: int, dev, buffer, at: int, scales: int, scale_ptr) -> Fp4Tensor:
    t = Fp4Tensor.__new__(Fp4Tensor)
    t.format, t.rows, t.K, t.device, t._fmt = form, rows, K, dev, fmt
    t._args, t._parts, t._buffer = (at, scales, scale_ptr), None, buffer
    return t


def _quantize(x: torch.Tensor, format: str, tensor_scale, both: bool):
    fmt, typ = _format(format), _type(x.dtype)
    dev = x.device
    index = _device(dev)
    if x.dim() != 2:
        raise ValueError(f"a 2-D tensor is required, got {tuple(x.shape)}")
    rows, K = x.shape
    if rows < 1 or K < 1:
        raise ValueError(f"an empty tensor cannot be quantised: {tuple(x.shape)}")
    ldx, unit = x.stride()
    if unit != 1 and K > 1 or ldx < K and rows > 1:
        x = x.contiguous()                        # transposed or overlapping views
        ldx = K
    elif rows == 1:
        ldx = K
    given = tensor_scale is not None
    if given:
        if fmt == 0:
            raise ValueError("mxfp4 has no tensor scale")
        if not (tensor_scale.dtype is torch.float32 and tensor_scale.numel() == 1 and tensor_scale.device == dev):
            raise ValueError(f"the tensor scale must be one fp32 on {dev}")
    # one allocation (every part a multiple of 16 bytes): codes and scales of either direction, the tensor scale, and the
    # scratch that the call alone uses
    codes, scales = rows * ((K + 31) // 32 * 16), scale_bytes(format, rows, K)
    codes_t, scales_t = (K * ((rows + 31) // 32 * 16), scale_bytes(format, K, rows)) if both else (0, 0)
    own_scale = fmt == 1 and not given
    buffer = torch.empty(codes + scales + codes_t + scales_t + (16 + 4 * WORKSPACE_FLOATS if own_scale else 0), dtype=torch.uint8, device=dev)
    at = buffer.data_ptr()
    at_s, at_ct = at + codes, at + codes + scales
    at_st, end = at_ct + codes_t, at_ct + codes_t + scales_t
    scale_ptr = end if own_scale else tensor_scale.data_ptr() if given else None
    _call("quantize", index, x.data_ptr(), typ, ldx, rows, K, fmt, scale_ptr, given, at, at_s,
          at_ct if both else None, at_st if both else None, end + 16 if own_scale else None)
    held = (buffer, tensor_scale)
    return (_held(format, fmt, rows, K, dev, held, at, at_s, scale_ptr),
            _held(format, fmt, K, rows, dev, held, at_ct, at_st, scale_ptr) if both else None)


def quantize_fp4(x: torch.Tensor, format: str = "nvfp4", tensor_scale: torch.Tensor | None = None) -> Fp4Tensor:
    """x [rows, K] (bf16, fp16 or fp32; rows may be a pitch apart) -> held form, blocks along the rows.
    ``tensor_scale`` (``nvfp4``): a positive fp32[1] to use in place of max|x| / 2688 - a calibrated one, for which x is
    read once instead of twice."""
    return _quantize(x, format, tensor_scale, False)[0]


def quantize_fp4_both(x: torch.Tensor, format: str = "nvfp4", tensor_scale: torch.Tensor | None = None):
    """(held form of x, held form of its transpose [K, rows] with blocks along x's columns), one tensor scale for both."""
    return _quantize(x, format, tensor_scale, True)


def dequantize_fp4(t: Fp4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that codes and scales stand for, [rows, K] of ``dtype``."""
    typ, index = _type(dtype), _device(t.device)
    out = torch.empty(t.rows, t.K, dtype=dtype, device=t.device)
    codes, scales, ts = t._args
    _call("dequantize", index, codes, scales, ts, t._fmt, t.rows, t.K, out.data_ptr(), typ)
    return out


def _product(A: Fp4Tensor, B: Fp4Tensor, out, out_dtype):
    dev = A.device
    index = _device(dev)
    if B._fmt != A._fmt or B.K != A.K:
        raise ValueError(f"operands of one format and depth are required: {A!r}, {B!r}")
    if B.device != dev:
        raise ValueError(f"operands on one device are required: {A!r}, {B!r}")
    if out is None:
        typ = _type(out_dtype)
        out = torch.empty(A.rows, B.rows, dtype=out_dtype, device=dev)
    else:
        typ = _type(out.dtype)
        if not (out.device == dev and out.is_contiguous() and out.shape == (A.rows, B.rows)):
            raise ValueError(f"out must be contiguous [{A.rows}, {B.rows}] on {dev}")
    return (*A._args, *B._args, out.data_ptr(), typ, A.rows, B.rows, A.K, A._fmt), out, index


def dense_gemm_fp4(A: Fp4Tensor, B: Fp4Tensor, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype = torch.bfloat16, tiling: int = 0, max_ctas: int = 0) -> torch.Tensor:
    """D[M,N] = A . B^T over the values of A [M,K] and B [N,K], any sizes; fp32 accumulation, rounded once to
    ``out_dtype`` (``out``'s type where it is given).  ``tiling``, ``max_ctas``: the tuner's knobs, 0 = automatic."""
    args, out, index = _product(A, B, out, out_dtype)
    _call("dense", index, *args, tiling, max_ctas)
    return out


def skinny_gemm_fp4(A: Fp4Tensor, B: Fp4Tensor, out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
                    flags: int = 0) -> torch.Tensor:
    """The same product for at most 32 rows of A (decode): a stream over B.  ``flags``: 0 or ``OVERLAP_PRIOR_KERNEL`` (the
    launch may request B while the preceding kernel of the stream drains; that kernel must not write B)."""
    args, out, index = _product(A, B, out, out_dtype)
    _call("skinny", index, *args, flags)
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
