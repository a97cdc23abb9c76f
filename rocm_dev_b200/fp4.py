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
MAX_EXTENT = 2 ** 31 - 1025                   # rows and columns of a tensor
_BYTE, _FLOAT = torch.uint8, torch.float32
# A quantiser's results of up to this many bytes are one allocation; larger ones have one for either direction, so that one
# can be dropped without the other, and one for the tensor scale.  An allocation costs 1.6 us of host time (8 x 4096 NVFP4
# 6.7 us a call in one, 8.4 in two; both directions 8.7 and 12.1), which shows until the device takes longer than the host:
# at this size 12 us for one direction, 15 for both.
ONE_ALLOCATION = 4 << 20

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
    rows, K)), ``tensor_scale`` fp32[1] (``nvfp4``) or None, all on ``device``.  ``torch.save`` and pickle store it; the parts
    by themselves are views of larger allocations (clone what a state dict is to hold)."""
    __slots__ = ("format", "rows", "K", "_fmt", "_parts", "_buffer", "_held")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, tensor_scale, format: str, rows: int, K: int):
        fmt = _format(format)
        if rows > MAX_EXTENT or K > MAX_EXTENT:
            raise ValueError(f"a held tensor has at most {MAX_EXTENT} rows and columns, got [{rows}, {K}]")
        if (codes.dtype is not _BYTE or codes.shape != (rows, (K + 31) // 32 * 16) or not codes.is_contiguous()
                or scales.dtype is not _BYTE or scales.numel() != (rows + 127) // 128 * ((K + 255) // 256) * (2048 if fmt else 1024)
                or not scales.is_contiguous()):
            raise ValueError(f"codes must be contiguous uint8 [{rows}, {row_bytes(K)}] and scales {scale_bytes(format, rows, K)} "
                             "contiguous bytes")
        if fmt == 0:
            if tensor_scale is not None:
                raise ValueError("mxfp4 has no tensor scale")
        elif tensor_scale is None or tensor_scale.dtype is not torch.float32 or tensor_scale.numel() != 1:
            raise ValueError("nvfp4 needs a tensor scale: one fp32")
        self.format, self.rows, self.K, self._fmt = format, rows, K, fmt
        self._parts, self._buffer, self._held = (codes, scales, tensor_scale), None, None
        self._now()

    def _now(self):
        """(addresses of codes, scales and tensor scale, device): of a caller's tensors as they are at the call."""
        held = self._held
        if held is not None:
            return held
        codes, scales, ts = self._parts
        dev = codes.device
        if scales.device != dev or ts is not None and ts.device != dev:
            raise ValueError("codes, scales and tensor scale must lie on one device")
        return (codes.data_ptr(), scales.data_ptr(), None if ts is None else ts.data_ptr()), dev

    def _views(self):
        # a quantiser's result is memory with the addresses in _held; its tensors are made when they are asked for, and from
        # then on they say where the data lies
        buffer, held = self._buffer, self._held
        if buffer is not None and held is not None:          # (another thread may be here too: _parts is there before these go)
            buf, ts = buffer
            (at_codes, at_scales, at_ts), base = held[0], buf.data_ptr()
            rb, sb = row_bytes(self.K), scale_bytes(self.format, self.rows, self.K)
            codes, scales = at_codes - base, at_scales - base
            if ts is None and at_ts is not None:
                # fp32 in the allocation of the bytes: a storage of its own over the same memory, since torch.save refuses
                # tensors of two types in one
                ts = torch.from_dlpack(torch.utils.dlpack.to_dlpack(buf[at_ts - base:at_ts - base + 4].view(_FLOAT)))
            self._parts = (buf[codes:codes + self.rows * rb].view(self.rows, rb), buf[scales:scales + sb], ts if ts is None else ts[:1])
            self._buffer = self._held = None
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

    @property
    def device(self) -> torch.device:
        return self._now()[1]

    def to(self, device) -> "Fp4Tensor":
        """The same tensor on another device (or on the host, to be stored)."""
        if torch.device(device) == self.device:
            return self
        move = lambda t: None if t is None else t.to(device)  # noqa: E731
        return Fp4Tensor(*map(move, self._views()), self.format, self.rows, self.K)

    def record_stream(self, stream) -> None:
        """``torch.Tensor.record_stream`` for every part: for a tensor made on another stream than the one it is used on."""
        for t in self._buffer or self._parts:
            if t is not None:
                t.record_stream(stream)

    def __copy__(self) -> "Fp4Tensor":
        return Fp4Tensor(*self._views(), self.format, self.rows, self.K)

    def __reduce__(self):
        # deep copies and files hold tensors, never an address: codes and scales once, and nothing else of their allocation
        codes, scales, ts = self._views()
        own = lambda t: t if t.untyped_storage().nbytes() == t.nbytes else t.clone()  # noqa: E731
        ts, n = ts if ts is None else own(ts), codes.numel()
        if codes.untyped_storage().data_ptr() == scales.untyped_storage().data_ptr() and scales.data_ptr() == codes.data_ptr() + n:
            return _whole, (own(codes.as_strided((n + scales.numel(),), (1,))), ts, self.format, self.rows, self.K)
        return Fp4Tensor, (codes, scales, ts, self.format, self.rows, self.K)

    def __repr__(self) -> str:
        return f"Fp4Tensor({self.format}, [{self.rows}, {self.K}], {self.device})"


def _whole(buf: torch.Tensor, tensor_scale, format: str, rows: int, K: int) -> Fp4Tensor:
    """What ``__reduce__`` took apart."""
    _format(format)
    if rows < 1 or K < 1 or buf.shape != (rows * row_bytes(K) + scale_bytes(format, rows, K),):
        raise ValueError(f"codes and scales of {format} [{rows}, {K}] in one flat tensor expected, got {tuple(buf.shape)}")
    n = rows * row_bytes(K)
    return Fp4Tensor(buf[:n].view(rows, -1), buf[n:], tensor_scale, format, rows, K)


torch.serialization.add_safe_globals([Fp4Tensor, _whole])        # torch.load reads them without weights_only=False


def _index(dev: torch.device) -> int:
    if dev.type != "cuda":
        raise ValueError(f"device tensors required, got one on {dev} (there is no CPU path)")
    return dev.index


def _bind():
    """The library's functions, through csrc/fastcall.c where it was built, else through ctypes."""
    global _entries
    L = lib()
    names = ("rdb_quantize_fp4", "rdb_dequantize_fp4", "rdb_dense_gemm_fp4_tuned", "rdb_skinny_gemm_fp4")
    try:
        from . import _fastcall as fast
        fast.bind(*(C.cast(getattr(L, n), C.c_void_p).value for n in names))
        _entries = (fast.quantize, fast.dequantize, fast.dense, fast.skinny)
    except ImportError:
        _entries = tuple(getattr(L, n) for n in names)
    return _entries


_entries = None
_QUANTIZE, _DEQUANTIZE, _DENSE, _SKINNY = range(4)


def _call(which: int, where: str, dev: int, *args) -> None:
    """Entry `which` with args and the current stream of device dev, dev being made the current device."""
    fn = (_entries or _bind())[which]
    if _current_device() == dev:
        code = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            code = fn(*args, _raw_stream(dev))
    if code:
        check(code, where)


def _result(form: str, fmt: int, rows: int, K: int, dev, buffer, scale, addresses) -> Fp4Tensor:
    t = Fp4Tensor.__new__(Fp4Tensor)
    t.format, t.rows, t.K, t._fmt = form, rows, K, fmt
    t._parts, t._buffer, t._held = None, (buffer, scale), (addresses, dev)
    return t


def _quantize(x: torch.Tensor, format: str, tensor_scale, both: bool):
    fmt, typ = _format(format), _type(x.dtype)
    if x.dim() != 2:
        raise ValueError(f"a 2-D tensor is required, got {tuple(x.shape)}")
    rows, K = x.shape
    if rows < 1 or K < 1:
        raise ValueError(f"an empty tensor cannot be quantised: {tuple(x.shape)}")
    if rows > MAX_EXTENT or K > MAX_EXTENT:
        raise ValueError(f"at most {MAX_EXTENT} rows and columns can be quantised: {tuple(x.shape)}")
    dev = x.device
    index = _index(dev)
    ldx, unit = x.stride()
    if unit != 1 and K > 1 or ldx < K and rows > 1:
        x = x.contiguous()                        # transposed or overlapping views
        ldx = K
    elif rows == 1:
        ldx = K
    per_word = 2048 if fmt else 1024              # scale bytes of 128 rows x 256 elements
    n = rows * ((K + 31) // 32 * 16)
    size = n + (rows + 127) // 128 * ((K + 255) // 256) * per_word
    m = size_t = 0
    if both:
        m = K * ((rows + 31) // 32 * 16)
        size_t = m + (K + 127) // 128 * ((rows + 255) // 256) * per_word
    given = at_ts = work = ts = None
    extra = 0                                     # the tensor scale and the scratch that the call alone uses
    if fmt == 0:
        if tensor_scale is not None:
            raise ValueError("mxfp4 has no tensor scale")
    elif tensor_scale is None:
        extra = 16 + 4 * WORKSPACE_FLOATS
    else:
        if not (tensor_scale.dtype is _FLOAT and tensor_scale.numel() == 1 and tensor_scale.device == dev):
            raise ValueError(f"the tensor scale must be one fp32 on {dev}")
        given = tensor_scale.data_ptr()
        extra = 16
    if size + size_t <= ONE_ALLOCATION:           # every part a multiple of 16 bytes
        buffer = buffer_t = torch.empty(size + size_t + extra, dtype=_BYTE, device=dev)
        at = buffer.data_ptr()
        at_t = at + size
        if extra:
            at_ts = at_t + size_t
    else:
        buffer = torch.empty(size, dtype=_BYTE, device=dev)
        at, at_t, buffer_t = buffer.data_ptr(), 0, None
        if both:
            buffer_t = torch.empty(size_t, dtype=_BYTE, device=dev)
            at_t = buffer_t.data_ptr()
        if extra:
            ts = torch.empty(extra // 4, dtype=_FLOAT, device=dev)
            at_ts = ts.data_ptr()
    if extra > 16:
        work = at_ts + 16
    if both:
        _call(_QUANTIZE, "rdb_quantize_fp4", index, x.data_ptr(), typ, ldx, rows, K, fmt, at_ts, given, at, at + n, at_t, at_t + m, work)
        return (_result(format, fmt, rows, K, dev, buffer, ts, (at, at + n, at_ts)),
                _result(format, fmt, K, rows, dev, buffer_t, ts, (at_t, at_t + m, at_ts)))
    _call(_QUANTIZE, "rdb_quantize_fp4", index, x.data_ptr(), typ, ldx, rows, K, fmt, at_ts, given, at, at + n, None, None, work)
    return _result(format, fmt, rows, K, dev, buffer, ts, (at, at + n, at_ts))


def quantize_fp4(x: torch.Tensor, format: str = "nvfp4", tensor_scale: torch.Tensor | None = None) -> Fp4Tensor:
    """x [rows, K] (bf16, fp16 or fp32; rows may be a pitch apart) -> held form, blocks along the rows.
    ``tensor_scale`` (``nvfp4``): a positive fp32[1] to use in place of max|x| * fp32(1 / 2688) - a calibrated one, for
    which x is read once instead of twice.  Its value is copied: changing it later leaves the result as it is.  An x without
    unit stride along its rows (a transposed view) is copied first; ``quantize_fp4_both`` makes both forms from one read."""
    return _quantize(x, format, tensor_scale, False)


def quantize_fp4_both(x: torch.Tensor, format: str = "nvfp4", tensor_scale: torch.Tensor | None = None):
    """(held form of x, held form of its transpose [K, rows] with blocks along x's columns), one tensor scale for both.
    Either frees its memory when it is dropped (a training step needs the first for the forward product alone), but where
    both together have no more than 4 MB, which are then kept by either."""
    return _quantize(x, format, tensor_scale, True)


def dequantize_fp4(t: Fp4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that codes and scales stand for, [rows, K] of ``dtype``."""
    typ = _type(dtype)
    (codes, scales, ts), dev = t._now()
    index = _index(dev)
    out = torch.empty(t.rows, t.K, dtype=dtype, device=dev)
    _call(_DEQUANTIZE, "rdb_dequantize_fp4", index, codes, scales, ts, t._fmt, t.rows, t.K, out.data_ptr(), typ)
    return out


def _product(A: Fp4Tensor, B: Fp4Tensor, out, out_dtype):
    a, dev = A._now()
    b, dev_b = B._now()
    index = _index(dev)
    if B._fmt != A._fmt or B.K != A.K or dev_b != dev:
        raise ValueError(f"operands of one format and depth, on one device, are required: {A!r}, {B!r}")
    if out is None:
        typ = _type(out_dtype)
        out = torch.empty(A.rows, B.rows, dtype=out_dtype, device=dev)
    else:
        typ = _type(out.dtype)
        if not (out.device == dev and out.is_contiguous() and out.shape == (A.rows, B.rows)):
            raise ValueError(f"out must be contiguous [{A.rows}, {B.rows}] on {dev}")
    return (*a, *b, out.data_ptr(), typ, A.rows, B.rows, A.K, A._fmt), out, index


def dense_gemm_fp4(A: Fp4Tensor, B: Fp4Tensor, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype = torch.bfloat16, tiling: int = 0, max_ctas: int = 0) -> torch.Tensor:
    """D[M,N] = A . B^T over the values of A [M,K] and B [N,K], any sizes; fp32 accumulation, rounded once to
    ``out_dtype`` (``out``'s type where it is given).  ``tiling``, ``max_ctas``: the tuner's knobs, 0 = automatic."""
    args, out, index = _product(A, B, out, out_dtype)
    _call(_DENSE, "rdb_dense_gemm_fp4", index, *args, tiling, max_ctas)
    return out


def skinny_gemm_fp4(A: Fp4Tensor, B: Fp4Tensor, out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
                    flags: int = 0) -> torch.Tensor:
    """The same product for at most 32 rows of A (decode): a stream over B.  ``flags``: 0 or ``OVERLAP_PRIOR_KERNEL`` (the
    launch may request B while the preceding kernel of the stream drains; that kernel must not write B, nor may the one
    before it where the preceding one is an fp8 call with this flag)."""
    args, out, index = _product(A, B, out, out_dtype)
    _call(_SKINNY, "rdb_skinny_gemm_fp4", index, *args, flags)
    return out


def pack_fp4_scales(scales: torch.Tensor, format: str, K: int) -> torch.Tensor:
    """Plain scale bytes [rows, ceil(K / block)] (as checkpoints hold them) -> the tiles that the kernels read.  ``nvfp4``: a
    scale's sign bit must be 0 (the products take scales as unsigned numbers)."""
    _format(format)
    b = BLOCK[format]
    if scales.dtype is not _BYTE or scales.dim() != 2 or K < 1 or scales.shape[1] != (K + b - 1) // b:
        raise ValueError(f"uint8 [rows, {(K + b - 1) // b}] expected, got {scales.dtype} {tuple(scales.shape)}")
    rows, blocks = scales.shape
    full = torch.zeros(((rows + 127) // 128 * 128, (K + 255) // 256 * (256 // b)), dtype=torch.uint8, device=scales.device)
    full[:rows, :blocks] = scales
    return full.reshape(full.shape[0] // 128, 4, 32, -1, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def unpack_fp4_scales(t: Fp4Tensor) -> torch.Tensor:
    """The plain scale bytes [rows, ceil(K / block)] of a held tensor."""
    b = BLOCK[t.format]
    full = t.scales.reshape((t.rows + 127) // 128, -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape((t.rows + 127) // 128 * 128, -1)
    return full[:t.rows, :(t.K + b - 1) // b].contiguous()
