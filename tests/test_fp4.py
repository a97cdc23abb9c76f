"""Microscaled 4-bit floating point: quantisers bit for bit, products against a 64-bit product of the held values.

Tolerance of a product, per element: half a step of the output type, 3 fp32 roundings for the tensor scales and their
products, and the summation-order noise 4 sqrt(K) 2^-24 sum|a b| of an fp32 accumulation (as in the fp8 tests): the
products themselves, and a block's scale times them, are exact."""
import copy
import ctypes
import pickle

import numpy as np
import pytest
import torch

FORMATS = ["mxfp4", "nvfp4"]
BLOCK = {"mxfp4": 32, "nvfp4": 16}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}    # half a step near zero
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


# ------------------------------------------------------------------ plain implementation (numpy)
def e2m1_codes(q):
    """Nearest code by distance, ties to the even one, signs kept."""
    a = np.minimum(np.abs(q.astype(np.float64)), 6.0)
    d = np.abs(a[..., None] - LEVELS[:8])
    best = d.min(axis=-1, keepdims=True)
    near = d == best
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(axis=-1), even.argmax(axis=-1), near.argmax(axis=-1))
    return (code | (np.signbit(q) << 3)).astype(np.uint8)


def e4m3_bytes(v):
    """Non-negative fp32 -> e4m3 bytes, nearest, ties to even, saturating."""
    all_ = torch.arange(0, 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).to(torch.float64).numpy()
    v = np.minimum(v.astype(np.float64), 448.0)
    hi = np.clip(np.searchsorted(all_, v), 1, 0x7E)
    lo = hi - 1
    dl, dh = v - all_[lo], all_[hi] - v
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)


def e4m3_values(b):
    return torch.from_numpy(np.ascontiguousarray(b)).view(torch.float8_e4m3fn).float().numpy()


def quantize(x, form, t=None):
    """fp32 [rows, K] -> (codes [rows, K32] one per byte, scale bytes [rows, blocks of the padded K], tensor scale)."""
    rows, K = x.shape
    b, kp = BLOCK[form], (K + 31) // 32 * 32
    v = np.zeros((rows, kp), np.float32)
    v[:, :K] = x
    v = v.reshape(rows, -1, b)
    bad = ~np.isfinite(v).all(axis=2)
    a = np.abs(v)
    amax = a.max(axis=2)
    with np.errstate(all="ignore"):
        if form == "mxfp4":
            e = np.where(amax > 0, np.frexp(np.where(bad, 1, amax))[1] - 3, -127).clip(-127, 127)
            q = np.ldexp(v.astype(np.float64), -e[..., None])
            s = (e + 127).astype(np.uint8)
            s[bad] = 0xFF
        else:
            if t is None:
                top = np.where(np.isfinite(v), a, 0).max()
                t = np.float32(1) if top == 0 else np.maximum(np.float32(top) * np.float32(1 / 2688), np.float32(2.0 ** -126))
            t = np.float32(t)
            s = e4m3_bytes(np.where(bad, 0, amax / (t * np.float32(6))))
            whole = e4m3_values(s) * t
            q = np.where(s[..., None] > 0, v / np.where(s > 0, whole, 1).astype(np.float32)[..., None], 0)
            s = np.where(bad, np.uint8(0x7F), s)
        q = np.where(bad[..., None], 0, q)          # codes of a block without values are not compared
    return e2m1_codes(q).reshape(rows, kp), s, t, bad


def values(codes, scales, form, K, t=None):
    """64-bit values of plain codes and scale bytes, without the tensor scale."""
    v = LEVELS[codes]
    s = np.where(scales == 0xFF, np.nan, 2.0 ** (scales.astype(np.float64) - 127)) if form == "mxfp4" else e4m3_values(scales).astype(np.float64)
    return (v.reshape(v.shape[0], -1, BLOCK[form]) * s[..., None]).reshape(v.shape[0], -1)[:, :K]


def plain(t):
    """A held tensor on the device -> (codes one per byte, plain scale bytes, tensor scale) by the documented layout."""
    import rocm_dev_b200 as R
    c = t.codes.cpu().numpy()
    codes = np.stack([c & 15, c >> 4], axis=-1).reshape(c.shape[0], -1)
    b = BLOCK[t.format]
    flat, across = t.scales.cpu().numpy(), (t.K + 255) // 256 * (256 // b) // 4
    r, k = np.arange(t.rows)[:, None], np.arange(across * 4)[None, :]
    s = flat[(r // 128 * across + k // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + k % 4]
    nb = codes.shape[1] // b
    assert not s[:, nb:].any(), "scales behind K must be zero"
    assert np.array_equal(R.unpack_fp4_scales(t).cpu().numpy(), s[:, :(t.K + b - 1) // b])
    return codes, s[:, :nb], None if t.tensor_scale is None else np.float32(t.tensor_scale.item())


def check_quantized(got, x, form, t=None):
    codes, scales, ts = plain(got)
    wc, ws, wt, bad = quantize(x, form, t)
    if form == "nvfp4":
        assert ts == wt
    assert np.array_equal(scales, ws)
    keep = np.repeat(~bad, BLOCK[form], axis=1)
    if form == "nvfp4":                              # a block whose scale is zero holds zeros of no sign
        zero = np.repeat(ws == 0, BLOCK[form], axis=1)
        assert not codes[zero & keep].any()
        keep &= ~zero
    assert np.array_equal(codes[keep], wc[keep])


def draw(rows, K, seed, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, K), generator=g) * std * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())
    return x.to(dtype)


def held(x, form, dev):
    import rocm_dev_b200 as R
    return R.quantize_fp4(x.to(dev), form)


def check_product(got, A, B):
    """`got` against the 64-bit product of what A and B hold."""
    (ca, sa, ta), (cb, sb, tb) = plain(A), plain(B)
    a, b = values(ca, sa, A.format, A.K), values(cb, sb, B.format, B.K)
    alpha = 1.0 if ta is None else float(ta) * float(tb)
    want, mag = a @ b.T * alpha, np.abs(a) @ np.abs(b).T * alpha
    tol = HALF[got.dtype] * np.abs(want) + TINY[got.dtype] + (4 * np.sqrt(A.K) + 3) * 2.0 ** -24 * mag
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.isfinite(err).all()
    assert (err <= tol).all(), f"{(err > tol).sum()} of {err.size} outside, worst {np.max(err / np.maximum(tol, 1e-300)):.3g} times the tolerance"


# ------------------------------------------------------------------ CPU
def test_sizes_of_the_held_form():
    import rocm_dev_b200 as R
    from rocm_dev_b200 import fp4
    L = R.lib()
    for rows, K in [(1, 1), (127, 31), (128, 256), (129, 257), (5, 4100), (2 ** 20, 14336)]:
        assert L.rdb_fp4_row_bytes(K) == fp4.row_bytes(K)
        for f in FORMATS:
            assert L.rdb_fp4_scale_bytes(fp4.FORMATS[f], rows, K) == fp4.scale_bytes(f, rows, K)
    assert L.rdb_fp4_row_bytes(0) == 0 and L.rdb_fp4_scale_bytes(1, 0, 5) == 0 and L.rdb_fp4_scale_bytes(2, 5, 5) == 0


def test_scale_tiles_round_trip():
    import rocm_dev_b200 as R
    for f, rows, K in [("mxfp4", 130, 700), ("nvfp4", 1, 16), ("nvfp4", 300, 1030)]:
        s = torch.randint(0, 255, (rows, -(-K // BLOCK[f])), dtype=torch.uint8)
        codes, ts = torch.zeros((rows, -(-K // 32) * 16), dtype=torch.uint8), None if f == "mxfp4" else torch.ones(1)
        t = R.Fp4Tensor(codes, R.pack_fp4_scales(s, f, K), ts, f, rows, K)
        assert torch.equal(R.unpack_fp4_scales(t), s)
        back = t.to("cpu")
        assert (back.format, back.rows, back.K) == (f, rows, K) and torch.equal(back.scales, t.scales)
        for again in (copy.deepcopy(t), pickle.loads(pickle.dumps(t))):
            assert torch.equal(again.codes, t.codes) and torch.equal(again.scales, t.scales) and repr(again) == repr(t)
            assert again._now()[0][0] == again.codes.data_ptr() != t.codes.data_ptr()


def _entries(through):
    """The library's functions through ctypes, or through csrc/fastcall.c, which has to hand on every argument in its place."""
    import types

    import rocm_dev_b200 as R
    L = R.lib()
    if through == "ctypes":
        return L
    fast = pytest.importorskip("rocm_dev_b200._fastcall")
    names = ("rdb_quantize_fp4", "rdb_dequantize_fp4", "rdb_dense_gemm_fp4_tuned", "rdb_skinny_gemm_fp4")
    fast.bind(*(ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in names))
    for f, n in ((fast.quantize, 14), (fast.dequantize, 9), (fast.dense, 15), (fast.skinny, 14)):
        for bad in ([0] * (n - 1), [0] * (n + 1), ["x"] + [0] * (n - 1), [0] * (n - 1) + [1.5]):
            with pytest.raises(TypeError):
                f(*bad)
    dense = lambda *a: fast.dense(*a[:12], 0, 0, a[12])  # noqa: E731
    return types.SimpleNamespace(rdb_quantize_fp4=fast.quantize, rdb_dequantize_fp4=fast.dequantize, rdb_dense_gemm_fp4_tuned=fast.dense,
                                 rdb_skinny_gemm_fp4=fast.skinny, rdb_dense_gemm_fp4=dense, rdb_skinny_gemm_fp4_tuned=L.rdb_skinny_gemm_fp4_tuned)


@pytest.mark.parametrize("through", ["ctypes", "c"])
def test_refusals_before_anything_is_launched(through):
    L = _entries(through)
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    Q = lambda **k: L.rdb_quantize_fp4(*{**dict(x=p, typ=0, ldx=64, rows=4, K=64, fmt=1, ts=p, given=None, codes=p, scales=p, ct=None, st=None, ws=p, stream=None), **k}.values())  # noqa: E731
    assert Q(rows=0) == 8 and Q(K=0) == 8 and Q(ldx=63) == 8
    assert Q(fmt=2) == 6 and Q(typ=3) == 6 and Q(x=None) == 6 and Q(codes=None) == 6 and Q(scales=None) == 6
    assert Q(ts=None) == 6 and Q(ws=None) == 6 and Q(ct=p) == 6 and Q(fmt=0) == 6 and Q(fmt=0, ts=None, given=p) == 6 and Q(given=p + 2) == 7
    assert Q(x=p + 1) == 7 and Q(codes=p + 8) == 7 and Q(scales=p + 4) == 7 and Q(ts=p + 2) == 7 and Q(typ=2, x=p + 2) == 7
    D = lambda **k: L.rdb_dequantize_fp4(*{**dict(codes=p, scales=p, ts=p, fmt=1, rows=4, K=64, out=p, typ=0, stream=None), **k}.values())  # noqa: E731
    assert D(rows=0) == 8 and D(fmt=-1) == 6 and D(typ=9) == 6 and D(ts=None) == 6 and D(out=None) == 6 and D(out=p + 1) == 7
    base = dict(A=p, sa=p, ta=p, B=p, sb=p, tb=p, D=p, typ=0, M=4, N=8, K=64, fmt=1)
    dense = lambda **k: L.rdb_dense_gemm_fp4(*{**base, **k}.values(), None)  # noqa: E731
    skinny = lambda flags=0, **k: L.rdb_skinny_gemm_fp4(*{**base, **k}.values(), flags, None)  # noqa: E731
    for call in (dense, skinny):
        assert call(M=0) == 8 and call(N=0) == 8 and call(K=-1) == 8
        assert call(fmt=5) == 6 and call(typ=-1) == 6 and call(A=None) == 6 and call(D=None) == 6 and call(ta=None) == 6
        assert call(fmt=0) == 6                                     # mxfp4 has no tensor scales
        assert call(A=p + 8) == 7 and call(sb=p + 1) == 7 and call(D=p + 1) == 7 and call(typ=2, D=p + 2) == 7
    assert skinny(M=33) == 1 and skinny(flags=2) == 6
    tiled = lambda **k: L.rdb_dense_gemm_fp4_tuned(*{**base, **dict(tiling=0, ctas=0), **k}.values(), None)  # noqa: E731
    assert tiled(tiling=3) == 6 and tiled(tiling=-1) == 6 and tiled(ctas=-1) == 6 and tiled(M=0) == 8
    tuned = lambda **k: L.rdb_skinny_gemm_fp4_tuned(*{**base, **dict(cols=0, split=0, st=0, flags=0), **k}.values(), None)  # noqa: E731
    assert tuned(cols=32) == 6 and tuned(cols=320) == 6 and tuned(split=9) == 6 and tuned(st=-1) == 6 and tuned(M=40) == 1


def test_refusals_of_the_python_face():
    import rocm_dev_b200 as R
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError):
        R.quantize_fp4(x, "fp4")
    with pytest.raises(TypeError):
        R.quantize_fp4(x.double())
    for bad in (x, x[0], torch.zeros(0, 4)):
        with pytest.raises(ValueError):
            R.quantize_fp4(bad)                                      # there is no CPU path
    codes, scales, one = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros(2048, dtype=torch.uint8), torch.ones(1)
    t = R.Fp4Tensor(codes, scales, one, "nvfp4", 4, 64)
    for bad in [(codes, scales, None, "nvfp4", 4, 64), (codes, scales, one, "mxfp4", 4, 64), (codes, scales[:-1], one, "nvfp4", 4, 64),
                (codes, scales, one.double(), "nvfp4", 4, 64), (codes, scales, one, "nvfp4", 4, 65), (codes, scales, one, "nvfp4", 5, 64),
                (codes.int(), scales, one, "nvfp4", 4, 64), (codes.t(), scales, one, "nvfp4", 32, 8), (codes, scales, one, "e2m1", 4, 64)]:
        with pytest.raises(ValueError):
            R.Fp4Tensor(*bad)
    for call in (lambda: R.dequantize_fp4(t), lambda: R.dense_gemm_fp4(t, t), lambda: R.skinny_gemm_fp4(t, t)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("through", ["ctypes", "c"])
def test_extents_beyond_32_bit_indices_are_refused(through):
    """Either entry hands on 32 bits of a size; beyond 2^31 - 1025 tile-rounded indices would overflow."""
    import rocm_dev_b200 as R
    L, most = _entries(through), 2 ** 31 - 1025
    buf = ctypes.create_string_buffer(512)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    for rows, K in ((most + 1, 1), (1, most + 1), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert L.rdb_quantize_fp4(p, 0, 2 ** 40, rows, K, 1, p, None, p, p, None, None, p, None) == 11
        assert L.rdb_dequantize_fp4(p, p, p, 1, rows, K, p, 0, None) == 11
        for M, N, k in ((rows, 1, K), (1, rows, K), (rows, K, 1)):
            assert L.rdb_dense_gemm_fp4(p, p, p, p, p, p, p, 0, M, N, k, 1, None) == 11
            assert L.rdb_skinny_gemm_fp4(p, p, p, p, p, p, p, 0, M, N, k, 1, 0, None) == 11
    for n in (most + 1, 2 ** 32 + 5):
        for shape in ((n, 1), (1, n)):
            wide = torch.zeros((1, 1), dtype=torch.bfloat16).expand(shape)
            for call in (R.quantize_fp4, R.quantize_fp4_both):
                with pytest.raises(ValueError, match=str(most)):
                    call(wide)
            codes = torch.empty((shape[0], (shape[1] + 31) // 32 * 16), dtype=torch.uint8, device="meta")
            scales = torch.empty((shape[0] + 127) // 128 * ((shape[1] + 255) // 256) * 1024, dtype=torch.uint8, device="meta")
            with pytest.raises(ValueError, match=str(most)):
                R.Fp4Tensor(codes, scales, None, "mxfp4", *shape)


# ------------------------------------------------------------------ quantisers
SHAPES = [(1, 1), (1, 16), (2, 17), (3, 31), (5, 32), (8, 4096), (130, 257), (33, 1000), (257, 129), (700, 48)]


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,K", SHAPES)
def test_quantize_bits(cuda_device, form, dtype, rows, K):
    import rocm_dev_b200 as R
    x = draw(rows, K, rows * 7 + K, dtype)
    r, c = R.quantize_fp4_both(x.to(cuda_device), form)
    one = R.quantize_fp4(x.to(cuda_device), form)
    v = x.float().numpy()
    check_quantized(r, v, form)
    check_quantized(one, v, form)
    check_quantized(c, np.ascontiguousarray(v.T), form)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("left,right", [(0, 8), (1, 2), (8, 24), (3, 0)])
def test_quantize_rows_a_pitch_apart(cuda_device, form, dtype, left, right):
    import rocm_dev_b200 as R
    wide = draw(70, left + 272 + right, 5, dtype).to(cuda_device)
    x = wide[:, left:left + 272]
    r, c = R.quantize_fp4_both(x, form)
    v = x.float().cpu().numpy()
    check_quantized(r, v, form)
    check_quantized(c, np.ascontiguousarray(v.T), form)
    check_quantized(R.quantize_fp4(x.t(), form), np.ascontiguousarray(v.T), form)      # a view with no unit stride
    check_quantized(R.quantize_fp4(x[:1].expand(5, -1), form), np.repeat(v[:1], 5, axis=0), form)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
def test_quantize_every_bf16_number(cuda_device, form):
    """All finite bf16 patterns: each value meets itself and larger ones in its block, subnormals and -0 included."""
    import rocm_dev_b200 as R
    bits = torch.arange(65536, dtype=torch.int32)
    bits = bits[(bits & 0x7F80) != 0x7F80].to(torch.int16)
    x = bits.view(torch.bfloat16).reshape(-1, 128)
    for v in (x, x.t().contiguous()):
        r, c = R.quantize_fp4_both(v.to(cuda_device), form)
        check_quantized(r, v.float().numpy(), form)
        check_quantized(c, v.float().numpy().T.copy(), form)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_quantize_borders(cuda_device, form, dtype):
    """Quotients on the borders between two codes and one step of the input type to either side of them."""
    import rocm_dev_b200 as R
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=dtype)
    around = torch.cat([ties, torch.nextafter(ties, ties * 0), torch.nextafter(ties, ties * 9)])
    x = torch.zeros(64, 32, dtype=dtype)
    x[:, :24] = around
    x[:, 24:] = 6.0
    x *= torch.linspace(1, 1.96875, 64, dtype=dtype)[:, None]
    x[1::2] *= -1
    t = None if form == "mxfp4" else torch.tensor([1.0])
    for k in (t,) if form == "mxfp4" else (t, torch.tensor([0.0123]), None):
        r, c = R.quantize_fp4_both(x.to(cuda_device), form, None if k is None else k.to(cuda_device))
        check_quantized(r, x.float().numpy(), form, None if k is None else k.item())
        check_quantized(c, x.float().numpy().T.copy(), form, None if k is None else k.item())


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
def test_quantize_what_is_no_number(cuda_device, form):
    """Infinities and NaNs take their own block's scale with them and leave the others - and the tensor scale - alone."""
    import rocm_dev_b200 as R
    x = draw(40, 320, 3, torch.float32)
    x[0, 0], x[3, 70], x[3, 319], x[39, 160] = float("inf"), float("nan"), float("-inf"), float("nan")
    x[5], x[6, :64] = 0.0, -0.0
    for v in (x, x.bfloat16()):
        r, c = R.quantize_fp4_both(v.to(cuda_device), form)
        check_quantized(r, v.float().numpy(), form)
        check_quantized(c, v.float().numpy().T.copy(), form)
        d = R.dequantize_fp4(r, torch.float32).cpu()
        b = BLOCK[form]
        assert torch.equal(torch.isnan(R.dequantize_fp4(c).cpu()).reshape(320, -1), torch.isnan(torch.from_numpy(values(*plain(c)[:2], form, 40))))
        bad = ~torch.isfinite(v.float()).reshape(40, -1, b).all(dim=2)
        assert torch.equal(torch.isnan(d).reshape(40, -1, b).all(dim=2), bad) and torch.equal(torch.isnan(d).reshape(40, -1, b).any(dim=2), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("fill", [0.0, 1e-45, 1e-38, 3.3e38])
def test_quantize_extreme_tensors(cuda_device, form, fill):
    import rocm_dev_b200 as R
    x = torch.full((20, 50), fill)
    x[:, ::3] = -fill / 3
    r, c = R.quantize_fp4_both(x.to(cuda_device), form)
    check_quantized(r, x.numpy(), form)
    check_quantized(c, x.numpy().T.copy(), form)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [1.1754944e-38, 1e-30, 3e-19, 1e-3, 7.0, 2e18, 1e30])
@pytest.mark.parametrize("size", [1e-36, 1e-20, 1.0, 1e19, 1e37])
def test_given_tensor_scales_far_from_the_values(cuda_device, dtype, t, size):
    """Saturated blocks where t is too small, zeros where it is too large."""
    import rocm_dev_b200 as R
    g = torch.Generator().manual_seed(4)
    x = (torch.randn((48, 160), generator=g) * size).to(dtype)
    x[3], x[:, 7] = 0.0, -0.0
    ts = torch.tensor([t], dtype=torch.float32)
    r, c = R.quantize_fp4_both(x.to(cuda_device), "nvfp4", ts.to(cuda_device))
    check_quantized(r, x.float().numpy(), "nvfp4", ts.item())
    check_quantized(c, x.float().numpy().T.copy(), "nvfp4", ts.item())


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 33), (130, 512), (65, 1001), (16, 4096)])
def test_dequantize(cuda_device, form, rows, K):
    import rocm_dev_b200 as R
    t = held(draw(rows, K, 9), form, cuda_device)
    codes, scales, ts = plain(t)
    want = values(codes, scales, form, K).astype(np.float32)         # exact in fp32
    want = want if ts is None else want * ts
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = R.dequantize_fp4(t, dtype).cpu()
        assert got.shape == (rows, K) and torch.equal(got, torch.from_numpy(want).to(dtype))


# ------------------------------------------------------------------ products
@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("where", ["skinny", "dense"])
def test_one_hot_operands_find_their_codes_and_scales(cuda_device, form, where):
    """A = rows of the identity (code 1.0, scale 1): D[m, n] is exactly the value B holds at (n, k(m))."""
    import rocm_dev_b200 as R
    M, N, K = (32 if where == "skinny" else 300), 330, 700
    B = held(draw(N, K, 2), form, cuda_device)
    k = (np.arange(M) * 37 + 5) % K
    eye = torch.zeros(M, K)
    eye[torch.arange(M), torch.from_numpy(k)] = 6.0                  # 6 -> code 6.0 (mxfp4: 4 * 1.5), a power-of-two scale
    one = torch.ones(1, device=cuda_device)
    A = R.quantize_fp4(eye.to(cuda_device), form, None if form == "mxfp4" else one)
    got = (R.skinny_gemm_fp4 if where == "skinny" else R.dense_gemm_fp4)(A, B, out_dtype=torch.float32)
    cb, sb, tb = plain(B)
    want = (6 * values(cb, sb, form, K)[:, k].T).astype(np.float32) * (np.float32(1) if tb is None else tb)
    torch.cuda.synchronize()
    assert R.lib().rdb_device_status() == 0
    assert np.array_equal(got.cpu().numpy(), want)


PRODUCTS = [(1, 1, 1), (1, 8, 16), (5, 64, 256), (8, 130, 257), (16, 256, 512), (17, 1001, 300), (32, 192, 2048), (3, 515, 4100),
            (31, 4096, 64), (1, 2048, 8192)]


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_skinny_product(cuda_device, form, dtype, M, N, K):
    import rocm_dev_b200 as R
    A, B = held(draw(M, K, 1, std=0.1), form, cuda_device), held(draw(N, K, 2, std=0.02), form, cuda_device)
    got = R.skinny_gemm_fp4(A, B, out_dtype=dtype)
    torch.cuda.synchronize()
    assert R.lib().rdb_device_status() == 0
    check_product(got, A, B)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("columns", [64, 128, 192, 256])
@pytest.mark.parametrize("split,stages", [(1, 0), (1, 1), (2, 2), (3, 0), (8, 0)])
def test_every_tile_width_and_split(cuda_device, form, columns, split, stages):
    import rocm_dev_b200 as R
    for M in (4, 29):
        A, B = held(draw(M, 2500, 3, std=0.1), form, cuda_device), held(draw(900, 2500, 4, std=0.02), form, cuda_device)
        out = torch.full((M, 900), float("nan"), device=cuda_device)
        args, _, dev = R.fp4._product(A, B, out, None)
        assert R.lib().rdb_skinny_gemm_fp4_tuned(*args, columns, split, stages, 0, torch.cuda.current_stream(dev).cuda_stream) == 0
        torch.cuda.synchronize()
        assert R.lib().rdb_device_status() == 0
        check_product(out, A, B)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("tiling,max_ctas", [(1, 0), (2, 0), (2, 2)])
@pytest.mark.parametrize("M,N,K,dtype", [(256, 256, 256, torch.float32), (256, 256, 2048, torch.bfloat16), (300, 700, 1100, torch.float32),
                                         (1, 1030, 64, torch.float16), (700, 513, 3000, torch.bfloat16), (1300, 1025, 520, torch.float32)])
def test_both_tilings(cuda_device, form, tiling, max_ctas, M, N, K, dtype):
    """max_ctas = 2: one pair walks every tile, through both accumulators."""
    import rocm_dev_b200 as R
    A, B = held(draw(M, K, 1, std=0.1), form, cuda_device), held(draw(N, K, 2, std=0.02), form, cuda_device)
    got = R.dense_gemm_fp4(A, B, out_dtype=dtype, tiling=tiling, max_ctas=max_ctas)
    torch.cuda.synchronize()
    assert R.lib().rdb_device_status() == 0
    check_product(got, A, B)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("M,N,K,dtype", [(1, 1, 1, torch.float32), (33, 100, 96, torch.bfloat16), (64, 64, 64, torch.float16),
                                         (65, 300, 1000, torch.float32), (128, 256, 256, torch.bfloat16), (129, 257, 513, torch.float32),
                                         (200, 4096, 128, torch.bfloat16), (333, 1001, 4100, torch.float32),
                                         (1024, 768, 2304, torch.bfloat16), (2, 5000, 320, torch.float16)])
def test_dense_product(cuda_device, form, M, N, K, dtype):
    import rocm_dev_b200 as R
    A, B = held(draw(M, K, 1, std=0.1), form, cuda_device), held(draw(N, K, 2, std=0.02), form, cuda_device)
    got = R.dense_gemm_fp4(A, B, out_dtype=dtype)
    torch.cuda.synchronize()
    assert R.lib().rdb_device_status() == 0
    check_product(got, A, B)


# ------------------------------------------------------------------ what else the documentation allows
def _product(A, B, **k):
    import rocm_dev_b200 as R
    return (R.skinny_gemm_fp4 if A.rows <= 32 and not k.get("tiling") else R.dense_gemm_fp4)(A, B, **k)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("M,tiling", [(5, 0), (200, 1), (300, 2)])
def test_what_is_no_number_stays_in_its_row_and_column(cuda_device, form, M, tiling):
    import rocm_dev_b200 as R
    N, K = 260, 700
    a, b = draw(M, K, 1), draw(N, K, 2)
    a[1, 3], b[7, 699] = float("nan"), float("inf")
    A, B = held(a, form, cuda_device), held(b, form, cuda_device)
    got = _product(A, B, out_dtype=torch.float32, **({"tiling": tiling} if tiling else {}))
    bad = torch.isnan(got).cpu()
    want = torch.zeros(M, N, dtype=torch.bool)
    want[1], want[:, 7] = True, True
    assert torch.equal(bad, want) and not torch.isinf(got).any()
    (ca, sa, ta), (cb, sb, tb) = plain(A), plain(B)
    x, y = values(ca, sa, form, K), values(cb, sb, form, K)
    alpha = 1.0 if ta is None else float(ta) * float(tb)
    fine = ~want.numpy()
    exact, mag = np.nan_to_num(x) @ np.nan_to_num(y).T * alpha, np.abs(np.nan_to_num(x)) @ np.abs(np.nan_to_num(y)).T * alpha
    err = np.abs(got.double().cpu().numpy() - exact)
    assert (err[fine] <= (2.0 ** -24 * np.abs(exact) + (4 * np.sqrt(K) + 3) * 2.0 ** -24 * mag)[fine]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("M,N,K,tiling", [(7, 70, 300, 0), (100, 130, 600, 1), (270, 300, 520, 2)])
@pytest.mark.parametrize("shift", [1, 2, 4, 5])
def test_outputs_at_any_address_and_nothing_around_them(cuda_device, form, M, N, K, tiling, shift):
    import rocm_dev_b200 as R
    A, B = held(draw(M, K, 1), form, cuda_device), held(draw(N, K, 2), form, cuda_device)
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.full((M * N + 64,), 7.0, dtype=dtype, device=cuda_device)
        out = wide[shift:shift + M * N].view(M, N)
        got = R.dense_gemm_fp4(A, B, out=out, tiling=tiling) if tiling else R.skinny_gemm_fp4(A, B, out=out)
        assert got.data_ptr() == out.data_ptr()
        check_product(got, A, B)
        assert (wide[:shift] == 7).all() and (wide[shift + M * N:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
def test_bytes_behind_the_last_row_do_not_matter(cuda_device, form):
    """Scale bytes of rows past the last (whole tiles of 128 rows are held) may be anything, a NaN included."""
    import rocm_dev_b200 as R
    for M, N, tiling in ((3, 200, 0), (130, 200, 1), (300, 200, 2)):
        A, B = held(draw(M, 520, 1), form, cuda_device), held(draw(N, 520, 2), form, cuda_device)
        want = R.dense_gemm_fp4(A, B, tiling=tiling) if tiling else R.skinny_gemm_fp4(A, B)
        for t in (A, B):
            tiles = t.scales.view(-(-t.rows // 128), -1, 32, 4, 4)
            r = torch.arange(t.rows, -(-t.rows // 128) * 128, device=cuda_device)
            tiles[r // 128, :, r % 32, r % 128 // 32, :] = 0xFF
        got = R.dense_gemm_fp4(A, B, tiling=tiling) if tiling else R.skinny_gemm_fp4(A, B)
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
def test_same_bits_call_after_call(cuda_device, form):
    import rocm_dev_b200 as R
    for M, N, K, tiling in ((8, 4096, 4096, 0), (96, 512, 4096, 1), (600, 1100, 2048, 2)):
        A, B = held(draw(M, K, 1), form, cuda_device), held(draw(N, K, 2), form, cuda_device)
        runs = [R.dense_gemm_fp4(A, B, tiling=tiling, out_dtype=torch.float32) if tiling else R.skinny_gemm_fp4(A, B, out_dtype=torch.float32)
                for _ in range(4)]
        assert all(torch.equal(r, runs[0]) for r in runs)


@pytest.mark.gpu
def test_launches_that_overlap_their_predecessor(cuda_device):
    """A chain of products in which each launch may request its weights while the one before it runs; the activations are
    quantised from the product before."""
    import rocm_dev_b200 as R
    W = [held(draw(1024, 1024, s, std=0.02), "nvfp4", cuda_device) for s in range(4)]
    x = draw(16, 1024, 9).to(cuda_device)

    def chain(flags):
        y = x
        for _ in range(3):
            for w in W:
                y = R.skinny_gemm_fp4(R.quantize_fp4(y), w, flags=flags)
        return y

    want = chain(0)
    for _ in range(5):
        assert torch.equal(chain(R.OVERLAP_PRIOR_KERNEL), want)
    assert R.lib().rdb_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
def test_two_captured_graphs_and_eager_calls_at_once(cuda_device, form):
    """Two graphs of quantiser and products replayed on two streams while eager calls run on a third: nothing is shared."""
    import rocm_dev_b200 as R
    streams = [torch.cuda.Stream(cuda_device) for _ in range(3)]
    W = held(draw(2048, 1024, 1, std=0.02), form, cuda_device)
    xs = [draw(m, 1024, 5 + m).to(cuda_device) for m in (16, 300, 64)]

    def step(x):
        r, c = R.quantize_fp4_both(x, form)
        y = _product(r, W)
        z = R.dense_gemm_fp4(c, c, out_dtype=torch.float32)
        return y, z, R.dequantize_fp4(r)

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, s in zip(xs[:2], streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step(x))
        graphs.append(g)
    for o in outs:
        for t in o:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = step(xs[2])
    torch.cuda.synchronize()
    assert R.lib().rdb_device_status() == 0
    for o, w in zip([*outs, eager], want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


@pytest.mark.gpu
def test_new_values_in_the_same_buffers_are_seen(cuda_device):
    """Nothing is kept by an address: operands overwritten in place, a replayed graph included."""
    import rocm_dev_b200 as R
    x = draw(8, 512, 1).to(cuda_device)
    W = held(draw(256, 512, 2), "nvfp4", cuda_device)
    s = torch.cuda.Stream(cuda_device)
    with torch.cuda.stream(s):
        R.skinny_gemm_fp4(R.quantize_fp4(x), W)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        y = R.skinny_gemm_fp4(R.quantize_fp4(x), W)
    for seed in (3, 4):
        x.copy_(draw(8, 512, seed))
        new = held(draw(256, 512, seed + 9), "nvfp4", cuda_device)
        W.codes.copy_(new.codes), W.scales.copy_(new.scales), W.tensor_scale.copy_(new.tensor_scale)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, R.skinny_gemm_fp4(R.quantize_fp4(x), new))


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
def test_copies_and_moved_tensors(cuda_device, form):
    """A held tensor that was copied, stored, or whose codes got other memory is read where it lies now."""
    import rocm_dev_b200 as R
    x = draw(33, 300, 1).to(cuda_device)
    t, c = R.quantize_fp4_both(x, form)
    for q, v in ((t, x), (c, x.t())):
        want = R.dequantize_fp4(q)
        for again in (copy.deepcopy(q), pickle.loads(pickle.dumps(q)), q.to("cpu").to(cuda_device)):
            assert torch.equal(R.dequantize_fp4(again), want) and again.codes.data_ptr() != q.codes.data_ptr()
    if form == "nvfp4":
        one = torch.ones(1, device=cuda_device)
        q = R.quantize_fp4(x, form, one)
        want = R.dequantize_fp4(q)
        one.fill_(2.0)                                       # a calibration that moves on
        assert torch.equal(R.dequantize_fp4(q), want) and q.tensor_scale.item() == 1.0
    del q, again
    own = copy.deepcopy(t)
    own.codes.data = torch.zeros_like(own.codes)             # what module.to() does to its parameters
    torch.cuda.empty_cache()
    assert not R.dequantize_fp4(own).any()


@pytest.mark.gpu
def test_another_device_than_the_current_one(cuda_device):
    import rocm_dev_b200 as R
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    other = torch.device("cuda:1")
    x = draw(8, 512, 1)
    a, b = held(x, "nvfp4", other), held(x, "nvfp4", cuda_device)
    assert torch.equal(R.skinny_gemm_fp4(a, a).cpu(), R.skinny_gemm_fp4(b, b).cpu()) and torch.cuda.current_device() == 0
    with pytest.raises(ValueError):
        R.skinny_gemm_fp4(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
def test_gradients_of_a_linear_layer(cuda_device, form):
    """y = x w^T with operands that the format holds exactly along either direction: the three products of a training step
    against the 64-bit formula, and the gradients against differences of the loss sum(dy * y), which is linear in each."""
    import rocm_dev_b200 as R
    M, N, K = 70, 130, 200
    g = torch.Generator().manual_seed(7)
    grid = torch.tensor([0.5, 1, 1.5, 2, 3, 4, 6, -0.5, -1, -1.5, -2, -3, -4, -6])
    pick = lambda *s: grid[torch.randint(0, 14, s, generator=g)]  # noqa: E731
    x, w, dy = pick(M, K), pick(N, K), pick(M, N)
    one = None if form == "mxfp4" else torch.ones(1, device=cuda_device)
    for t in (x, w, dy):
        t[::32], t[:, ::32] = 6.0, 6.0
        r, c = R.quantize_fp4_both(t.to(cuda_device), form, one)
        check_quantized(r, t.numpy(), form, 1.0)
        check_quantized(c, t.numpy().T.copy(), form, 1.0)
        # a 6 in every block, whose scale is 1 then, whichever way the blocks lie.  (Every 32nd alone leaves blocks of 16
        # without one: with 4 as the largest magnitude their scale is e4m3(4 / 6) = 0.6875, and 4 is held as 4.125.)
        t[::16], t[:, ::16] = 6.0, 6.0
    both = [R.quantize_fp4_both(t.to(cuda_device), form, one) for t in (x, w, dy)]
    for t, (r, c) in zip((x, w, dy), both):
        assert torch.equal(R.dequantize_fp4(r, torch.float32).cpu(), t) and torch.equal(R.dequantize_fp4(c, torch.float32).cpu(), t.t())
    (xr, xc), (wr, wc), (gr, gc) = both
    y, dx, dw = (R.dense_gemm_fp4(a, b, out_dtype=torch.float32).double().cpu() for a, b in ((xr, wr), (gr, wc), (gc, xc)))
    x, w, dy = x.double(), w.double(), dy.double()
    # multiples of 1/4 below 2^24 / 4: every sum is exact in fp32
    assert torch.equal(y, x @ w.t()) and torch.equal(dx, dy @ w) and torch.equal(dw, dy.t() @ x)
    loss = lambda x, w: (dy * (x @ w.t())).sum()  # noqa: E731
    for i, j in ((0, 0), (33, 199), (69, 64)):
        d = torch.zeros_like(x)
        d[i, j] = 0.25
        assert ((loss(x + d, w) - loss(x - d, w)) / 0.5 - dx[i, j]).abs() < 1e-6
    for i, j in ((0, 199), (129, 0), (64, 77)):
        d = torch.zeros_like(w)
        d[i, j] = 0.25
        assert ((loss(x, w + d) - loss(x, w - d)) / 0.5 - dw[i, j]).abs() < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("M", [4, 150])
def test_a_layer_run_as_it_is_served(cuda_device, form, M):
    """Quantise, project up, quantise, project down: each product against the 64-bit product of what its operands hold, and
    the whole against the same steps in plain form."""
    import rocm_dev_b200 as R
    x = draw(M, 512, 1)
    up, down = draw(1000, 512, 2, std=0.02), draw(512, 1000, 3, std=0.02)
    U, D = held(up, form, cuda_device), held(down, form, cuda_device)
    X = held(x, form, cuda_device)
    h = _product(X, U)
    check_product(h, X, U)
    H = R.quantize_fp4(h, form)
    check_quantized(H, h.float().cpu().numpy(), form)
    y = _product(H, D, out_dtype=torch.float32)
    check_product(y, H, D)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda_device):
    """x of 2.3e9 elements (4.6 GB of bf16, codes of 1.15 GB, values of 4.6 GB): the last rows as in a tensor of their own; and
    a product whose output passes 2^32 bytes."""
    import rocm_dev_b200 as R
    rows, K = 140_001, 16_384
    free, _ = torch.cuda.mem_get_info(cuda_device)
    if free < 40e9:
        pytest.skip("too little memory")
    x = torch.empty((rows, K), dtype=torch.bfloat16, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(0)
    for i in range(0, rows, 20_000):
        x[i:i + 20_000] = torch.randn((min(20_000, rows - i), K), generator=g, device=cuda_device).bfloat16()
    for form in FORMATS:
        r, c = R.quantize_fp4_both(x, form)
        one = R.quantize_fp4(x, form)
        tail = slice(rows - 97, rows)
        t = R.quantize_fp4(x[tail], form, r.tensor_scale)
        assert torch.equal(r.codes, one.codes) and torch.equal(r.codes[tail], t.codes)
        assert torch.equal(R.unpack_fp4_scales(r)[tail], R.unpack_fp4_scales(t))
        tc = R.quantize_fp4(x[:, -3:].t().contiguous(), form, r.tensor_scale)
        assert torch.equal(c.codes[-3:], tc.codes) and torch.equal(R.unpack_fp4_scales(c)[-3:], R.unpack_fp4_scales(tc))
        v = R.dequantize_fp4(one)
        assert torch.equal(v[tail], R.dequantize_fp4(t))
        del r, c, one, v
    del x
    M, N = 70_000, 32_776
    A, B = held(draw(M, 64, 1), "nvfp4", cuda_device), held(draw(N, 64, 2), "nvfp4", cuda_device)
    d = R.dense_gemm_fp4(A, B)
    rows = slice(M - 140, M)
    cut = R.Fp4Tensor(A.codes[rows].contiguous(), R.pack_fp4_scales(R.unpack_fp4_scales(A)[rows], "nvfp4", 64), A.tensor_scale, "nvfp4", 140, 64)
    assert torch.equal(d[rows], R.dense_gemm_fp4(cut, B))
    torch.cuda.synchronize()
    assert R.lib().rdb_device_status() == 0


@pytest.mark.gpu
def test_refusals_on_the_device(cuda_device):
    import rocm_dev_b200 as R
    A, B = held(draw(40, 64, 1), "nvfp4", cuda_device), held(draw(8, 64, 2), "nvfp4", cuda_device)
    with pytest.raises(R.RdbError) as e:
        R.skinny_gemm_fp4(A, B)
    assert e.value.code == 1
    for bad in (held(draw(8, 96, 2), "nvfp4", cuda_device), held(draw(8, 64, 2), "mxfp4", cuda_device), B.to("cpu")):
        with pytest.raises(ValueError):
            R.dense_gemm_fp4(A, bad)
    for out in (torch.empty(40, 9, device=cuda_device), torch.empty(8, 40, device=cuda_device).t(), torch.empty(40, 8)):
        with pytest.raises(ValueError):
            R.dense_gemm_fp4(A, B, out=out)
    with pytest.raises(TypeError):
        R.dense_gemm_fp4(A, B, out_dtype=torch.float64)
    x = draw(4, 64, 1).to(cuda_device)
    with pytest.raises(ValueError):
        R.quantize_fp4(x, "mxfp4", torch.ones(1, device=cuda_device))
    with pytest.raises(ValueError):
        R.quantize_fp4(x, "nvfp4", torch.ones(1))
    with pytest.raises(ValueError):
        R.quantize_fp4(x[:, :0])


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
def test_weights_written_two_launches_before_an_overlapping_one(cuda_device, form):
    """The flag allows B to be requested while the PRECEDING kernel runs: what the one before that wrote has to be there,
    however long it took."""
    import rocm_dev_b200 as R
    x = draw(4, 4096, 1).to(cuda_device)
    scale = None if form == "mxfp4" else torch.full((1,), 1e-3, device=cuda_device)
    ws = [(torch.randn((2048, 4096), generator=torch.Generator(cuda_device).manual_seed(s), device=cuda_device) * 0.1).bfloat16() for s in range(2)]
    want = [R.skinny_gemm_fp4(R.quantize_fp4(x, form), R.quantize_fp4(w, form, scale)) for w in ws]
    torch.cuda.synchronize()
    s, w = torch.cuda.Stream(cuda_device), ws[0].clone()
    g = torch.cuda.CUDAGraph()                              # launches follow one another faster than from Python
    with torch.cuda.graph(g, stream=s):
        W = R.quantize_fp4(w, form, scale)
        got = R.skinny_gemm_fp4(R.quantize_fp4(x, form), W, flags=R.OVERLAP_PRIOR_KERNEL)
    for i in range(20):
        w.copy_(ws[i % 2])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want[i % 2]), i


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("shift", [0, 16, 32, 48])
def test_quantized_buffers_at_any_16_bytes(cuda_device, form, shift):
    """Codes and scales that start on 16 bytes but no more, and nothing written around them."""
    import rocm_dev_b200 as R
    from rocm_dev_b200 import fp4
    rows, K = 96, 320
    x = draw(rows, K, 1).to(cuda_device)
    want_r, want_c = R.quantize_fp4_both(x, form)
    sizes = [rows * fp4.row_bytes(K), fp4.scale_bytes(form, rows, K), K * fp4.row_bytes(rows), fp4.scale_bytes(form, K, rows)]
    for both in (False, True):
        bufs = [torch.full((n + 160,), 0xAB, dtype=torch.uint8, device=cuda_device) for n in sizes]
        at = [b.data_ptr() + 16 + shift for b in bufs]
        ts, ws = torch.empty(1, device=cuda_device), torch.empty(fp4.WORKSPACE_FLOATS, device=cuda_device)
        code = R.lib().rdb_quantize_fp4(x.data_ptr(), 0, K, rows, K, fp4.FORMATS[form], None if form == "mxfp4" else ts.data_ptr(), None, at[0], at[1], at[2] if both else None,
                                        at[3] if both else None, ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert code == 0
        parts = [b[16 + shift:16 + shift + n] for b, n in zip(bufs, sizes)]
        if form == "nvfp4":
            assert torch.equal(ts, want_r.tensor_scale)
        for i, t in enumerate((want_r, want_c) if both else (want_r,)):
            assert torch.equal(parts[2 * i].view(t.rows, -1), t.codes)
            got = R.Fp4Tensor(parts[2 * i].clone().view(t.rows, -1), parts[2 * i + 1].clone(), None if form == "mxfp4" else ts, form, t.rows, t.K)
            assert torch.equal(R.unpack_fp4_scales(got), R.unpack_fp4_scales(t))
        for b, n, used in zip(bufs, sizes, (1, 1, both, both)):
            assert (b[:16 + shift] == 0xAB).all() and (b[16 + shift + n:] == 0xAB).all()
            assert used or (b == 0xAB).all()


@pytest.mark.gpu
@pytest.mark.parametrize("follow", ["skinny", "skinny, overlapping", "dense", "fp8 skinny", "fp8 list", "sparse"])
def test_the_kernel_before_may_run_longer_than_a_wait_may_last(cuda_device, follow):
    """Launches start while the one before them runs; their waits for data are limited (to 1 ms here, the kernel before runs
    about 15 ms on two SMs) and may begin only when that one has finished."""
    import rocm_dev_b200 as R
    from rocm_dev_b200 import quant
    A, B = held(draw(8192, 8192, 1), "mxfp4", cuda_device), held(draw(8192, 8192, 2), "mxfp4", cuda_device)
    D = torch.empty(8192, 8192, dtype=torch.bfloat16, device=cuda_device)
    a, w = held(draw(16, 2048, 3), "nvfp4", cuda_device), held(draw(1024, 2048, 4), "nvfp4", cuda_device)
    qa, qw, sa, sw = (t.to(cuda_device) for t in quant.synthetic_gemm_operands(16, 1024, 2048, seed=5))
    vals, meta = (t.to(cuda_device) for t in R.pack_2of4(R.prune_2of4(qw.cpu())))
    out = torch.empty(16, 1024, dtype=torch.bfloat16, device=cuda_device)

    def call():
        out.zero_()
        if long:
            R.dense_gemm_fp4(A, B, out=D, tiling=2, max_ctas=2)
        if follow == "dense":
            R.dense_gemm_fp4(a, w, out=out, tiling=1)
        elif follow == "fp8 skinny":
            assert R.skinny_gemm_fp8_tuned(qa, qw, sa, sw, out, flags=R.OVERLAP_PRIOR_KERNEL) == 0
        elif follow == "fp8 list":
            assert R.skinny_gemm_fp8_grouped([(qa, qw, sa, sw, out)], flags=R.OVERLAP_PRIOR_KERNEL) == 0
        elif follow == "sparse":
            R.sparse_gemm_fp8(qa, vals, meta, sa, sw, out=out, flags=R.OVERLAP_PRIOR_KERNEL)
        else:
            R.skinny_gemm_fp4(a, w, out=out, flags=R.OVERLAP_PRIOR_KERNEL if "overlapping" in follow else 0)
        torch.cuda.synchronize()
        return out.clone()

    long = False
    want = call()
    assert R.lib().rdb_device_status() == 0
    long = True
    assert R.lib().rdb_set_wait_budget_ns(1_000_000) == 0
    try:
        got = call()
        status = R.lib().rdb_device_status()
    finally:
        assert R.lib().rdb_set_wait_budget_ns(1_000_000_000) == 0
    assert status == 0 and torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,tiling", [(5, 130, 4096, 0), (100, 200, 520, 1), (300, 270, 1000, 2)])
@pytest.mark.parametrize("a,b", [(1e-20, 1e-20), (1e-16, 1e-16), (1e-30, 1e-7), (1e-35, 1e35), (1e-3, 1e-33), (1e37, 1e-6), (1e16, 1e16)])
def test_tensor_scales_whose_product_leaves_fp32(cuda_device, M, N, K, tiling, a, b):
    """The result counts, not ta * tb: operands of 1e-20 have scales of 4e-24 and a product of 1e-37 at K = 4096."""
    import rocm_dev_b200 as R
    x, y = (torch.randn((r, K), generator=torch.Generator().manual_seed(r)).abs() * s for r, s in ((M, a), (N, b)))
    x[1] = 0.0
    A, B = held(x, "nvfp4", cuda_device), held(y, "nvfp4", cuda_device)
    for dtype in (torch.float32, torch.bfloat16):
        got = _product(A, B, out_dtype=dtype, **({"tiling": tiling} if tiling else {}))
        check_product(got, A, B)
        assert not got[1].any() and got[0].all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,tiling", [(5, 0), (300, 2)])
def test_tensor_scales_whose_product_is_infinite(cuda_device, M, tiling):
    """Zeros stay zeros where every other value is beyond fp32, or vanishes."""
    x, y = (torch.randn((r, 256), generator=torch.Generator().manual_seed(r)).abs() for r in (M, 70))
    x[1] = 0.0
    for a, b, want in ((1e30, 1e30, float("inf")), (1e-35, 1e-35, 0.0)):
        A, B = held(x * a, "nvfp4", cuda_device), held(y * b, "nvfp4", cuda_device)
        got = _product(A, B, out_dtype=torch.float32, **({"tiling": tiling} if tiling else {}))
        assert not got[1].any() and (got[0] == want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("six", [False, True])
def test_divisors_with_every_bit_set(cuda_device, dtype, six):
    """Powers of two over a divisor 2^k (2 - 2^-23): the quotient rounds to just above a power of two, which is a border
    between two codes (0.25) and between two scales (2^-10), and one unit in the divisor's reciprocal decides.  six: 6 t is
    that divisor, not t."""
    import rocm_dev_b200 as R
    t = np.float32(1) - np.float32(2.0 ** -24)
    if six:
        near = np.float32(4 / 3) + np.arange(-64, 64, dtype=np.float32) * np.float32(2.0 ** -23)
        t = near[((near * np.float32(6)).view(np.uint32) & 0x7FFFFF) == 0x7FFFFF][0]
    x = torch.zeros(64, 160)
    for i in range(14):                                              # block scales 2^-6 .. 2^7 where t is the divisor
        x[i, ::16], x[i, 1::4], x[i, 2::4] = 6.0 * 2.0 ** (i - 6), 0.25 * 2.0 ** (i - 6), -0.25 * 2.0 ** (i - 6)
    for i in range(14, 40):                                          # largest magnitudes 2^-16 .. 2^9
        x[i, ::16], x[i, 3::16] = 2.0 ** (i - 30), 2.0 ** (i - 32)
    x = x.to(dtype)
    ts = torch.from_numpy(np.array([t])).to(cuda_device)
    for v in (x, x.t().contiguous()):
        for aligned in (True, False):
            wide = torch.zeros(v.shape[0], v.shape[1] + 3, dtype=dtype)
            wide[:, 1:-2] = v
            y = v.to(cuda_device) if aligned else wide.to(cuda_device)[:, 1:-2]
            r, c = R.quantize_fp4_both(y, "nvfp4", ts)
            for got, want in ((r, v), (R.quantize_fp4(y, "nvfp4", ts), v), (c, v.t())):
                check_quantized(got, np.ascontiguousarray(want.float().numpy()), "nvfp4", t)


def test_16_bit_maxima_make_no_divisor_with_every_bit_set():
    """Tensor scales computed from 16-bit maxima keep the quantiser's short quotient: none of their products with a block
    scale's significand (1 to 15/8; 12/8 stands for 6 t too) has all 23 bits set, whatever the exponents."""
    top = np.arange(1024, 2048, dtype=np.float32)                    # significands of fp16, those of bf16 among them
    t = top * np.float32(1 / 2688)
    for k in range(8, 16):
        assert not ((t * np.float32(k)).view(np.uint32) & 0x7FFFFF == 0x7FFFFF).any()


def _rounded(v):
    """A Fraction to fp32 (no range limits), ties to even."""
    from fractions import Fraction as F
    if v == 0:
        return v
    a = abs(v)
    e = a.numerator.bit_length() - a.denominator.bit_length()
    step = F(2) ** (e - (F(2) ** e > a) - 23)
    n, rest = divmod(a, step)
    n += rest * 2 > step or rest * 2 == step and n % 2
    return n * step * (1 if v > 0 else -1)


def test_the_short_quotient_decides_as_the_division_does():
    """Quotients of 11-bit significands next to every border of e2m1, and of e4m3's three lowest binades: q = RN(a inv), then
    RN(q + inv RN(a - q d)).  With the rounded reciprocal the side of the border is the division's, always; with one a unit
    off as well, but for divisors whose 23 bits are all set."""
    from fractions import Fraction as F
    tie = {F(1, 4): -1, F(3, 4): 1, F(5, 4): -1, F(7, 4): 1, F(5, 2): -1, F(7, 2): 1, F(5): -1}       # the even code's side
    tie |= {F(2 * i + 1, 1024): 1 if i % 2 else -1 for i in range(16)}
    side = lambda v, b: (v > b) - (v < b) or tie[b]  # noqa: E731
    exceptions = set()
    for b in tie:
        for X in range(1024, 2048):
            d0 = X / b                                               # brought into [1, 2): divisors next to X / border
            k = d0.numerator.bit_length() - d0.denominator.bit_length()
            k -= F(2) ** k > d0
            a = F(X) / F(2) ** k
            n0 = int(a / b * 2 ** 23)
            for n in (n0 - 1, n0, n0 + 1):
                d = F(n, 2 ** 23) if n >= 2 ** 23 else F(2 * n + 1, 2 ** 24)      # below 1: steps half as wide
                want = side(_rounded(a / d), b)
                inv = np.float32(float(_rounded(1 / d)))
                for off in (inv, np.nextafter(inv, np.float32(0)), np.nextafter(inv, np.float32(9))):
                    r = F(float(off))
                    q = _rounded(a * r)
                    if side(_rounded(q + r * _rounded(a - q * d)), b) != want:
                        assert off != inv
                        exceptions.add(d)
    assert exceptions and all(d.numerator == 2 ** 24 - 1 for d in exceptions)


@pytest.mark.gpu
def test_parts_that_got_other_memory_are_read_where_they_lie(cuda_device):
    """Of a quantiser's own result too, once its tensors have been asked for."""
    import rocm_dev_b200 as R
    x = draw(33, 300, 1).to(cuda_device)
    t, other = R.quantize_fp4(x), R.quantize_fp4(draw(33, 300, 2).to(cuda_device))
    shallow = copy.copy(t)
    assert torch.equal(R.dequantize_fp4(shallow), R.dequantize_fp4(t)) and shallow.codes.data_ptr() == t.codes.data_ptr()
    t.codes.data, t.scales.data, t.tensor_scale.data = other.codes.clone(), other.scales.clone(), other.tensor_scale.clone()
    for q in (t, copy.deepcopy(t), pickle.loads(pickle.dumps(t))):
        assert torch.equal(R.dequantize_fp4(q), R.dequantize_fp4(other))
    s = torch.cuda.Stream(cuda_device)
    with torch.cuda.stream(s):
        q = R.quantize_fp4(x)
    q.record_stream(torch.cuda.current_stream())
    t.record_stream(s)


def _stored(x):
    import io
    f = io.BytesIO()
    torch.save(x, f)
    return f.getvalue()


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("asked", [False, True])
@pytest.mark.parametrize("rows,K", [(256, 512), (2048, 4096)])
def test_files_hold_a_quantised_tensor_and_nothing_else(cuda_device, form, asked, rows, K):
    """torch.save, pickle and a state dict of the parts, for results of either quantiser, whether or not their tensors have
    been asked for: no more bytes than codes, scales and tensor scale (and a kilobyte or so of names)."""
    import io

    import rocm_dev_b200 as R
    x = draw(rows, K, 1).to(cuda_device)
    for t in (R.quantize_fp4(x, form), *R.quantize_fp4_both(x, form), R.quantize_fp4(x, form, None if form == "mxfp4" else torch.ones(1, device=cuda_device))):
        want = R.dequantize_fp4(t)
        if asked:
            t.codes, t.scales, t.tensor_scale
        most = t.rows * R.fp4.row_bytes(t.K) + R.fp4.scale_bytes(form, t.rows, t.K) + 4096
        data = _stored(t)
        assert len(data) < most and len(pickle.dumps(t)) < most
        for again in (torch.load(io.BytesIO(data)), torch.load(io.BytesIO(data), map_location="cpu").to(cuda_device), pickle.loads(pickle.dumps(t))):
            assert repr(again) == repr(t) and torch.equal(R.dequantize_fp4(again), want)
            assert len(_stored(again)) < most
        parts = {k: v for k, v in (("codes", t.codes), ("scales", t.scales), ("tensor_scale", t.tensor_scale)) if v is not None}
        back = torch.load(io.BytesIO(_stored(parts)))
        own = R.Fp4Tensor(back["codes"], back["scales"], back.get("tensor_scale"), form, t.rows, t.K)
        assert torch.equal(R.dequantize_fp4(own), want)


def test_a_stored_tensor_of_the_wrong_size_is_refused():
    from rocm_dev_b200 import fp4
    n = 4 * fp4.row_bytes(64) + fp4.scale_bytes("nvfp4", 4, 64)
    assert fp4._whole(torch.zeros(n, dtype=torch.uint8), torch.ones(1), "nvfp4", 4, 64).rows == 4
    for bad in ((torch.zeros(n - 1, dtype=torch.uint8), torch.ones(1), "nvfp4", 4, 64), (torch.zeros(n), torch.ones(1), "nvfp4", 4, 64),
                (torch.zeros((1, n), dtype=torch.uint8), torch.ones(1), "nvfp4", 4, 64), (torch.zeros(8, dtype=torch.uint8), torch.ones(1), "nvfp4", 4, 64),
                (torch.zeros(n, dtype=torch.uint8), None, "nvfp4", 4, 64)):
        with pytest.raises(ValueError):
            fp4._whole(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
def test_either_direction_can_be_dropped(cuda_device, form):
    import rocm_dev_b200 as R
    x = draw(1024, 4096, 1).to(cuda_device)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(cuda_device)
    r, c = R.quantize_fp4_both(x, form)
    both = torch.cuda.memory_allocated(cuda_device) - before
    size = r.codes.numel() + r.scales.numel()
    want = R.dequantize_fp4(c).clone()
    del r
    left = torch.cuda.memory_allocated(cuda_device) - before - want.numel() * 2
    assert both - left >= size and left <= size + 16384
    assert torch.equal(R.dequantize_fp4(c), want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,form", [(3, 65535 * 128 + 5, "mxfp4"), (3, 65535 * 128 + 5, "nvfp4"), (40, 65535 * 256 + 9, "mxfp4")])
def test_more_columns_than_one_grid_has_tiles(cuda_device, M, N, form):
    """The same as the two halves of B by themselves.  Positive operands: every sum of 32 products is off by no more than
    (4 sqrt(32) + 3) 2^-24 of itself on either side."""
    import rocm_dev_b200 as R
    g = torch.Generator(device=cuda_device).manual_seed(0)
    A, B = (R.quantize_fp4(torch.randn((r, 32), generator=g, device=cuda_device, dtype=torch.bfloat16).abs(), form) for r in (M, N))
    half = N // 256 * 128                                            # whole scale tiles: both halves are views
    per_tile = R.fp4.scale_bytes(form, 128, 32)
    cuts = [R.Fp4Tensor(B.codes[a:b], B.scales[a // 128 * per_tile:-(-b // 128) * per_tile], B.tensor_scale, form, b - a, 32) for a, b in ((0, half), (half, N))]
    calls = [R.dense_gemm_fp4] + ([R.skinny_gemm_fp4] if M <= 32 else [])
    for f in calls:
        got = f(A, B, out_dtype=torch.float32)
        for cut, part in zip(cuts, (got[:, :half], got[:, half:])):
            want = f(A, cut, out_dtype=torch.float32)
            assert ((part - want).abs() <= 2 * (4 * 32 ** 0.5 + 4) * 2.0 ** -24 * want).all()
        del got, part, want
    torch.cuda.synchronize()
    assert R.lib().rdb_device_status() == 0
    with pytest.raises(R.RdbError) as e:
        R.dense_gemm_fp4(A, B, tiling=1)
    assert e.value.code == 11


def test_plain_scales_of_the_wrong_form_are_refused():
    import rocm_dev_b200 as R
    s = torch.zeros((5, 4), dtype=torch.uint8)
    assert R.pack_fp4_scales(s, "nvfp4", 64).numel() == R.fp4.scale_bytes("nvfp4", 5, 64)
    for bad in ((s, "fp4", 64), (s, "nvfp4", 65), (s, "mxfp4", 64), (s.int(), "nvfp4", 64), (s[0], "nvfp4", 64), (s, "nvfp4", 0)):
        with pytest.raises(ValueError):
            R.pack_fp4_scales(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMATS)
def test_k_is_cut_no_further_than_the_clusters_are_resident(cuda_device, form):
    """Over row counts, tile counts and depths: all clusters of a plan that cuts K fit on the device at once, counted by the
    shared memory that the plan asks for, and no SM gets more CTAs than its 512 columns serve."""
    import rocm_dev_b200 as R
    L = R.lib()
    if torch.cuda.get_device_properties(cuda_device).multi_processor_count != 148:
        pytest.skip("the counts are those of 148 SMs")
    one, two = [0, 148, 74, 45, 33, 26, 22, 15, 15], [0, 296, 148, 93, 71, 56, 45, 37, 33]
    out = [ctypes.c_int() for _ in range(4)]

    def plan(M, N, K):
        assert L.rdb_fp4_split_plan(M, N, K, R.fp4.FORMATS[form], *map(ctypes.byref, out)) == 0
        return [o.value for o in out]

    cut = 0
    for M in (1, 16, 17, 32, 33, 64, 128, 200, 256):
        for K in (512, 1024, 2048, 4096, 8192, 14336, 100_000):
            for tiles in (*range(1, 100), 120, 148, 149, 300):
                N = 128 * tiles
                columns, S, stages, smem = plan(M, N, K)
                per_stage = 4 * (4 if form == "nvfp4" else 2) * (1 + -(-columns // 128))
                per_sm = 233472 // (smem + 1184)
                assert per_sm * max(32, 2 ** (columns + stages * per_stage - 1).bit_length()) <= 512
                if S > 1:
                    cut += 1
                    assert -(-N // columns) * -(-M // 128) <= (one if per_sm == 1 or M > 32 else two)[S], (M, N, K, S)
                    assert S <= -(-K // 256)
    assert cut > 1000
    assert plan(32, 8192, 8192)[1] == (2 if form == "nvfp4" else 4)          # one CTA to an SM, two
    for bad in ((0, 1, 1, 1), (1, 1, 1, 2), (1, 2 ** 31 - 1, 1, 1)):
        assert L.rdb_fp4_split_plan(*bad, *map(ctypes.byref, out)) in (6, 8, 11)
    assert L.rdb_fp4_split_plan(1, 1, 1, 1, None, None, None, None) == 6
