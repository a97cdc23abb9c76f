"""Microscaled 4-bit floating point: the quantisers and the products, as cases that can be timed and compared.

Two formats.  Elements are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), rounded to the nearest, ties to the even
code, beyond 6 to 6.
  mxfp4   blocks of 32 along K share a power of two, 2^(floor(log2(largest magnitude)) - 2), held as its exponent + 127;
  nvfp4   blocks of 16 along K share an e4m3 scale, and the tensor one fp32 scale t = largest magnitude / 2688 (448 x 6;
          1 for an all-zero tensor): block scale s = e4m3(block's largest magnitude / (6 t)), element = e2m1(x / (t s)),
          6 t, t s and the two quotients rounded to fp32.
Codes are [rows, ceil(K / 32) * 16] bytes, two to a byte, the even index in the low half, zeros behind K.  Scales lie in
tiles of 128 rows x 4 blocks, 512 bytes each: row r, block b of a tile at (r % 32) * 16 + (r / 32) * 4 + b; tiles run along
K first, and K is filled up to a multiple of 256 with zero scales.
The products are D = A . B^T over the values that codes and scales stand for, accumulated in fp32, times both tensor
scales, rounded once.
"""
import math

import torch

own = False

BLOCK = {"mxfp4": 32, "nvfp4": 16}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # a decode step's activations before a projection: the smallest call, all latency
        {"name": "quantize-decode", "op": "quantize", "format": "nvfp4", "rows": 8, "K": 4096, "pad": 0, "x": "bf16", "out": "bf16"},
        # a long prompt's activations
        {"name": "quantize-prefill", "op": "quantize", "format": "mxfp4", "rows": 8192, "K": 8192, "pad": 0, "x": "bf16", "out": "bf16"},
        # a slice of a wider buffer, with odd sizes and rows that start off 16 bytes
        {"name": "quantize-strided", "op": "quantize", "format": "nvfp4", "rows": 1021, "K": 4099, "pad": 5, "x": "fp16", "out": "fp32"},
        # activations of a training step, which its forward product reads by rows and its weight gradient by columns
        {"name": "both-activations", "op": "both", "format": "nvfp4", "rows": 4096, "K": 14336, "pad": 0, "x": "bf16", "out": "bf16"},
        # a batch of odd length, kept in fp32
        {"name": "both-ragged", "op": "both", "format": "mxfp4", "rows": 777, "K": 2500, "pad": 3, "x": "fp32", "out": "fp32"},
        # a square product, all tensor cores
        {"name": "dense-square", "op": "dense", "format": "nvfp4", "M": 8192, "N": 8192, "K": 8192, "out": "bf16"},
        # a prompt's tokens through the widest projection
        {"name": "dense-prefill", "op": "dense", "format": "mxfp4", "M": 2048, "N": 28672, "K": 4096, "out": "bf16"},
        # a short prompt with no size a multiple of anything
        {"name": "dense-ragged", "op": "dense", "format": "nvfp4", "M": 333, "N": 1001, "K": 4100, "out": "fp32"},
        # one linear layer's training step: both directions of x, w and dy, then the output and the two gradients
        {"name": "train-linear", "op": "train", "format": "nvfp4", "M": 2048, "N": 6144, "K": 4096, "out": "bf16"},
        # one token through the smallest projection
        {"name": "skinny-token", "op": "skinny", "format": "nvfp4", "M": 1, "N": 4096, "K": 4096, "out": "bf16"},
        # a batch of tokens through the widest projection: the weights' stream
        {"name": "skinny-wide", "op": "skinny", "format": "nvfp4", "M": 16, "N": 28672, "K": 4096, "out": "bf16"},
        # the largest decode batch through the deepest projection
        {"name": "skinny-deep", "op": "skinny", "format": "mxfp4", "M": 32, "N": 4096, "K": 14336, "out": "fp16"},
    ]


def _size(rng, low, high):
    """Spread over the logarithm; every third one a multiple of 128, so that even and odd sizes both come."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(128, n // 128 * 128) if rng.random() < 1 / 3 and high >= 128 else max(low, min(high, n))


def draw(rng):
    c = {"op": rng.choice(["quantize", "both", "dense", "dense", "train", "skinny", "skinny"]), "format": rng.choice(["mxfp4", "nvfp4"])}
    if c["op"] in ("quantize", "both"):
        c["rows"] = _size(rng, 1, 16384)
        c["K"] = _size(rng, 1, min(16384, 4096 * 14336 // c["rows"]))
        c["pad"] = rng.choice([0, 0, rng.randint(1, 64)])
        c["x"] = rng.choice(["bf16", "fp16", "fp32"])
    elif c["op"] == "skinny":
        c["M"] = rng.randint(1, 32)
        c["N"] = _size(rng, 1, 28672)
        c["K"] = _size(rng, 1, min(14336, 28672 * 4096 // c["N"]))
    else:
        most = 8192 ** 3 // (3 if c["op"] == "train" else 1)
        c["M"] = _size(rng, 1, 4096 if c["op"] == "train" else 8192)
        c["N"] = _size(rng, 1, min(28672, most // (c["M"] * 128)))
        c["K"] = _size(rng, 1, min(14336, most // (c["M"] * c["N"])))
    c["out"] = rng.choice(["bf16", "fp16", "fp32"])
    return c


# ------------------------------------------------------------------ plain form
_LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _up(n, m):
    return (n + m - 1) // m * m


def _tiled(s):
    """[rows, blocks] scale bytes -> the tiles that the products read (flat)."""
    rows, blocks = s.shape
    return s.reshape(rows // 128, 4, 32, blocks // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _untiled(flat, rows, blocks):
    """The flat tiles -> [rows, blocks]."""
    tiles = flat.reshape(_up(rows, 128) // 128, -1, 32, 4, 4)
    s = tiles.permute(0, 3, 2, 1, 4).reshape(_up(rows, 128), -1)
    return s[:rows, :blocks]


def _e2m1_codes(v):
    """fp32 -> e2m1 codes: how many of the borders lie below; a border goes to its even neighbour."""
    a = v.abs()
    c = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return c | (torch.signbit(v).to(torch.uint8) << 3)


def _power(e):
    """2^e in fp32 for whole e of -127 to 127: the exponent field itself, the lowest one a subnormal number."""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _quantize(x, form):
    """(codes, tiled scales, tensor scale or None) of a [rows, K] tensor."""
    rows, K = x.shape
    b = BLOCK[form]
    xb = torch.nn.functional.pad(x.float(), (0, _up(K, 32) - K)).reshape(rows, -1, b)
    amax = xb.abs().amax(dim=2, keepdim=True)
    if form == "mxfp4":
        t = None
        e = torch.clamp(torch.frexp(amax)[1] - 3, -127, 127)      # frexp's mantissa lies in [0.5, 1)
        e = torch.where(amax > 0, e, torch.full_like(e, -127))
        scale = (e + 127).to(torch.uint8)
        q = xb * _power(-e)
    else:
        top = amax.max()
        t = torch.where(top > 0, torch.clamp(top / 2688.0, min=2.0 ** -126), torch.ones_like(top)).reshape(1)
        s8 = torch.clamp(amax / (t * 6.0), max=448.0).to(torch.float8_e4m3fn)
        scale = s8.view(torch.uint8)
        s = s8.float() * t
        q = torch.where(s > 0, xb / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(xb))
    codes = _e2m1_codes(q).reshape(rows, -1)
    codes = codes[:, 0::2] | (codes[:, 1::2] << 4)
    scale = scale.reshape(rows, -1)
    scale = torch.nn.functional.pad(scale, (0, _up(K, 256) // b - scale.shape[1], 0, _up(rows, 128) - rows))
    return codes.contiguous(), _tiled(scale), t


def _values(codes, scales, form, K):
    """What codes and scales stand for, without the tensor scale, in fp32 (exact)."""
    rows = codes.shape[0]
    b = BLOCK[form]
    level = torch.tensor(_LEVELS + [-v for v in _LEVELS], device=codes.device)
    pair = torch.stack([level.repeat(16), level.repeat_interleave(16)], dim=1)          # by a whole byte
    v = pair[codes.int()].reshape(rows, -1, b)
    s = _untiled(scales, rows, v.shape[1])
    s = _power(s.int() - 127) if form == "mxfp4" else s.contiguous().view(torch.float8_e4m3fn).float()
    return (v * s.unsqueeze(2)).reshape(rows, -1)[:, :K]


def _dequantize(q, form, K, dtype):
    codes, scales, t = q
    v = _values(codes, scales, form, K)
    return (v if t is None else v * t).to(dtype)


def _product(a, b, form, K, dtype):
    d = _values(a[0], a[1], form, K) @ _values(b[0], b[1], form, K).t()
    return (d if a[2] is None else d * (a[2] * b[2])).to(dtype)


# ------------------------------------------------------------------ inputs
def _gauss(g, rows, K, dtype, std=1.0, pad=0):
    """A [rows, K] view of a buffer that is `pad` wider on both sides.  Rows differ in size as a layer's channels do."""
    x = torch.randn((rows, K + 2 * pad), generator=g, device="cuda")
    x *= std * torch.exp2(torch.randint(-2, 3, (rows, 1), generator=g, device="cuda").float())
    return x.to(dtype)[:, pad:pad + K]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    form = case["format"]
    s = dict(case)
    if case["op"] in ("quantize", "both"):
        s["x"] = _gauss(g, case["rows"], case["K"], TYPES[case["x"]], pad=case["pad"])
    elif case["op"] == "train":
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = _gauss(g, M, K, torch.bfloat16)
        s["w"] = _gauss(g, N, K, torch.bfloat16, 0.02)
        s["dy"] = _gauss(g, M, N, torch.bfloat16, 1e-3)
    else:
        # a program that serves keeps its weights quantised, and has quantised its activations before
        s["a"] = _quantize(_gauss(g, case["M"], case["K"], torch.bfloat16), form)
        s["b"] = _quantize(_gauss(g, case["N"], case["K"], torch.bfloat16, 0.02), form)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    form, out = s["format"], TYPES[s["out"]]
    if own:
        import rocm_dev_b200 as R
        if s["op"] == "quantize":
            return R.dequantize_fp4(R.quantize_fp4(s["x"], form), out)
        if s["op"] == "both":
            r, c = R.quantize_fp4_both(s["x"], form)
            return R.dequantize_fp4(r, out), R.dequantize_fp4(c, out)
        if s["op"] == "train":
            xr, xc = R.quantize_fp4_both(s["x"], form)
            wr, wc = R.quantize_fp4_both(s["w"], form)
            gr, gc = R.quantize_fp4_both(s["dy"], form)
            return R.dense_gemm_fp4(xr, wr, out_dtype=out), R.dense_gemm_fp4(gr, wc, out_dtype=out), R.dense_gemm_fp4(gc, xc, out_dtype=torch.float32)
        a = R.Fp4Tensor(*s["a"], form, s["M"], s["K"])
        b = R.Fp4Tensor(*s["b"], form, s["N"], s["K"])
        product = R.skinny_gemm_fp4 if s["op"] == "skinny" else R.dense_gemm_fp4
        return product(a, b, out_dtype=out)
    if s["op"] in ("quantize", "both"):
        x = s["x"]
        r = _dequantize(_quantize(x, form), form, x.shape[1], out)
        return r if s["op"] == "quantize" else (r, _dequantize(_quantize(x.t(), form), form, x.shape[0], out))
    if s["op"] == "train":
        x, w, dy = s["x"], s["w"], s["dy"]
        M, N, K = s["M"], s["N"], s["K"]
        y = _product(_quantize(x, form), _quantize(w, form), form, K, out)
        dx = _product(_quantize(dy, form), _quantize(w.t(), form), form, N, out)
        dw = _product(_quantize(dy.t(), form), _quantize(x.t(), form), form, M, torch.float32)
        return y, dx, dw
    return _product(s["a"], s["b"], form, s["K"], out)


# ------------------------------------------------------------------ what a pass cannot do without
def _held(rows, K, form):
    """Bytes of a quantised tensor: half a byte an element, a byte a block, the tensor scale."""
    return rows * K / 2 + rows * math.ceil(K / BLOCK[form]) + (4 if form == "nvfp4" else 0)


def work(case):
    form = case["format"]
    if case["op"] in ("quantize", "both"):
        n = case["rows"] * case["K"]
        ways = [(case["rows"], case["K"]), (case["K"], case["rows"])][: 1 if case["op"] == "quantize" else 2]
        # x once; for each direction the quantised form, and the values that are read back from it
        return {"bytes": n * SIZE[case["x"]] + sum(_held(r, k, form) + n * SIZE[case["out"]] for r, k in ways), "flops": 3 * n * len(ways)}
    M, N, K = case["M"], case["N"], case["K"]
    o = SIZE[case["out"]]
    if case["op"] == "train":
        read = 2 * (M * K + N * K + M * N)
        return {"bytes": read + M * N * o + M * K * o + N * K * 4, "flops": 6 * M * N * K}
    return {"bytes": _held(M, K, form) + _held(N, K, form) + M * N * o, "flops": 2 * M * N * K}


# ------------------------------------------------------------------ the definition in 64 bits
def _r32(v):
    return v.to(torch.float32).to(torch.float64)


def _nearest(v, mantissa, least, most):
    """v >= 0 to the nearest number of a small float type (ties to even): steps of 2^(exponent - mantissa), the exponent
    no lower than `least`, nothing above `most`."""
    e = torch.clamp(torch.frexp(v)[1].to(torch.float64) - 1, min=least)
    step = torch.exp2(e - mantissa)
    return torch.clamp(torch.round(v / step) * step, max=most)


def _exact_values(x, form):
    """The values that the quantised x stands for, in 64 bits, and the tensor scale that they still lack."""
    rows, K = x.shape
    b = BLOCK[form]
    v = torch.zeros((rows, (K + b - 1) // b * b), dtype=torch.float64, device=x.device)
    v[:, :K] = x
    v = v.reshape(rows, -1, b)
    top = v.abs().amax(dim=2, keepdim=True)
    if form == "mxfp4":
        s = torch.exp2(torch.clamp(torch.frexp(top)[1].to(torch.float64) - 3, -127, 127))
        t = 1.0
        whole = s
    else:
        t = _r32(top.max() / 2688)
        t = torch.ones_like(t) if float(t) == 0 and float(top.max()) == 0 else torch.clamp(t, min=2.0 ** -126)
        s = _nearest(_r32(top / _r32(6 * t)), 3, -6, 448.0)
        whole = _r32(s * t)
    q = _r32(v / torch.where(whole > 0, whole, torch.full_like(whole, math.inf)))
    q = torch.sign(q) * _nearest(q.abs(), 1, 0, 6.0)
    return (q * s).reshape(rows, -1)[:, :K], t


def _exact_held(q, form, K):
    """The same for a tensor that is already quantised: each code and each scale byte by its bits."""
    codes, flat, t = q
    rows, b = codes.shape[0], BLOCK[form]
    k = torch.arange(K, device=codes.device)
    code = (codes[:, k // 2] >> (4 * (k % 2)).to(torch.uint8)) & 15
    low, exp = (code & 1).to(torch.float64), ((code >> 1) & 3).to(torch.float64)
    v = torch.where(exp > 0, (1 + low / 2) * torch.exp2(exp - 1), low / 2)
    v = torch.where(code >= 8, -v, v)
    r, blk = torch.arange(rows, device=codes.device)[:, None], torch.arange((K + b - 1) // b, device=codes.device)[None, :]
    across = (K + 255) // 256 * (256 // b) // 4
    byte = flat[(r // 128 * across + blk // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + blk % 4]
    if form == "mxfp4":
        s = torch.exp2(byte.to(torch.float64) - 127)
    else:
        m, e = (byte & 7).to(torch.float64), (byte >> 3).to(torch.float64)
        s = torch.where(e > 0, (1 + m / 8) * torch.exp2(e - 7), m / 8 * 2.0 ** -6)
    return v * s[:, k // b], 1.0 if t is None else t.to(torch.float64)


def exact(case, seed):
    s, form = prepare(case, seed), case["format"]

    def whole(x):
        v, t = _exact_values(x, form)
        return v * t

    def product(a, b):
        return a[0] @ b[0].t() * (a[1] * b[1])

    if case["op"] == "quantize":
        return whole(s["x"])
    if case["op"] == "both":
        return whole(s["x"]), whole(s["x"].t())
    if case["op"] == "train":
        x, w, dy = s["x"], s["w"], s["dy"]
        return (product(_exact_values(x, form), _exact_values(w, form)), product(_exact_values(dy, form), _exact_values(w.t(), form)),
                product(_exact_values(dy.t(), form), _exact_values(x.t(), form)))
    return product(_exact_held(s["a"], form, case["K"]), _exact_held(s["b"], form, case["K"]))
