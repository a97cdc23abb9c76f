// Quantisers into microscaled 4-bit floating point (fp4.cuh describes the held form) and the way back.
//
// MXFP4: a block of 32 with largest magnitude a > 0 is scaled by 2^e, e = floor(log2 a) - 2 (2 = exponent of e2m1's
// largest number) clamped to [-127, 127]; e = -127 for a = 0.  Element = e2m1(x * 2^-e).
// NVFP4: the tensor has one fp32 scale t - given, or max|x| * fp32(1 / 2688) (2688 = 448 * 6) but no lower than 2^-126, 1
// for an all-zero tensor - and a block of 16 an e4m3 scale s = e4m3_sat(a / (6 t)).  Element = e2m1(x / (t s)), zero where s is.  6 t,
// t s and both quotients are rounded to fp32 (IEEE), which makes the codes reproducible bit for bit.
// e2m1 rounds to nearest, ties to the even code, and saturates at 6.  A block that holds an infinity or a NaN gets the
// scale type's NaN (0xFF, 0x7F): whatever is computed from it is NaN, and the other blocks keep their values - t is the
// largest FINITE magnitude.
#include <cuda_fp8.h>

#include <type_traits>

#include "fp4.cuh"
#include "host_util.h"
#include "ptx.cuh"

RDB_DEFINE_WAIT_BUDGET_SETTER()

namespace rdb {
namespace fp4 {

constexpr int kThreads = 256;
constexpr int kAmaxBlocks = RDB_FP4_WORKSPACE_FLOATS;    // upper bound of the first pass's grid: one partial maximum each
constexpr uint32_t kInf = 0x7F800000u;

// The next kernel may start once this one's predecessor has finished, not before: a launch that fetches its weights early
// then overlaps this kernel alone, never one further back that may have written them.
__device__ __forceinline__ void start_after_prior() {
    pdl_wait_prior();
    pdl_launch_dependents();
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 32 bytes with one load (a whole sector); p is 32-byte aligned.
__device__ __forceinline__ void ldg32(const void* p, uint32_t* w) {
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
}

__device__ __forceinline__ void stg32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// Words of memory as floats.
template <class T, int N>
__device__ __forceinline__ void unpack(const uint32_t* w, float* v) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(w + i));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

// Largest magnitude of elements held in words, as fp32 bits: non-negative floats order like integers, infinities and NaNs
// above every number.  16-bit types are compared two at a time: the halves of the result are the maxima of the halves
// (a NaN wins and stays one).
template <class T, int WORDS>
__device__ __forceinline__ uint32_t halves_magnitude(const uint32_t* w) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
        for (int i = 1; i < WORDS; i++) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        return m;
    } else {
        __half2 m = __habs2(*reinterpret_cast<const __half2*>(w));
#pragma unroll
        for (int i = 1; i < WORDS; i++) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(w + i)));
        return *reinterpret_cast<const uint32_t*>(&m) & 0x7FFF7FFFu;
    }
}
template <class T>
__device__ __forceinline__ uint32_t bits_of_half(uint32_t h) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) return h << 16;
    else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h))));
}
template <class T, int N>
__device__ __forceinline__ uint32_t magnitude(const uint32_t* w) {
    if constexpr (sizeof(T) == 4) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; i++) m = max(m, w[i] & 0x7FFFFFFFu);
        return m;
    } else {
        const uint32_t m = halves_magnitude<T, N / 2>(w);
        return bits_of_half<T>(max(m & 0xFFFFu, m >> 16));
    }
}

// The same over the finite elements alone.
template <class T, int N>
__device__ __forceinline__ uint32_t finite_magnitude(const uint32_t* w) {
    uint32_t m = magnitude<T, N>(w);
    if (m >= kInf) {
        float v[N];
        unpack<T, N>(w, v);
        m = 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t a = __float_as_uint(v[i]) & 0x7FFFFFFFu;
            if (a < kInf) m = max(m, a);
        }
    }
    return m;
}

// The same of 16 or 32 floats: a tree of sm_100's three-operand maxima (a NaN wins).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float m;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}
template <int N>
__device__ __forceinline__ uint32_t magnitude(const float* v) {
    float m[N / 16];
#pragma unroll
    for (int h = 0; h < N / 16; h++) {
        const float* u = v + 16 * h;
        m[h] = max3(max3(max3(u[0], u[1], u[2]), max3(u[3], u[4], u[5]), max3(u[6], u[7], u[8])),
                    max3(max3(u[9], u[10], u[11]), max3(u[12], u[13], u[14]), u[15]), 0.0f);
    }
    return __float_as_uint(N == 16 ? m[0] : max3(m[0], m[N / 16 - 1], 0.0f)) & 0x7FFFFFFFu;
}

// 8 floats -> 8 e2m1 codes.
__device__ __forceinline__ uint32_t pack8(const float* q) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r) : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
    return r;
}

// Two fp32 operations in one instruction (sm_100).
struct Pair { uint64_t v; };
__device__ __forceinline__ Pair pair(float x, float y) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(x), "f"(y));
    return p;
}
__device__ __forceinline__ void split(Pair p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p.v)); }
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair p;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
    return p;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair p;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return p;
}

// Quotients a / d of many numerators by one divisor d > 0, rounded to fp32 as the IEEE division does as far as the result
// tells.  With inv near 1 / d: q = a * inv, then the step q + inv * (a - q d).  It is NEGATIVE quotients that are
// computed: with -q and -1 / d the step keeps the sign of a zero.
// fp32 numerators: inv = RN(1 / d) and two steps - after the first, q is within a unit of the last place, and from such a q
// the second gives the rounded quotient (Markstein).  16-bit numerators: one step, after which the code or scale byte is the
// division's - all quotients of 11-bit significands next to a border of e2m1 or e4m3 were gone through, with exact
// arithmetic.  With inv = RN(1 / d) that holds for every divisor; with an approximate reciprocal (one unit off) for all but
// those whose 23 bits are all set: a power of two over 2 - 2^-23 lies 2^-25 units from where the rounded quotient leaves the
// border.  No tensor scale computed from a 16-bit maximum makes such a divisor; for a given one (PATCH) its reciprocal, whose
// bits are known, replaces the approximation.  (RN(1 / d) for every block costs more: 4096 x 14336 bf16 by rows 32.4 us
// in place of 25.4.)
struct Scale {
    float t, t6, n6;             // tensor scale; 6 t and -1 / (6 t), both for numerators that are multiplied by `move`
    float move;                  // 1, or a power of two for tensor scales so far from 1 that the steps would leave fp32
};
template <class T, bool PATCH>
__device__ __forceinline__ float neg_reciprocal(float d) {
    if constexpr (sizeof(T) == 4) return -__frcp_rn(d);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    if constexpr (PATCH) {
        // 1 / (2^k (2 - 2^-23)) rounds to 2^(-k - 1) (1 + 2^-23): exponent field 253 less d's, lowest bit set
        const uint32_t bits = __float_as_uint(d);
        if ((~bits & 0x7FFFFFu) == 0) r = __uint_as_float(0x7F000000u - bits);
    }
    return -r;
}
template <class T>
constexpr int kSteps = sizeof(T) == 4 ? 2 : 1;

// One block: v[BLOCK] -> BLOCK / 8 words of codes, returns the scale byte.  CAREFUL: sc.move is not 1, or the tensor scale
// was given and quotients may overflow.
template <class T, int FMT, bool CAREFUL>
__device__ __forceinline__ uint32_t encode_block(float* v, uint32_t amax, const Scale& sc, uint32_t* codes) {
    constexpr int B = Format<FMT>::BLOCK;
    if constexpr (FMT == RDB_FP4_MXFP4) {
        // the exponent field of the largest magnitude is floor(log2) + 127 (0 for subnormals, whose clamp is 0 too)
        const uint32_t byte = max(static_cast<int>(amax >> 23) - 2, 0);
        const float inv = __uint_as_float((254 - byte) << 23);       // 2^(127 - byte), exact products below
        const Pair inv2 = pair(inv, inv);
#pragma unroll
        for (int g = 0; g < B / 8; g++) {
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; i += 2) split(mul2(pair(v[8 * g + i], v[8 * g + i + 1]), inv2), q[i], q[i + 1]);
            codes[g] = pack8(q);
        }
        return amax >= kInf ? 0xFF : byte;
    } else {
        float a = __uint_as_float(amax);
        if constexpr (CAREFUL) {
            a *= sc.move;
            const float top = 1024.0f * sc.t6, most = top / sc.move;     // beyond it everything saturates
            if (!(a <= top)) {
                a = top;
#pragma unroll
                for (int i = 0; i < B; i++) v[i] = fminf(fmaxf(v[i], -most), most);
            }
        }
        float n = a * sc.n6;
#pragma unroll
        for (int k = 0; k < kSteps<T>; k++) n = __fmaf_rn(__fmaf_rn(n, sc.t6, a), sc.n6, n);
        uint16_t e;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(e) : "f"(0.0f), "f"(-n));
        uint32_t h2;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(e));
        const uint32_t byte = e;
        float d = __half2float(__ushort_as_half(static_cast<unsigned short>(h2))) * sc.t;
        if constexpr (CAREFUL) d *= sc.move;
        const float ninv = neg_reciprocal<T, CAREFUL>(d);
        const Pair d2 = pair(d, d), n2 = pair(ninv, ninv);
        const uint32_t keep = byte != 0 ? ~0u : 0u;                  // a scale of zero: zeros
#pragma unroll
        for (int g = 0; g < B / 8; g++) {
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                Pair x = pair(v[8 * g + i], v[8 * g + i + 1]);
                if constexpr (CAREFUL) x = mul2(x, pair(sc.move, sc.move));
                Pair y = mul2(x, n2);
#pragma unroll
                for (int k = 0; k < kSteps<T>; k++) y = fma2(fma2(y, d2, x), n2, y);
                split(y, q[i], q[i + 1]);
            }
            codes[g] = (pack8(q) ^ 0x88888888u) & keep;
        }
        return amax >= kInf ? 0x7F : byte;
    }
}

__device__ __forceinline__ Scale scale_of(float t) {
    Scale sc;
    sc.t = t;
    sc.move = t < 8.6736174e-19f ? 18446744073709551616.0f : t > 1.1529215e18f ? 5.4210109e-20f : 1.0f;   // 2^-60, 2^64; 2^60, 2^-64
    sc.t6 = t * 6.0f * sc.move;
    sc.n6 = -__frcp_rn(sc.t6);
    return sc;
}
__device__ __forceinline__ Scale scale_of_maximum(uint32_t m) {
    constexpr float inv = 1.0f / 2688.0f;                // rounded to fp32 before it multiplies: part of the definition
    return scale_of(m == 0 ? 1.0f : fmaxf(__fmul_rn(__uint_as_float(m), inv), 1.17549435e-38f));
}

// The tensor scale (NVFP4: given, or from the first pass's partial maxima), for the whole block: every thread takes part.
template <int FMT, int THREADS>
__device__ __forceinline__ Scale fetch_scale(float* tscale, const float* given, const uint32_t* partial, int partials) {
    Scale sc = {1.0f, 6.0f, 0.0f, 1.0f};
    if constexpr (FMT == RDB_FP4_NVFP4) {
        if (partial) {
            __shared__ uint32_t warp_max[THREADS / 32];
            uint32_t m = 0;
            for (int i = threadIdx.x; i < partials; i += THREADS) m = max(m, __ldcg(partial + i));
            m = __reduce_max_sync(0xffffffffu, m);
            if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < THREADS / 32; w++) m = max(m, warp_max[w]);
            sc = scale_of_maximum(m);
        } else {
            sc = scale_of(*given);
        }
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *tscale = sc.t;
    }
    return sc;
}

// First pass of a call that computes the tensor scale: one partial maximum per CTA.  A warp takes stretches of 1024
// elements of a row: single elements up to the first 16-byte boundary and behind the last, whole vectors between them.
// Bound by HBM: 4096 x 14336 bf16 (117 MB) takes 24 us before the row quantiser, 15 to 17 before the two-way one, which
// begins with the rows that were read last.
constexpr int kAmaxStretch = 1024;
template <class T>
__global__ void __launch_bounds__(kThreads) amax_kernel(const T* __restrict__ x, long long ldx, int rows, int K, uint32_t* __restrict__ partial) {
    __shared__ uint32_t warp_max[kThreads / 32];
    start_after_prior();
    constexpr int N = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
    const int per_row = (K - 1) / kAmaxStretch + 1;
    const long long units = static_cast<long long>(per_row) * rows;
    uint32_t m = 0;
    for (long long u = blockIdx.x * static_cast<long long>(kThreads / 32) + (threadIdx.x >> 5); u < units; u += static_cast<long long>(gridDim.x) * (kThreads / 32)) {
        const long long r = u / per_row;
        const int k = static_cast<int>(u - r * per_row) * kAmaxStretch;
        const int n = K - k < kAmaxStretch ? K - k : kAmaxStretch;
        const T* p = x + r * ldx + k;
        int head = static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
        if (head > n) head = n;
        const int vectors = (n - head) / N, tail = head + vectors * N;
        auto single = [&](int i) {
            const uint32_t a = __float_as_uint(to_f32(p[i])) & 0x7FFFFFFFu;
            if (a < kInf) m = max(m, a);
        };
        if (lane < head) single(lane);
        if (tail + lane < n) single(tail + lane);
        const uint4* q = reinterpret_cast<const uint4*>(p + head);
        int i = lane;
        for (; i + 96 < vectors; i += 128) {
            uint4 w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = __ldg(q + i + 32 * j);
#pragma unroll
            for (int j = 0; j < 4; j++) m = max(m, finite_magnitude<T, N>(&w[j].x));
        }
        for (; i < vectors; i += 32) {
            const uint4 w = __ldg(q + i);
            m = max(m, finite_magnitude<T, N>(&w.x));
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < kThreads / 32; w++) m = max(m, warp_max[w]);
        partial[blockIdx.x] = m;
    }
}

template <int B>
__device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t* c) {
    if constexpr (B == 16) *reinterpret_cast<uint2*>(p) = make_uint2(c[0], c[1]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(c[0], c[1], c[2], c[3]);
}

// Blocks along the rows, x on 16-byte boundaries and K a multiple of the block: a thread holds a whole block, so nothing
// but the scale bytes passes between threads.  A warp takes 32 blocks of the rows r, r + 32, r + 64, r + 96 of a 128-row
// tile: four loads in flight, and the four scale words of a lane quartet are 16 consecutive bytes of the scale tile.
// ALIGN: 32 or 16 bytes.  Bound by HBM: 4096 x 14336 bf16 takes 24 us in MXFP4 and 25 in NVFP4 with a given scale (23 at
// the copy rate), fp32 46 (42).
template <class T, int FMT, int ALIGN>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, long long ldx, int rows, int K, float* tscale,
                                                                 const float* given, const uint32_t* partial, int partials, uint8_t* __restrict__ codes,
                                                                 uint8_t* __restrict__ scales) {
    constexpr int B = Format<FMT>::BLOCK, WORDS = B * sizeof(T) / 4, HELD = WORDS > 16 ? 2 : 4;
    start_after_prior();
    const Scale scale = fetch_scale<FMT, kThreads>(tscale, given, partial, partials);
    const size_t pitch = row_bytes(K);
    const int tiles = scale_tiles_per_row(FMT, K);
    const int lane = threadIdx.x & 31, b = blockIdx.x * 32 + lane, blocks = K / B;
    const int octets = static_cast<int>((rows + 127ll) / 128 * 4);
    auto body = [&](auto careful) {
        // after the maximum's pass the last rows first: it read them last, and they may still be in L2
        for (int n = blockIdx.y; n < octets; n += gridDim.y) {
            const int o = partial ? octets - 1 - n : n;
            const int r0 = (o >> 2) * 128 + (o & 3) * 8 + (threadIdx.x >> 5);
            if (r0 >= rows) continue;
            uint32_t byte[4] = {0, 0, 0, 0};
#pragma unroll
            for (int h = 0; h < 4; h += HELD) {
                uint32_t w[HELD][WORDS];
#pragma unroll
                for (int j = 0; j < HELD; j++) {
                    const int r = r0 + 32 * (h + j);
                    if (r < rows && b < blocks) {
                        const uint32_t* p = reinterpret_cast<const uint32_t*>(x + r * ldx + static_cast<size_t>(b) * B);
                        if constexpr (ALIGN == 32) {
#pragma unroll
                            for (int i = 0; i < WORDS; i += 8) ldg32(p + i, w[j] + i);
                        } else {
#pragma unroll
                            for (int i = 0; i < WORDS; i += 4) *reinterpret_cast<uint4*>(w[j] + i) = __ldg(reinterpret_cast<const uint4*>(p + i));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < WORDS; i++) w[j][i] = 0;
                    }
                }
#pragma unroll
                for (int j = 0; j < HELD; j++) {
                    const int r = r0 + 32 * (h + j);
                    if (r >= rows) break;
                    float v[B];
                    unpack<T, B>(w[j], v);
                    uint32_t c[B / 8];
                    const uint32_t amax = FMT == RDB_FP4_MXFP4 ? magnitude<T, B>(w[j]) : magnitude<B>(v);     // each the faster one here
                    byte[h + j] = encode_block<T, FMT, decltype(careful)::value>(v, amax, scale, c);
                    if (static_cast<size_t>(b) * (B / 2) < pitch) store_codes<B>(codes + r * pitch + static_cast<size_t>(b) * (B / 2), c);
                }
            }
            uint32_t word[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                word[j] = byte[j] << (8 * (lane & 3));
                word[j] |= __shfl_xor_sync(0xffffffffu, word[j], 1);
                word[j] |= __shfl_xor_sync(0xffffffffu, word[j], 2);
            }
            if ((lane & 3) == 0 && (b >> 2) < tiles)
                *reinterpret_cast<uint4*>(scales + scale_word(r0, b >> 2, tiles)) = make_uint4(word[0], word[1], word[2], word[3]);
        }
    };
    if (FMT == RDB_FP4_NVFP4 && (scale.move != 1.0f || !partial)) body(std::true_type());
    else body(std::false_type());
}

// A tensor small enough for the registers of one cluster (a decode step's activations): maximum and codes in one launch, x
// read once.  The blocks of the rows are dealt to the threads of the cluster's CTAs, HELD to a thread; the CTAs exchange
// their maxima through distributed shared memory.
constexpr int kSmallThreads = 512, kSmallCluster = 8;
template <class T, int HELD>
__global__ void __launch_bounds__(kSmallThreads) quantize_small_kernel(const T* __restrict__ x, long long ldx, int rows, int K, float* tscale,
                                                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    constexpr int B = 16, WORDS = B * sizeof(T) / 4, FMT = RDB_FP4_NVFP4;
    __shared__ uint32_t warp_max[kSmallThreads / 32], cta_max;
    start_after_prior();
    const size_t pitch = row_bytes(K);
    const int tiles = scale_tiles_per_row(FMT, K), per_row = 4 * tiles, total = rows * per_row, blocks = K / B;
    const int first = blockIdx.x * kSmallThreads + threadIdx.x, step = gridDim.x * kSmallThreads;
    uint32_t w[HELD][WORDS], amax[HELD], m = 0;
#pragma unroll
    for (int j = 0; j < HELD; j++) {
        const int i = first + j * step, r = i / per_row, b = i - r * per_row;
        if (i < total && b < blocks) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(x + r * ldx + static_cast<size_t>(b) * B);
#pragma unroll
            for (int k = 0; k < WORDS; k += 4) *reinterpret_cast<uint4*>(w[j] + k) = __ldg(reinterpret_cast<const uint4*>(p + k));
        } else {
#pragma unroll
            for (int k = 0; k < WORDS; k++) w[j][k] = 0;
        }
    }
#pragma unroll
    for (int j = 0; j < HELD; j++) {
        amax[j] = magnitude<T, B>(w[j]);
        m = max(m, amax[j] < kInf ? amax[j] : finite_magnitude<T, B>(w[j]));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSmallThreads / 32; i++) m = max(m, warp_max[i]);
    if (gridDim.x > 1) {
        if (threadIdx.x == 0) cta_max = m;
        cluster_arrive_release();
        cluster_wait_acquire();
        for (unsigned c = 0; c < gridDim.x; c++) {
            uint32_t o;
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(o) : "r"(mapa_smem(smem_u32(&cta_max), c)) : "memory");
            m = max(m, o);
        }
        cluster_arrive_release();                        // (waited for at the end: nobody leaves before all have read)
    }
    const Scale scale = scale_of_maximum(m);
    if (first == 0) *tscale = scale.t;
    auto body = [&](auto careful) {
#pragma unroll
        for (int j = 0; j < HELD; j++) {
            const int i = first + j * step, r = i / per_row, b = i - r * per_row;
            uint32_t byte = 0;
            if (i < total && static_cast<size_t>(b) * (B / 2) < pitch) {
                float v[B];
                unpack<T, B>(w[j], v);
                uint32_t c[B / 8];
                byte = encode_block<T, FMT, decltype(careful)::value>(v, amax[j], scale, c);
                store_codes<B>(codes + r * pitch + static_cast<size_t>(b) * (B / 2), c);
            }
            uint32_t word = byte << (8 * (threadIdx.x & 3));
            word |= __shfl_xor_sync(0xffffffffu, word, 1);
            word |= __shfl_xor_sync(0xffffffffu, word, 2);
            if ((threadIdx.x & 3) == 0 && i < total) *reinterpret_cast<uint32_t*>(scales + scale_word(r, b >> 2, tiles)) = word;
        }
    };
    if (scale.move != 1.0f) body(std::true_type());
    else body(std::false_type());
    if (gridDim.x > 1) cluster_wait_acquire();
}

// Blocks along the rows, and along the columns too, of 128 x 128 tiles in shared memory: x is read once whatever its
// alignment, and both directions' scale bytes make whole 512-byte tiles.  Shared memory: rows of W words, in which the
// 8-word group g of row r lies at g ^ (r / B) % 4 - a column's reader takes words of four row blocks at once (lane = 8
// words x 4 row blocks), which the exchange puts into different banks.  Persistent blocks: while a tile is encoded, the
// next one is copied into the other buffer (x on 16-byte boundaries; else the copy waits).
constexpr int kTileThreads = 512;
template <class T, int FMT>
struct TileCfg {
    static constexpr int B = Format<FMT>::BLOCK, NB = 128 / B;      // blocks across the tile
    static constexpr int W = 32 * sizeof(T);                        // words of a row
    static constexpr int CPW = 4 / sizeof(T);                       // columns in a word
    static constexpr int TILE_WORDS = 128 * W;
    static constexpr int BUFFERS = 2;
    static constexpr int SMEM = BUFFERS * TILE_WORDS * 4 + 2 * NB * 128;
    static constexpr int PER_SM = sizeof(T) == 2 ? 2 : 1;
};
__device__ __forceinline__ void cp_async16(uint32_t smem, const void* src, bool exists) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(src), "r"(exists ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 16 bytes of a row from element c on, zeros behind its K elements.  Off a 16-byte boundary: the aligned words that hold
// them, shifted together - where all lie inside the row; else element by element.
template <class T>
__device__ __forceinline__ uint4 load_vector(const T* row, long long c, int K, bool aligned) {
    constexpr int VE = 16 / sizeof(T);
    const T* p = row + c;
    if (aligned && c + VE <= K) return __ldg(reinterpret_cast<const uint4*>(p));
    if constexpr (sizeof(T) == 4) {
        if (c + VE <= K) {
            const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
            return make_uint4(__ldg(q), __ldg(q + 1), __ldg(q + 2), __ldg(q + 3));
        }
    } else {
        const int odd = (reinterpret_cast<uintptr_t>(p) >> 1) & 1;
        if (c >= odd && c + VE + odd <= K) {
            const uint32_t* q = reinterpret_cast<const uint32_t*>(p - odd);
            const uint32_t w[5] = {__ldg(q), __ldg(q + 1), __ldg(q + 2), __ldg(q + 3), odd ? __ldg(q + 4) : 0u};
            const uint32_t s = 16 * odd;
            return make_uint4(__funnelshift_r(w[0], w[1], s), __funnelshift_r(w[1], w[2], s), __funnelshift_r(w[2], w[3], s), __funnelshift_r(w[3], w[4], s));
        }
    }
    alignas(16) T e[VE];
#pragma unroll
    for (int i = 0; i < VE; i++) e[i] = c + i < K ? p[i] : from_f32<T>(0.0f);
    return *reinterpret_cast<const uint4*>(e);
}

// Bound by instructions (shifted loads, a transpose through shared memory): 4096 x 14336 bf16 off 16 bytes takes 60 us by
// rows, both ways 74 in MXFP4 and 82 in NVFP4, where aligned rows take 24, 34 and 50.
template <class T, int FMT, bool COLS>
__global__ void __launch_bounds__(kTileThreads, TileCfg<T, FMT>::PER_SM)
quantize_tile_kernel(const T* __restrict__ x, long long ldx, int rows, int K, int vec, unsigned tiles_x, unsigned tiles_all, float* tscale,
                     const float* given, const uint32_t* partial, int partials, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                     uint8_t* __restrict__ codes_t, uint8_t* __restrict__ scales_t) {
    using C = TileCfg<T, FMT>;
    constexpr int B = C::B, NB = C::NB, W = C::W, CPW = C::CPW, BW = B * sizeof(T) / 4;
    extern __shared__ __align__(16) uint32_t buffers[];
    uint8_t* sc = reinterpret_cast<uint8_t*>(buffers + C::BUFFERS * C::TILE_WORDS);     // [NB / 4][512] along the rows
    uint8_t* sc_t = sc + NB * 128;                                                      // the same along the columns
    start_after_prior();
    auto at = [](int r, int w) { return r * W + (w ^ (((r / B) & 3) << 3)); };
    const size_t pitch = row_bytes(K), pitch_t = row_bytes(rows);
    constexpr int V = W / 4, VE = 16 / sizeof(T), STEP = kTileThreads / V;     // vectors of a row, elements of a vector, rows a pass

    // The block's tiles are n = blockIdx.x, + gridDim.x, ... counted from the last one: the maximum's pass read those
    // last, and they may still be in L2.  (tr, tc): row and column of tile n; moving on by gridDim.x tiles.
    const unsigned tiles_y = tiles_all / tiles_x, hop_y = gridDim.x / tiles_x, hop_x = gridDim.x - hop_y * tiles_x;
    auto advance = [&](int& tr, int& tc) {
        tr -= hop_y;
        tc -= hop_x;
        if (tc < 0) { tc += tiles_x; tr--; }
    };
    // tile -> buffer, zeros outside x
    const int fr = threadIdx.x / V, fv = threadIdx.x % V;
    auto fetch = [&](int tr, int tc, uint32_t* tile) {
        const long long c = tc * 128ll + fv * VE, row = tr * 128ll + fr;
        const T* p = x + row * ldx;
        if (vec && c + VE <= K) {
            if (tr * 128ll + 128 <= rows) {
                p += c;
#pragma unroll
                for (int j = 0; j < 128 / STEP; j++, p += STEP * ldx) cp_async16(smem_u32(tile + at(fr + j * STEP, 4 * fv)), p, true);
            } else {
#pragma unroll
                for (int j = 0; j < 128 / STEP; j++) {
                    const bool exists = row + j * STEP < rows;
                    cp_async16(smem_u32(tile + at(fr + j * STEP, 4 * fv)), exists ? p + j * STEP * ldx + c : x, exists);
                }
            }
        } else {
            uint4 q[128 / STEP];
#pragma unroll
            for (int j = 0; j < 128 / STEP; j++)
                q[j] = row + j * STEP < rows && c < K ? load_vector(p + j * STEP * ldx, c, K, vec) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 128 / STEP; j++) *reinterpret_cast<uint4*>(tile + at(fr + j * STEP, 4 * fv)) = q[j];
        }
        cp_async_commit();
    };

    int tr = static_cast<int>(tiles_y - 1 - blockIdx.x / tiles_x), tc = static_cast<int>(tiles_x - 1 - blockIdx.x % tiles_x);
    int ntr = tr, ntc = tc, turn = 0;
    fetch(tr, tc, buffers);
    const Scale scale = fetch_scale<FMT, kTileThreads>(tscale, given, partial, partials);
    auto body = [&](auto careful) {
    for (unsigned n = blockIdx.x; n < tiles_all; n += gridDim.x, turn ^= 1, tr = ntr, tc = ntc) {
        if (n + gridDim.x < tiles_all) {
            advance(ntr, ntc);
            fetch(ntr, ntc, buffers + (turn ^ 1) * C::TILE_WORDS);
            cp_async_wait<1>();
        } else {
            cp_async_wait<0>();
        }
        __syncthreads();
        const int rows_left = static_cast<int>(rows - tr * 128ll < 128 ? rows - tr * 128ll : 128);       // may be negative: scales only
        const int cols_left = static_cast<int>(K - tc * 128ll < 128 ? K - tc * 128ll : 128);
        const uint32_t* tile = buffers + turn * C::TILE_WORDS;

        // ---- blocks along the rows
        if (rows_left > 0) {
            const int b = threadIdx.x % NB;
            const size_t k2 = tc * 64ull + b * (B / 2);
            uint8_t* to = codes + (tr * 128ull + threadIdx.x / NB) * pitch + k2;
            const bool inside = k2 < pitch;
#pragma unroll
            for (int j = 0; j < 128 * NB / kTileThreads; j++) {
                const int r = threadIdx.x / NB + j * (kTileThreads / NB);
                uint32_t w[BW];
#pragma unroll
                for (int i = 0; i < BW; i += 4) *reinterpret_cast<uint4*>(w + i) = *reinterpret_cast<const uint4*>(tile + at(r, b * BW + i));
                float v[B];
                unpack<T, B>(w, v);
                uint32_t c[B / 8];
                sc[(b >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (b & 3)] = static_cast<uint8_t>(encode_block<T, FMT, decltype(careful)::value>(v, magnitude<B>(v), scale, c));
                if (inside && r < rows_left) store_codes<B>(to + static_cast<size_t>(j * (kTileThreads / NB)) * pitch, c);
            }
        }
        // ---- blocks along the columns: a warp takes 8 words x 4 row blocks; where that makes fewer tasks than warps, each
        // of a word's two columns is a task
        if constexpr (COLS) {
            constexpr int TASKS = (W / 8) * (NB / 4), SPLIT = TASKS < kTileThreads / 32 ? CPW : 1;
            const int lane = threadIdx.x & 31, g = lane >> 3;
#pragma unroll 1
            for (int i = threadIdx.x >> 5; i < TASKS * SPLIT; i += kTileThreads / 32) {
                const int task = i % TASKS, h0 = SPLIT > 1 ? i / TASKS : 0;
                const int word = (task % (W / 8)) * 8 + (lane & 7), rb = (task / (W / 8)) * 4 + g;
                uint32_t raw[B];
                const uint32_t* from = tile + at(rb * B, word);
#pragma unroll
                for (int j = 0; j < B; j++) raw[j] = from[j * W];
                const size_t k2 = tr * 64ull + rb * (B / 2);
                uint8_t* to = codes_t + (tc * 128ull + word * CPW) * pitch_t + k2;
                const bool inside = k2 < pitch_t;
#pragma unroll
                for (int h = 0; h < CPW / SPLIT; h++) {
                    const int half = SPLIT > 1 ? h0 : h, col = word * CPW + half;
                    float v[B];
#pragma unroll
                    for (int j = 0; j < B; j++) {
                        if constexpr (CPW == 1) v[j] = __uint_as_float(raw[j]);
                        else if constexpr (std::is_same_v<T, __nv_bfloat16>) v[j] = __uint_as_float(half ? raw[j] & 0xFFFF0000u : raw[j] << 16);
                        else v[j] = __half2float(__ushort_as_half(static_cast<unsigned short>(half ? raw[j] >> 16 : raw[j])));
                    }
                    uint32_t c[B / 8];
                    sc_t[(rb >> 2) * 512 + (col & 31) * 16 + (col >> 5) * 4 + (rb & 3)] = static_cast<uint8_t>(encode_block<T, FMT, decltype(careful)::value>(v, magnitude<B>(v), scale, c));
                    if (inside && col < cols_left) store_codes<B>(to + (half ? pitch_t : 0), c);
                }
            }
        }
        __syncthreads();
        // ---- whole scale tiles
        constexpr int VECS = NB / 4 * 32;
        if (threadIdx.x < VECS) {
            if (rows_left > 0)
                *reinterpret_cast<uint4*>(scales + (static_cast<size_t>(tr) * scale_tiles_per_row(FMT, K) + tc * (NB / 4)) * TILE_BYTES + threadIdx.x * 16) =
                    reinterpret_cast<const uint4*>(sc)[threadIdx.x];
        } else if (COLS && threadIdx.x < 2 * VECS) {
            const int i = threadIdx.x - VECS;
            if (cols_left > 0)
                *reinterpret_cast<uint4*>(scales_t + (static_cast<size_t>(tc) * scale_tiles_per_row(FMT, rows) + tr * (NB / 4)) * TILE_BYTES + i * 16) =
                    reinterpret_cast<const uint4*>(sc_t)[i];
        }
    }
    };
    if (FMT == RDB_FP4_NVFP4 && (scale.move != 1.0f || !partial)) body(std::true_type());
    else body(std::false_type());
}

// Both directions for x on 16-byte boundaries.  Persistent blocks with a ring of tiles - 128 rows of four blocks - that TMA
// boxes of 128 bytes x 128 rows fill (SWIZZLE_128B: 16-byte chunk c of row r at c ^ r % 8).  Two groups of four warps take
// alternate tiles; the warp that is last to finish one requests the next into its place, and nothing else holds the warps
// together (a ninth warp that only requested tiles cost the others a quarter of their registers).  A thread makes the four
// blocks of one row, or of the one or two columns in a word: their scale bytes are a whole scale word, their codes whole
// 32-byte stores, and no data passes between threads.  Bank conflicts: along a row the 8 lanes of a 16-byte phase hold 8
// rows, whose chunks the swizzle spreads; along the columns the 32 lanes read the 32 words of one row.
template <class T, int FMT>
struct BothCfg {
    static constexpr int B = Format<FMT>::BLOCK, BW = B * sizeof(T) / 4, CPW = 4 / sizeof(T);
    static constexpr int COLS = 4 * B;                              // columns of a tile
    static constexpr int BOXES = COLS * sizeof(T) / 128, BOX_BYTES = 128 * 128;
    static constexpr int GROUPS = 128 / COLS;                       // scale words of a column in a tile: 2 or 1
    static constexpr int STAGE = BOXES * BOX_BYTES;
    // an even ring: the groups take alternate tiles, and only with a slot of its own does a group wait for consecutive
    // completions of a barrier (a parity wait cannot tell completion n from n + 2)
    static constexpr int STAGES = STAGE == 16384 ? 4 : 2;
    static constexpr int PER_SM = STAGE == 65536 ? 1 : 2;
    static constexpr int SMEM = 1024 + STAGES * STAGE;
};
constexpr int kBothThreads = 256;

// 32 bytes of codes at byte `at` of a row of `pitch` bytes (a multiple of 16), as far as they lie in it.  wide: rows start
// on 32-byte boundaries.
__device__ __forceinline__ void store32(uint8_t* p, const uint32_t* c, size_t at, size_t pitch, bool wide) {
    if (wide) {
        if (at < pitch) stg32(p, c);
    } else {
        if (at < pitch) *reinterpret_cast<uint4*>(p) = make_uint4(c[0], c[1], c[2], c[3]);
        if (at + 16 < pitch) *reinterpret_cast<uint4*>(p + 16) = make_uint4(c[4], c[5], c[6], c[7]);
    }
}

// 4096 x 14336 bf16 takes 34 us in MXFP4 and 48 to 50 in NVFP4 (28 at the copy rate).  NVFP4, with two scales in 32 elements
// and a division for each, is bound by instructions: without loads and stores 43 us of 48 remain (MXFP4 26 of 37), issue
// slots are 58 % busy.  Two CTAs of 127 registers per SM; three of 80 took 74 us where two took 50, both measured cold.
template <class T, int FMT>
__global__ void __launch_bounds__(kBothThreads, BothCfg<T, FMT>::PER_SM)
quantize_both_kernel(const __grid_constant__ CUtensorMap tm, int rows, int K, unsigned tiles_x, unsigned tiles_all, float* tscale, const float* given, const uint32_t* partial,
                     int partials, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, uint8_t* __restrict__ codes_t,
                     uint8_t* __restrict__ scales_t, int* status) {
    using C = BothCfg<T, FMT>;
    constexpr int B = C::B, BW = C::BW, CPW = C::CPW, COLS = C::COLS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t bars[C::STAGES];
    __shared__ unsigned finished[C::STAGES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full0 = smem_u32(bars);
    // tiles n = blockIdx.x, + gridDim.x, ... counted from the last one (the maximum's pass read those last)
    auto request = [&](unsigned n, int s) {
        const unsigned id = tiles_all - 1 - n, tr = id / tiles_x, tc = id - tr * tiles_x;
        const uint64_t pol = l2_policy_evict_first();
        mbar_arrive_expect_tx(full0 + 8 * s, C::STAGE);
#pragma unroll
        for (int b = 0; b < C::BOXES; b++)
            tma_load_2d(smem_u32(smem) + s * C::STAGE + b * C::BOX_BYTES, &tm, tc * COLS + b * (128 / static_cast<int>(sizeof(T))), tr * 128, full0 + 8 * s, pol);
    };
    if (threadIdx.x == 0) {
        prefetch_tensormap(&tm);
        for (int i = 0; i < C::STAGES; i++) {
            mbar_init(full0 + 8 * i, 1);
            finished[i] = 0;
        }
        fence_barrier_init();
        pdl_wait_prior();
        for (int i = 0; i < C::STAGES && blockIdx.x + i * gridDim.x < tiles_all; i++) request(blockIdx.x + i * gridDim.x, i);
    }
    __syncthreads();
    start_after_prior();
    const Scale scale = fetch_scale<FMT, kBothThreads>(tscale, given, partial, partials);

    const size_t pitch = row_bytes(K), pitch_t = row_bytes(rows);
    const bool wide = ((reinterpret_cast<uintptr_t>(codes) | pitch) & 31) == 0, wide_t = ((reinterpret_cast<uintptr_t>(codes_t) | pitch_t) & 31) == 0;
    const int tiles_k = scale_tiles_per_row(FMT, K), tiles_r = scale_tiles_per_row(FMT, rows);
    const int group = warp >> 2, q = warp & 3;
    auto body = [&](auto careful) {
        // four blocks of row r of the tile
        auto along_row = [&](const uint8_t* tile, unsigned tr, unsigned tc, int r) {
            const long long row = tr * 128ll + r;
            const uint8_t* line = tile + r * 128;
            const uint32_t turn = (r & 7) << 4;
            uint8_t* to = codes + row * pitch + tc * (COLS / 2ull);
            const bool exists = row < rows;
            uint32_t word = 0;
#pragma unroll 1
            for (int k2 = 0; k2 < COLS / 2; k2 += 32) {             // 32 bytes of codes: four blocks of 16, or two of 32
                uint32_t c[8];
#pragma unroll
                for (int b = 0; b < 64 / B; b++) {
                    uint32_t w[BW];
#pragma unroll
                    for (int i = 0; i < BW; i += 4) {
                        const int at = k2 * 2 * static_cast<int>(sizeof(T)) + (b * BW + i) * 4;
                        *reinterpret_cast<uint4*>(w + i) = *reinterpret_cast<const uint4*>(line + at / 128 * C::BOX_BYTES + ((at % 128) ^ turn));
                    }
                    float v[B];
                    unpack<T, B>(w, v);
                    // the four scale bytes come in from the top
                    word = word >> 8 | encode_block<T, FMT, decltype(careful)::value>(v, magnitude<B>(v), scale, c + b * (B / 8)) << 24;
                }
                if (exists) store32(to + k2, c, tc * (COLS / 2ull) + k2, pitch, wide);
            }
            if (exists) *reinterpret_cast<uint32_t*>(scales + scale_word(row, tc, tiles_k)) = word;
        };
        // four blocks of each column in word `lane` of a box; g: which 4 B rows
        auto along_columns = [&](const uint8_t* tile, unsigned tr, unsigned tc, int box, int g) {
            const uint8_t* from = tile + box * C::BOX_BYTES + g * (COLS * 128);
            const long long col = tc * static_cast<long long>(COLS) + box * (128 / static_cast<int>(sizeof(T))) + lane * CPW;
            const size_t k0 = tr * 64ull + g * (COLS / 2);
            uint8_t* to = codes_t + col * pitch_t + k0;
            uint32_t word[CPW];
#pragma unroll
            for (int h = 0; h < CPW; h++) word[h] = 0;
#pragma unroll 1
            for (int k2 = 0; k2 < COLS / 2; k2 += 32) {
                uint32_t c[CPW][8];
#pragma unroll
                for (int b = 0; b < 64 / B; b++) {
                    uint32_t raw[B];
#pragma unroll
                    for (int j = 0; j < B; j++) raw[j] = *reinterpret_cast<const uint32_t*>(from + (2 * k2 + b * B + j) * 128 + ((lane * 4) ^ ((j & 7) << 4)));
#pragma unroll
                    for (int h = 0; h < CPW; h++) {
                        float v[B];
#pragma unroll
                        for (int j = 0; j < B; j++) {
                            if constexpr (CPW == 1) v[j] = __uint_as_float(raw[j]);
                            else if constexpr (std::is_same_v<T, __nv_bfloat16>) v[j] = __uint_as_float(h ? raw[j] & 0xFFFF0000u : raw[j] << 16);
                            else v[j] = __half2float(__ushort_as_half(static_cast<unsigned short>(h ? raw[j] >> 16 : raw[j])));
                        }
                        word[h] = word[h] >> 8 | encode_block<T, FMT, decltype(careful)::value>(v, magnitude<B>(v), scale, c[h] + b * (B / 8)) << 24;
                    }
                }
#pragma unroll
                for (int h = 0; h < CPW; h++)
                    if (col + h < K) store32(to + h * pitch_t + k2, c[h], k0 + k2, pitch_t, wide_t);
            }
#pragma unroll
            for (int h = 0; h < CPW; h++)
                if (col + h < K) *reinterpret_cast<uint32_t*>(scales_t + scale_word(col + h, tr * C::GROUPS + g, tiles_r)) = word[h];
        };

        int i = 0;
        for (unsigned n = blockIdx.x; n < tiles_all; n += gridDim.x, i++) {
            if ((i & 1) != group) continue;
            const int s = i % C::STAGES;
            if (!mbar_wait(full0 + 8 * s, (i / C::STAGES) & 1)) { report_timeout(status); break; }
            const unsigned id = tiles_all - 1 - n, tr = id / tiles_x, tc = id - tr * tiles_x;
            const uint8_t* tile = smem + s * C::STAGE;
            if constexpr (CPW == 2) {                               // two warps take the rows, two the columns
                if (q < 2) {
                    along_row(tile, tr, tc, q * 64 + lane);
                    along_row(tile, tr, tc, q * 64 + 32 + lane);
                } else {
                    along_columns(tile, tr, tc, C::BOXES == 2 ? q - 2 : 0, C::BOXES == 2 ? 0 : q - 2);
                }
            } else {                                                // each warp a quarter of either
                along_row(tile, tr, tc, q * 32 + lane);
                along_columns(tile, tr, tc, C::BOXES == 4 ? q : q & 1, C::BOXES == 4 ? 0 : q >> 1);
            }
            __syncwarp();
            if (lane == 0) {
                __threadfence_block();
                if ((atomicAdd(finished + s, 1u) & 3u) == 3u) {     // all four warps have read the tile
                    __threadfence_block();
                    if (tiles_all - n > C::STAGES * gridDim.x) request(n + C::STAGES * gridDim.x, s);
                }
            }
            __syncwarp();
        }
    };
    if (FMT == RDB_FP4_NVFP4 && (scale.move != 1.0f || !partial)) body(std::true_type());
    else body(std::false_type());
}

// Eight codes -> eight halves (exact).
__device__ __forceinline__ void decode8(uint32_t w, __half2* h) {
    uint32_t o[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]) : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = *reinterpret_cast<const __half2*>(o + i);
}

// Scale byte -> the value that multiplies e2m1, without the tensor scale.
template <int FMT>
__device__ __forceinline__ float scale_value(uint32_t byte) {
    if constexpr (FMT == RDB_FP4_MXFP4) {
        return byte == 0xFF ? __uint_as_float(0x7FFFFFFFu) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
    } else {
        __nv_fp8_e4m3 s8;
        s8.__x = static_cast<__nv_fp8_storage_t>(byte);
        return static_cast<float>(s8);
    }
}

template <class T, int FMT>
__device__ __forceinline__ void decode_block(uint32_t codes, uint32_t scale, float t, T* v) {
    const float f = scale_value<FMT>(scale);
    __half2 h[4];
    decode8(codes, h);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 e = __half22float2(h[i]);
        v[2 * i] = from_f32<T>(e.x * f * t);
        v[2 * i + 1] = from_f32<T>(e.y * f * t);
    }
}

// A warp takes 256 elements (8 per lane) of the rows r, r + 32, r + 64, r + 96 of a 128-row tile: their scale words are one
// 16-byte load.  element * scale is exact in fp32, the tensor scale's product rounds, the output type rounds again.
// vec: rows of the output start on boundaries of 8 elements; else the values pass through shared memory, so that neighbouring
// lanes store neighbouring elements.  Bound by HBM: 4096 x 14336 takes 25 us to bf16, 43 to fp32.
template <class T, int FMT>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                              const float* tscale, int rows, int K, int vec, T* __restrict__ out) {
    constexpr int B = Format<FMT>::BLOCK;
    start_after_prior();
    __shared__ __align__(16) T stage[kThreads / 32][256];
    const float t = FMT == RDB_FP4_NVFP4 ? *tscale : 1.0f;
    const size_t pitch = row_bytes(K);
    const int tiles = scale_tiles_per_row(FMT, K);
    const int lane = threadIdx.x & 31;
    const long long k0 = blockIdx.x * 256ll;
    const int octets = static_cast<int>((rows + 127ll) / 128 * 4);
    for (int o = blockIdx.y; o < octets; o += gridDim.y) {
        const int r0 = (o >> 2) * 128 + (o & 3) * 8 + (threadIdx.x >> 5);
        if (r0 >= rows) continue;
        if (vec) {
            const long long k = k0 + 8 * lane;
            if (k >= K) continue;
            uint32_t c[4];
#pragma unroll
            for (int j = 0; j < 4; j++) c[j] = r0 + 32 * j < rows ? __ldg(reinterpret_cast<const uint32_t*>(codes + (r0 + 32 * j) * pitch + k / 2)) : 0;
            const int b = static_cast<int>(k / B);
            const uint4 s4 = __ldg(reinterpret_cast<const uint4*>(scales + scale_word(r0, b >> 2, tiles)));
            const uint32_t s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = r0 + 32 * j;
                if (r >= rows) break;
                alignas(16) T v[8];
                decode_block<T, FMT>(c[j], (s[j] >> (8 * (b & 3))) & 0xFF, t, v);
                T* p = out + r * static_cast<size_t>(K) + k;
                if constexpr (sizeof(T) == 2) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
                else stg32(p, reinterpret_cast<const uint32_t*>(v));
            }
        } else {
            T* mine = stage[threadIdx.x >> 5];
            const long long k = k0 + 8 * lane;
            const int b = static_cast<int>(k / B);
            const uint4 s4 = k < K ? __ldg(reinterpret_cast<const uint4*>(scales + scale_word(r0, b >> 2, tiles))) : make_uint4(0, 0, 0, 0);
            const uint32_t s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = r0 + 32 * j;
                if (r >= rows) break;
                const uint32_t c = k < K ? __ldg(reinterpret_cast<const uint32_t*>(codes + r * pitch + k / 2)) : 0;
                alignas(16) T v[8];
                decode_block<T, FMT>(c, (s[j] >> (8 * (b & 3))) & 0xFF, t, v);
#pragma unroll
                for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; i++) reinterpret_cast<uint4*>(mine + 8 * lane)[i] = reinterpret_cast<const uint4*>(v)[i];
                __syncwarp();
                T* to = out + r * static_cast<size_t>(K) + k0;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (k0 + 32 * i + lane < K) to[32 * i + lane] = mine[32 * i + lane];
                __syncwarp();
            }
        }
    }
}

// Every kernel of this file waits for its predecessor before it touches memory: the early start only hides the launch.
static int launch(const void* kernel, dim3 grid, int threads, int smem, void** args, cudaStream_t stream, int cluster = 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    if (cudaLaunchKernelExC(&cfg, kernel, args) != cudaSuccess) { cudaGetLastError(); return RDB_CUDA_ERROR; }
    return RDB_SUCCESS;
}

// Grid of the kernels that walk octets of rows (grid.y strides).
static dim3 octet_grid(int rows, long long columns) {
    long long y = rows < 32 ? (rows + 7) / 8 : (static_cast<long long>(rows) + 127) / 128 * 4;
    return dim3(static_cast<unsigned>(columns), static_cast<unsigned>(y < 65535 ? y : 65532));
}

template <class T, int FMT, bool COLS>
static int launch_tiles(int rows, int K, void** args, unsigned* tiles_x, unsigned* tiles_all, int sm_count, cudaStream_t stream) {
    using C = TileCfg<T, FMT>;
    static bool attr_set[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return RDB_CUDA_ERROR;
    auto kernel = quantize_tile_kernel<T, FMT, COLS>;
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return RDB_CUDA_ERROR;
        attr_set[dev] = true;
    }
    // scales are filled up to 256 elements along either direction that is quantised
    const long long x = (static_cast<long long>(K) + 255) / 256 * 2;
    const long long y = COLS ? (static_cast<long long>(rows) + 255) / 256 * 2 : (static_cast<long long>(rows) + 127) / 128;
    if (x * y > 0x7FFFFFFFll) return RDB_SIZE_ABOVE_LIMIT;
    *tiles_x = static_cast<unsigned>(x);
    *tiles_all = static_cast<unsigned>(x * y);
    const unsigned grid = static_cast<unsigned>(sm_count * C::PER_SM);
    return launch(reinterpret_cast<const void*>(kernel), dim3(*tiles_all < grid ? *tiles_all : grid), kTileThreads, C::SMEM, args, stream);
}

template <class T, int FMT>
static int launch_both(const T* x, long long ldx, int rows, int K, float* tscale, const float* given, uint32_t* partial, int partials, uint8_t* codes, uint8_t* scales,
                       uint8_t* codes_t, uint8_t* scales_t, const DeviceInfo* info, cudaStream_t stream) {
    using C = BothCfg<T, FMT>;
    static bool attr_set[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return RDB_CUDA_ERROR;
    auto kernel = quantize_both_kernel<T, FMT>;
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return RDB_CUDA_ERROR;
        attr_set[dev] = true;
    }
    // scales are filled up to 256 elements along either direction
    const long long tx = (static_cast<long long>(K) + 255) / 256 * (256 / C::COLS), all = tx * ((static_cast<long long>(rows) + 255) / 256 * 2);
    if (all > 0x7FFFFFFFll) return RDB_SIZE_ABOVE_LIMIT;
    CUtensorMap tm;
    const int r = make_tmap_2d(&tm, x, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, sizeof(T), rows, K,
                               static_cast<uint64_t>(ldx) * sizeof(T), 128 / sizeof(T), 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r != RDB_SUCCESS) return r;
    unsigned tiles_x = static_cast<unsigned>(tx), tiles_all = static_cast<unsigned>(all);
    int* status = info->status_dev;
    void* args[] = {&tm, &rows, &K, &tiles_x, &tiles_all, &tscale, &given, &partial, &partials, &codes, &scales, &codes_t, &scales_t, &status};
    const unsigned grid = static_cast<unsigned>(info->sm_count * C::PER_SM);
    return launch(reinterpret_cast<const void*>(kernel), dim3(tiles_all < grid ? tiles_all : grid), kBothThreads, C::SMEM, args, stream);
}

template <class T, int FMT>
static int quantize(const void* x_, long long ldx, int rows, int K, float* tscale, const float* given, uint8_t* codes, uint8_t* scales,
                    uint8_t* codes_t, uint8_t* scales_t, float* workspace, const DeviceInfo* info, cudaStream_t stream) {
    constexpr int B = Format<FMT>::BLOCK;
    const T* x = static_cast<const T*>(x_);
    const size_t row = static_cast<size_t>(ldx) * sizeof(T);
    const bool by32 = (reinterpret_cast<uintptr_t>(x) & 31u) == 0 && row % 32 == 0, by16 = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && row % 16 == 0;
    const bool direct = !codes_t && by16 && K % B == 0;      // a thread can take whole blocks straight from memory
    const long long all_blocks = 4ll * scale_tiles_per_row(FMT, K) * rows;
    // Up to 2 blocks a thread of 8 CTAs: a launch and a pass over x less (bf16, 8 x 4096: 2.6 us against 3.4 in two
    // launches, 32 x 4096: 3.2 against 3.5).  Beyond that one cluster is slower than all SMs: 32 x 8192 took 4.6 against 3.6.
    if (FMT == RDB_FP4_NVFP4 && !given && direct && all_blocks <= 2ll * kSmallCluster * kSmallThreads) {
        void* args[] = {&x, &ldx, &rows, &K, &tscale, &codes, &scales};
        int ctas = 1;
        while (ctas < kSmallCluster && all_blocks > static_cast<long long>(ctas) * kSmallThreads) ctas *= 2;
        return launch(all_blocks <= static_cast<long long>(ctas) * kSmallThreads ? reinterpret_cast<const void*>(quantize_small_kernel<T, 1>)
                                                                                 : reinterpret_cast<const void*>(quantize_small_kernel<T, 2>),
                      dim3(ctas), kSmallThreads, 0, args, stream, ctas);
    }
    uint32_t* partial = nullptr;
    int partials = 0;
    if (FMT == RDB_FP4_NVFP4 && !given) {
        partial = reinterpret_cast<uint32_t*>(workspace);
        const long long units = ((K - 1) / kAmaxStretch + 1ll) * rows, blocks = (units + 7) / 8;
        partials = static_cast<int>(blocks < kAmaxBlocks ? blocks : kAmaxBlocks);
        if (partials > info->sm_count * 6) partials = info->sm_count * 6;
        void* args[] = {&x, &ldx, &rows, &K, &partial};
        const int r = launch(reinterpret_cast<const void*>(amax_kernel<T>), dim3(partials), kThreads, 0, args, stream);
        if (r != RDB_SUCCESS) return r;
    }
    if (direct) {
        void* args[] = {&x, &ldx, &rows, &K, &tscale, &given, &partial, &partials, &codes, &scales};
        dim3 grid = octet_grid(rows, (4ll * scale_tiles_per_row(FMT, K) + 31) / 32);
        // what a block does once (the partial maxima) is shared by several octets where there are blocks enough: 16 per SM
        if (partial) {
            const unsigned enough = (16u * info->sm_count + grid.x - 1) / grid.x;
            if (grid.y > 2 * enough) grid.y = enough;
        }
        return launch(by32 ? reinterpret_cast<const void*>(quantize_rows_kernel<T, FMT, 32>) : reinterpret_cast<const void*>(quantize_rows_kernel<T, FMT, 16>),
                      grid, kThreads, 0, args, stream);
    }
    if (codes_t && by16 && static_cast<unsigned long long>(row) < (1ull << 40))
        return launch_both<T, FMT>(x, ldx, rows, K, tscale, given, partial, partials, codes, scales, codes_t, scales_t, info, stream);
    int vec = by16;
    unsigned tiles_x = 0, tiles_all = 0;
    void* args[] = {&x, &ldx, &rows, &K, &vec, &tiles_x, &tiles_all, &tscale, &given, &partial, &partials, &codes, &scales, &codes_t, &scales_t};
    return codes_t ? launch_tiles<T, FMT, true>(rows, K, args, &tiles_x, &tiles_all, info->sm_count, stream) : launch_tiles<T, FMT, false>(rows, K, args, &tiles_x, &tiles_all, info->sm_count, stream);
}

template <class T>
static int dequantize(const uint8_t* codes, const uint8_t* scales, const float* tscale, int format, int rows, int K, void* out_, cudaStream_t stream) {
    T* out = static_cast<T*>(out_);
    int vec = (reinterpret_cast<uintptr_t>(out) & (8 * sizeof(T) - 1)) == 0 && K % 8 == 0;     // 8 elements to a store
    void* args[] = {&codes, &scales, &tscale, &rows, &K, &vec, &out};
    return launch(format == RDB_FP4_NVFP4 ? reinterpret_cast<const void*>(dequantize_kernel<T, RDB_FP4_NVFP4>) : reinterpret_cast<const void*>(dequantize_kernel<T, RDB_FP4_MXFP4>),
                  octet_grid(rows, (static_cast<long long>(K) + 255) / 256), kThreads, 0, args, stream);
}

static int check(int type, int rows, int K, int format) {
    if (rows < 1 || K < 1) return RDB_BAD_SHAPE;
    if (format != RDB_FP4_MXFP4 && format != RDB_FP4_NVFP4) return RDB_INVALID_CONFIG;
    if (type != RDB_TYPE_BF16 && type != RDB_TYPE_FP16 && type != RDB_TYPE_FP32) return RDB_INVALID_CONFIG;
    if (rows > MAX_EXTENT || K > MAX_EXTENT) return RDB_SIZE_ABOVE_LIMIT;
    return RDB_SUCCESS;
}

}  // namespace fp4
}  // namespace rdb

extern "C" {

size_t rdb_fp4_row_bytes(int K) { return K < 1 ? 0 : rdb::fp4::row_bytes(K); }

size_t rdb_fp4_scale_bytes(int format, int rows, int K) {
    if (rdb::fp4::check(RDB_TYPE_BF16, rows, K, format) != RDB_SUCCESS) return 0;
    return rdb::fp4::scale_bytes(format, rows, K);
}

int rdb_quantize_fp4(const void* x, int x_type, long long ldx, int rows, int K, int format, float* tensor_scale, const float* given_scale,
                     uint8_t* codes, uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, float* workspace, void* stream) {
    using namespace rdb::fp4;
    const int ok = check(x_type, rows, K, format);
    if (ok != RDB_SUCCESS) return ok;
    if (ldx < K) return RDB_BAD_SHAPE;
    if (!x || !codes || !scales || (codes_t == nullptr) != (scales_t == nullptr)) return RDB_INVALID_CONFIG;
    if (format == RDB_FP4_NVFP4 ? !tensor_scale || (!given_scale && !workspace) : tensor_scale || given_scale) return RDB_INVALID_CONFIG;
    const uintptr_t size = x_type == RDB_TYPE_FP32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % size || !rdb::aligned16(codes) || !rdb::aligned16(scales) || !rdb::aligned16(codes_t) ||
        !rdb::aligned16(scales_t) || (reinterpret_cast<uintptr_t>(tensor_scale) & 3u) || (reinterpret_cast<uintptr_t>(given_scale) & 3u) || (reinterpret_cast<uintptr_t>(workspace) & 3u))
        return RDB_BAD_ALIGNMENT;
    int err = 0;
    rdb::DeviceInfo* info = rdb::device_info(&err);
    if (!info) return err;
    auto s = static_cast<cudaStream_t>(stream);
#define RDB_QUANTIZE(T, F) quantize<T, F>(x, ldx, rows, K, tensor_scale, given_scale, codes, scales, codes_t, scales_t, workspace, info, s)
    if (format == RDB_FP4_NVFP4)
        return x_type == RDB_TYPE_BF16 ? RDB_QUANTIZE(__nv_bfloat16, RDB_FP4_NVFP4) : x_type == RDB_TYPE_FP16 ? RDB_QUANTIZE(__half, RDB_FP4_NVFP4) : RDB_QUANTIZE(float, RDB_FP4_NVFP4);
    return x_type == RDB_TYPE_BF16 ? RDB_QUANTIZE(__nv_bfloat16, RDB_FP4_MXFP4) : x_type == RDB_TYPE_FP16 ? RDB_QUANTIZE(__half, RDB_FP4_MXFP4) : RDB_QUANTIZE(float, RDB_FP4_MXFP4);
#undef RDB_QUANTIZE
}

int rdb_dequantize_fp4(const uint8_t* codes, const uint8_t* scales, const float* tensor_scale, int format, int rows, int K, void* out,
                       int out_type, void* stream) {
    using namespace rdb::fp4;
    const int ok = check(out_type, rows, K, format);
    if (ok != RDB_SUCCESS) return ok;
    if (!codes || !scales || !out || (format == RDB_FP4_NVFP4 && !tensor_scale)) return RDB_INVALID_CONFIG;
    if (!rdb::aligned16(codes) || !rdb::aligned16(scales) || reinterpret_cast<uintptr_t>(out) % (out_type == RDB_TYPE_FP32 ? 4 : 2) ||
        (reinterpret_cast<uintptr_t>(tensor_scale) & 3u))
        return RDB_BAD_ALIGNMENT;
    auto s = static_cast<cudaStream_t>(stream);
    if (out_type == RDB_TYPE_BF16) return dequantize<__nv_bfloat16>(codes, scales, tensor_scale, format, rows, K, out, s);
    if (out_type == RDB_TYPE_FP16) return dequantize<__half>(codes, scales, tensor_scale, format, rows, K, out, s);
    return dequantize<float>(codes, scales, tensor_scale, format, rows, K, out, s);
}

}  // extern "C"
