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
#include "fp8_codec.cuh"
#include "host_util.h"
#include "ptx.cuh"

namespace rdb {
namespace fp4 {

constexpr int kThreads = 256;
constexpr int kAmaxBlocks = RDB_FP4_WORKSPACE_FLOATS;    // upper bound of the first pass's grid: one partial maximum each
constexpr uint32_t kInf = 0x7F800000u;

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

// The words of a vector load as floats.
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

// N elements from p, of which the first `valid` exist; the others read as zero.
template <class T, int N>
__device__ __forceinline__ void load_block(const T* p, int valid, bool vec, float* v) {
    if (vec && valid >= N) {
        constexpr int WORDS = N * sizeof(T) / 4;
        uint32_t w[WORDS];
#pragma unroll
        for (int i = 0; i < WORDS; i += 8) ldg32(reinterpret_cast<const uint32_t*>(p) + i, w + i);
        unpack<T, N>(w, v);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = i < valid ? to_f32(p[i]) : 0.0f;
    }
}

// Largest magnitude as fp32 bits: non-negative floats order like integers, infinities and NaNs above every number.
template <int N>
__device__ __forceinline__ uint32_t magnitude(const float* v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; i++) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
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

// x / s rounded to fp32 like the IEEE division, for a divisor shared by a block (BlockDivisor's correction step).  bf16
// numerators need one step; wider ones a second, whose starting point is within one unit of the quotient's last place -
// the first product can miss by one and a half.
template <class T>
__device__ __forceinline__ void divide8(const ar::BlockDivisor& d, const float* x, float* q) {
    d.div8(x, q);
    if constexpr (!std::is_same_v<T, __nv_bfloat16>) {
        if (d.fast) {
#pragma unroll
            for (int i = 0; i < 8; i++) q[i] = copysignf(__fmaf_rn(__fmaf_rn(-q[i], d.s, x[i]), d.inv, q[i]), x[i]);
        }
    }
}

// One block: v[BLOCK] -> BLOCK / 8 words of codes, returns the scale byte.  t, t6: the tensor scale and 6 t (NVFP4).
template <class T, int FMT>
__device__ __forceinline__ uint32_t encode_block(const float* v, uint32_t amax, float t, float t6, uint32_t* codes) {
    constexpr int B = Format<FMT>::BLOCK;
    uint32_t byte;
    if constexpr (FMT == RDB_FP4_MXFP4) {
        // the exponent field of the largest magnitude is floor(log2) + 127 (0 for subnormals, whose clamp is 0 too)
        const uint32_t e = amax >> 23;
        byte = e >= 2 ? e - 2 : 0;
        const float inv = __uint_as_float((254 - byte) << 23);       // 2^(127 - byte), exact products below
#pragma unroll
        for (int g = 0; g < B / 8; g++) {
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; i++) q[i] = v[8 * g + i] * inv;
            codes[g] = pack8(q);
        }
        if (amax >= kInf) byte = 0xFF;
    } else {
        byte = __nv_cvt_float_to_fp8(__fdiv_rn(__uint_as_float(amax), t6), __NV_SATFINITE, __NV_E4M3) & 0x7F;
        __nv_fp8_e4m3 s8;
        s8.__x = static_cast<__nv_fp8_storage_t>(byte);
        ar::BlockDivisor d;
        d.set(static_cast<float>(s8) * t);
#pragma unroll
        for (int g = 0; g < B / 8; g++) {
            float q[8];
            divide8<T>(d, v + 8 * g, q);
            codes[g] = byte != 0 ? pack8(q) : 0;
        }
        if (amax >= kInf) byte = 0x7F;
    }
    return byte;
}

// The tensor scale from the first pass's partial maxima (every warp for itself: they are in L2), or the given one.
__device__ __forceinline__ float tensor_scale(const float* given, const uint32_t* partial, int count) {
    if (!partial) return *given;
    uint32_t m = 0;
    for (int i = threadIdx.x & 31; i < count; i += 32) m = max(m, __ldcg(partial + i));
    m = __reduce_max_sync(0xffffffffu, m);
    constexpr float inv = 1.0f / 2688.0f;            // rounded to fp32 before it multiplies: part of the definition
    return m == 0 ? 1.0f : fmaxf(__fmul_rn(__uint_as_float(m), inv), 1.17549435e-38f);
}

template <class T>
__global__ void __launch_bounds__(kThreads) amax_kernel(const T* __restrict__ x, long long ldx, int rows, int K, bool vec,
                                                        uint32_t* __restrict__ partial) {
    __shared__ uint32_t warp_max[kThreads / 32];
    pdl_launch_dependents();
    pdl_wait_prior();
    constexpr int N = 32 / sizeof(T);
    const long long per_row = (K + N - 1) / N, chunks = per_row * rows;
    uint32_t m = 0;
    for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i < chunks; i += static_cast<long long>(gridDim.x) * kThreads) {
        const long long r = i / per_row;
        const int k = static_cast<int>(i - r * per_row) * N;
        float v[N];
        load_block<T, N>(x + r * ldx + k, K - k, vec, v);
        uint32_t a = magnitude<N>(v);
        if (a >= kInf) {                     // only then element by element: the finite ones count
            a = 0;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const uint32_t b = __float_as_uint(v[j]) & 0x7FFFFFFFu;
                if (b < kInf) a = max(a, b);
            }
        }
        m = max(m, a);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
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

// Blocks along the rows: one thread per block; the four threads of a scale word join their bytes.
template <class T, int FMT>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, long long ldx, int rows, int K, bool vec,
                                                                 float* tscale, const uint32_t* partial, int partials,
                                                                 uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    constexpr int B = Format<FMT>::BLOCK;
    pdl_launch_dependents();
    pdl_wait_prior();
    float t = 1.0f, t6 = 6.0f;
    if constexpr (FMT == RDB_FP4_NVFP4) {
        t = tensor_scale(tscale, partial, partials);
        t6 = t * 6.0f;
        if (partial && blockIdx.x == 0 && threadIdx.x == 0) *tscale = t;
    }
    const size_t pitch = row_bytes(K);
    const int tiles = scale_tiles_per_row(FMT, K), per_row = 4 * tiles;     // a multiple of 8: words never straddle rows
    const long long total = static_cast<long long>(rows) * per_row;
    for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i - (threadIdx.x & 31) < total;
         i += static_cast<long long>(gridDim.x) * kThreads) {
        uint32_t byte = 0;
        const long long r = i / per_row;
        const int b = static_cast<int>(i - r * per_row);
        if (i < total && static_cast<size_t>(b) * (B / 2) < pitch) {
            float v[B];
            const int k = b * B;
            load_block<T, B>(x + r * ldx + k, K - k, vec, v);
            uint32_t c[B / 8];
            byte = encode_block<T, FMT>(v, magnitude<B>(v), t, t6, c);
            store_codes<B>(codes + r * pitch + static_cast<size_t>(b) * (B / 2), c);
        }
        uint32_t word = byte << (8 * (threadIdx.x & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 1);
        word |= __shfl_xor_sync(0xffffffffu, word, 2);
        if ((threadIdx.x & 3) == 0 && i < total) *reinterpret_cast<uint32_t*>(scales + scale_word(r, b >> 2, tiles)) = word;
    }
}

// Blocks along the columns: one thread per block of one column of x, i.e. along a row of the transposed tensor.
template <class T, int FMT>
__global__ void __launch_bounds__(kThreads) quantize_cols_kernel(const T* __restrict__ x, long long ldx, int rows, int K,
                                                                 float* tscale, const uint32_t* partial, int partials,
                                                                 uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    constexpr int B = Format<FMT>::BLOCK;
    pdl_launch_dependents();
    pdl_wait_prior();
    float t = 1.0f, t6 = 6.0f;
    if constexpr (FMT == RDB_FP4_NVFP4) {
        t = tensor_scale(tscale, partial, partials);
        t6 = t * 6.0f;
        if (partial && blockIdx.x == 0 && threadIdx.x == 0) *tscale = t;
    }
    const size_t pitch = row_bytes(rows);
    const int tiles = scale_tiles_per_row(FMT, rows);
    const long long total = static_cast<long long>(K) * tiles;              // a thread does the four blocks of a word
    for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * kThreads) {
        const int col = static_cast<int>(i / K);
        const size_t c = i - static_cast<long long>(col) * K;               // neighbours take neighbouring columns
        uint32_t word = 0;
        for (int j = 0; j < 4; j++) {
            const long long r0 = (4ll * col + j) * B;
            if (static_cast<size_t>(r0 / 2) >= pitch) break;
            float v[B];
#pragma unroll
            for (int q = 0; q < B; q++) v[q] = r0 + q < rows ? to_f32(x[(r0 + q) * ldx + c]) : 0.0f;
            uint32_t o[B / 8];
            word |= encode_block<T, FMT>(v, magnitude<B>(v), t, t6, o) << (8 * j);
            store_codes<B>(codes + c * pitch + r0 / 2, o);
        }
        *reinterpret_cast<uint32_t*>(scales + scale_word(c, col, tiles)) = word;
    }
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

__device__ __forceinline__ float element_value(uint32_t code) {
    const uint32_t m = code & 7;
    // exponent field 1..3 -> 2^(e - 1) (1 + m / 2); 0 -> m / 2
    const float a = m < 2 ? 0.5f * m : __uint_as_float(((m >> 1) + 126) << 23 | (m & 1) << 22);
    return code & 8 ? -a : a;
}

template <class T, int FMT>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                              const float* tscale, int rows, int K, T* __restrict__ out) {
    constexpr int B = Format<FMT>::BLOCK;
    pdl_launch_dependents();
    pdl_wait_prior();
    const float t = FMT == RDB_FP4_NVFP4 ? *tscale : 1.0f;
    const size_t pitch = row_bytes(K);
    const int tiles = scale_tiles_per_row(FMT, K);
    const long long per_row = (K + 1) / 2, total = per_row * rows;
    for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * kThreads) {
        const long long r = i / per_row;
        const int k = static_cast<int>(i - r * per_row) * 2, b = k / B;
        const uint32_t c = codes[r * pitch + k / 2];
        const float s = scale_value<FMT>(scales[scale_word(r, b >> 2, tiles) + (b & 3)]);
        T* o = out + r * static_cast<size_t>(K) + k;
        o[0] = from_f32<T>(element_value(c & 15) * s * t);
        if (k + 1 < K) o[1] = from_f32<T>(element_value(c >> 4) * s * t);
    }
}

static int launch(const void* kernel, long long items, long long cap, void** args, cudaStream_t stream, int* grid_out = nullptr) {
    long long blocks = (items + kThreads - 1) / kThreads;
    if (blocks > cap) blocks = cap;
    if (blocks < 1) blocks = 1;
    if (grid_out) *grid_out = static_cast<int>(blocks);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    // every kernel of this file waits for its predecessor before it touches memory: the early start only hides the launch
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelExC(&cfg, kernel, args) != cudaSuccess) { cudaGetLastError(); return RDB_CUDA_ERROR; }
    return RDB_SUCCESS;
}

template <class T, int FMT>
static int quantize(const void* x_, long long ldx, int rows, int K, float* tscale, bool given, uint8_t* codes, uint8_t* scales,
                    uint8_t* codes_t, uint8_t* scales_t, float* workspace, const DeviceInfo* info, cudaStream_t stream) {
    const T* x = static_cast<const T*>(x_);
    bool vec = (reinterpret_cast<uintptr_t>(x) & 31u) == 0 && (static_cast<size_t>(ldx) * sizeof(T)) % 32 == 0;
    const long long cap = info->sm_count * 8ll;
    uint32_t* partial = nullptr;
    int partials = 0;
    if (FMT == RDB_FP4_NVFP4 && !given) {
        partial = reinterpret_cast<uint32_t*>(workspace);
        void* args[] = {&x, &ldx, &rows, &K, &vec, &partial};
        const int per_row = (K + 32 / static_cast<int>(sizeof(T)) - 1) / (32 / static_cast<int>(sizeof(T)));
        const int r = launch(reinterpret_cast<const void*>(amax_kernel<T>), static_cast<long long>(per_row) * rows,
                             cap < kAmaxBlocks ? cap : kAmaxBlocks, args, stream, &partials);
        if (r != RDB_SUCCESS) return r;
    }
    if (codes) {
        void* args[] = {&x, &ldx, &rows, &K, &vec, &tscale, &partial, &partials, &codes, &scales};
        const int r = launch(reinterpret_cast<const void*>(quantize_rows_kernel<T, FMT>), 4ll * scale_tiles_per_row(FMT, K) * rows, cap, args, stream);
        if (r != RDB_SUCCESS) return r;
    }
    if (codes_t) {
        void* args[] = {&x, &ldx, &rows, &K, &tscale, &partial, &partials, &codes_t, &scales_t};
        const int r = launch(reinterpret_cast<const void*>(quantize_cols_kernel<T, FMT>), static_cast<long long>(scale_tiles_per_row(FMT, rows)) * K, cap, args, stream);
        if (r != RDB_SUCCESS) return r;
    }
    return RDB_SUCCESS;
}

template <class T>
static int dequantize(const uint8_t* codes, const uint8_t* scales, const float* tscale, int format, int rows, int K, void* out_,
                      const DeviceInfo* info, cudaStream_t stream) {
    T* out = static_cast<T*>(out_);
    void* args[] = {&codes, &scales, &tscale, &rows, &K, &out};
    return launch(format == RDB_FP4_NVFP4 ? reinterpret_cast<const void*>(dequantize_kernel<T, RDB_FP4_NVFP4>) : reinterpret_cast<const void*>(dequantize_kernel<T, RDB_FP4_MXFP4>),
                  (static_cast<long long>(K) + 1) / 2 * rows, info->sm_count * 8ll, args, stream);
}

static int check(int type, int rows, int K, int format) {
    if (rows < 1 || K < 1) return RDB_BAD_SHAPE;
    if (format != RDB_FP4_MXFP4 && format != RDB_FP4_NVFP4) return RDB_INVALID_CONFIG;
    if (type != RDB_TYPE_BF16 && type != RDB_TYPE_FP16 && type != RDB_TYPE_FP32) return RDB_INVALID_CONFIG;
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

int rdb_quantize_fp4(const void* x, int x_type, long long ldx, int rows, int K, int format, float* tensor_scale, int scale_given,
                     uint8_t* codes, uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, float* workspace, void* stream) {
    using namespace rdb::fp4;
    const int ok = check(x_type, rows, K, format);
    if (ok != RDB_SUCCESS) return ok;
    if (ldx < K) return RDB_BAD_SHAPE;
    if (!x || (!codes && !codes_t) || (codes && !scales) || (codes_t && !scales_t)) return RDB_INVALID_CONFIG;
    if (format == RDB_FP4_NVFP4 && (!tensor_scale || (!scale_given && !workspace))) return RDB_INVALID_CONFIG;
    const uintptr_t size = x_type == RDB_TYPE_FP32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % size || !rdb::aligned16(codes) || !rdb::aligned16(scales) || !rdb::aligned16(codes_t) ||
        !rdb::aligned16(scales_t) || (reinterpret_cast<uintptr_t>(tensor_scale) & 3u) || (reinterpret_cast<uintptr_t>(workspace) & 3u))
        return RDB_BAD_ALIGNMENT;
    int err = 0;
    rdb::DeviceInfo* info = rdb::device_info(&err);
    if (!info) return err;
    auto s = static_cast<cudaStream_t>(stream);
#define RDB_QUANTIZE(T, F) quantize<T, F>(x, ldx, rows, K, tensor_scale, scale_given != 0, codes, scales, codes_t, scales_t, workspace, info, s)
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
    int err = 0;
    rdb::DeviceInfo* info = rdb::device_info(&err);
    if (!info) return err;
    auto s = static_cast<cudaStream_t>(stream);
    if (out_type == RDB_TYPE_BF16) return dequantize<__nv_bfloat16>(codes, scales, tensor_scale, format, rows, K, out, info, s);
    if (out_type == RDB_TYPE_FP16) return dequantize<__half>(codes, scales, tensor_scale, format, rows, K, out, info, s);
    return dequantize<float>(codes, scales, tensor_scale, format, rows, K, out, info, s);
}

}  // extern "C"
