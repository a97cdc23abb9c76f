// Block-scaled tensor-core steps for 4-bit operands: inline PTX around tcgen05.mma kind::mxf4 / kind::mxf4nvf4 and the
// copies that bring scale tiles into TMEM.
#pragma once

#include "fp4.cuh"
#include "ptx.cuh"

namespace rdb {
namespace fp4 {

// Instruction descriptor: e2m1 x e2m1 -> f32, both operands K-major; bit 23 tells powers of two (e8m0) from e4m3 scales.
// Scale id (bits 4-5 for B, 29-30 for A): the byte of a scale word at which the step's scales begin.
template <int FMT>
__host__ __device__ constexpr uint32_t idesc_fp4(int umma_m, int umma_n, int scale_id) {
    return (1u << 7) | (1u << 10) | (FMT == RDB_FP4_MXFP4 ? 1u << 23 : 0u) | (static_cast<uint32_t>(umma_n >> 3) << 17) |
           (static_cast<uint32_t>(umma_m >> 4) << 24) | (static_cast<uint32_t>(scale_id) << 4) | (static_cast<uint32_t>(scale_id) << 29);
}

// The issuing warp runs its loop with all lanes, so that addresses and descriptors stay in uniform registers, and only the
// tcgen05 instructions themselves are predicated by `leader` (one elected lane): a loop inside `if (lane == 0)` has to
// move every operand from the vector registers first, and that was what a stage's issue time went into.

// Descriptors as their low word; the high one is a constant of the layout.
// Operand: 128-byte rows, SWIZZLE_128B, 8-row groups 1024 bytes apart.  Scale tile: 32 rows of 16 bytes, no swizzle, 8-row
// groups 128 bytes apart.
constexpr uint32_t DESC_HI_OPERAND = (1024u >> 4) | (1u << 14) | (2u << 29), DESC_HI_SCALES = (128u >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t desc_lo_operand(uint32_t smem_addr) { return ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_lo_scales(uint32_t smem_addr) { return (smem_addr & 0x3FFFFu) >> 4; }

// 512 bytes -> four TMEM columns, the 32 rows repeated in each of the four lane quadrants.  Ordered before later MMAs of
// the issuing thread.
template <bool PAIR>
__device__ __forceinline__ void tmem_cp_scales(uint32_t leader, uint32_t taddr, uint32_t desc_lo) {
#define RDB_CP_SCALES(GROUP)                                                                            \
    asm volatile(                                                                                       \
        "{\n\t.reg .pred q;\n\t.reg .b64 d;\n\t"                                                       \
        "setp.ne.b32 q, %0, 0;\n\t"                                                                     \
        "mov.b64 d, {%2, %3};\n\t"                                                                      \
        "@q tcgen05.cp.cta_group::" GROUP ".32x128b.warpx4 [%1], d;\n\t}"                                \
        ::"r"(leader), "r"(taddr), "r"(desc_lo), "r"(DESC_HI_SCALES) : "memory")
    if constexpr (PAIR) RDB_CP_SCALES("2");
    else RDB_CP_SCALES("1");
#undef RDB_CP_SCALES
}

// D[tmem] (+)= A[smem] * B[smem]^T with block scales from TMEM, one step of 64 elements of K.
template <int FMT, bool PAIR>
__device__ __forceinline__ void tc_mma_fp4(uint32_t leader, uint32_t tmem_d, uint32_t desc_a, uint32_t desc_b, uint32_t idesc,
                                           uint32_t scale_a, uint32_t scale_b, bool accumulate) {
#define RDB_MMA_FP4(GROUP, KIND)                                                                        \
    asm volatile(                                                                                       \
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"                                                 \
        "setp.ne.b32 p, %6, 0;\n\t"                                                                     \
        "setp.ne.b32 q, %8, 0;\n\t"                                                                     \
        "mov.b64 a, {%1, %7};\n\t"                                                                      \
        "mov.b64 b, {%2, %7};\n\t"                                                                      \
        "@q tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], a, b, %3, [%4], [%5], p;\n\t}"         \
        ::"r"(tmem_d), "r"(desc_a), "r"(desc_b), "r"(idesc), "r"(scale_a), "r"(scale_b),                \
          "r"(static_cast<uint32_t>(accumulate)), "r"(DESC_HI_OPERAND), "r"(leader) : "memory")
    if constexpr (FMT == RDB_FP4_NVFP4) {
        if constexpr (PAIR) RDB_MMA_FP4("2", "mxf4nvf4.block_scale.scale_vec::4X");
        else RDB_MMA_FP4("1", "mxf4nvf4.block_scale.scale_vec::4X");
    } else {
        if constexpr (PAIR) RDB_MMA_FP4("2", "mxf4.block_scale.scale_vec::2X");
        else RDB_MMA_FP4("1", "mxf4.block_scale.scale_vec::2X");
    }
#undef RDB_MMA_FP4
}

// Arrive on an mbarrier (in both CTAs of a pair, at the same offset) when everything the leader issued has finished.
__device__ __forceinline__ void commit(uint32_t leader, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}"
        ::"r"(leader), "r"(bar) : "memory");
}
__device__ __forceinline__ void commit_both(uint32_t leader, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%1], %2;\n\t}"
        ::"r"(leader), "r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}

// A stage of scale tiles is contiguous in memory: one untiled copy.
__device__ __forceinline__ void bulk_load_scales(uint32_t dst_smem, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst_smem), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar) : "memory");
}

// The product of two tensor scales, ready for an accumulator v: (v * pre) * mul = v * ta * tb, rounded once.  As one fp32
// number ta * tb underflows below 2^-126 (operands around 1e-16 and smaller) or overflows where the result need not.  pre
// is a power of two, 1 unless the product's exponent leaves [-100, 100].  v * pre is exact: the accumulator is a multiple
// of 2^-20 (the smallest element times scale, squared) below 2^54 (the largest, squared, 2^31 times), so |exponent of pre|
// <= 106 keeps it a normal number; what is cut off there leaves fp32's range anyway.
struct Alpha { float pre, mul; };
__device__ __forceinline__ Alpha alpha_of(const float* ta, const float* tb) {
    if (!ta) return {1.0f, 1.0f};
    int ea, eb;
    const float m = frexpf(__ldg(ta), &ea) * frexpf(__ldg(tb), &eb);     // in [1/4, 1)
    const int e = ea + eb, near = min(max(e, -100), 100), rest = min(max(e - near, -106), 106);
    return {ldexpf(1.0f, rest), ldexpf(m, near)};
}
template <int N>
__device__ __forceinline__ void times_pre(float* v, const Alpha& a) {
    if (a.pre != 1.0f) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] *= a.pre;
    }
}

__device__ __forceinline__ uint32_t pack2(int type, float x, float y) {
    if (type == RDB_TYPE_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void store1(void* D, int type, size_t at, float v) {
    if (type == RDB_TYPE_FP32) reinterpret_cast<float*>(D)[at] = v;
    else if (type == RDB_TYPE_BF16) reinterpret_cast<__nv_bfloat16*>(D)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(D)[at] = __float2half_rn(v);
}

// Four consecutive outputs of row m at column n, rounded once; vec: 4 outputs can be stored at once.
__device__ __forceinline__ void store4(void* D, int type, size_t N, int m, int n, const float* v, bool vec) {
    const size_t at = static_cast<size_t>(m) * N + n;
    if (type == RDB_TYPE_FP32) {
        float* p = reinterpret_cast<float*>(D) + at;
        if (vec && n + 4 <= N) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (n + j < N) p[j] = v[j];
        return;
    }
    const uint32_t w[2] = {pack2(type, v[0], v[1]), pack2(type, v[2], v[3])};
    uint16_t* p = reinterpret_cast<uint16_t*>(D) + at;
    if (vec && n + 4 <= N) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (n + j < N) p[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
}

}  // namespace fp4
}  // namespace rdb
