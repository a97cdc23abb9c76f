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

// Shared-memory descriptor of a scale tile: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t addr) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) | (1ull << 46);
}

// 512 bytes -> four TMEM columns, the 32 rows repeated in each of the four lane quadrants.  Ordered before later MMAs of
// the issuing thread.
template <bool PAIR>
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint32_t smem_addr) {
    if constexpr (PAIR)
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(smem_desc_scales(smem_addr)) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(smem_desc_scales(smem_addr)) : "memory");
}

// D[tmem] (+)= A[smem] * B[smem]^T with block scales from TMEM, one step of 64 elements of K.
template <int FMT, bool PAIR>
__device__ __forceinline__ void tc_mma_fp4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t scale_a,
                                           uint32_t scale_b, bool accumulate) {
#define RDB_MMA_FP4(GROUP, KIND)                                                                        \
    asm volatile(                                                                                       \
        "{\n\t.reg .pred p;\n\t"                                                                        \
        "setp.ne.b32 p, %6, 0;\n\t"                                                                     \
        "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}"         \
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(static_cast<uint32_t>(accumulate)) : "memory")
    if constexpr (FMT == RDB_FP4_NVFP4) {
        if constexpr (PAIR) RDB_MMA_FP4("2", "mxf4nvf4.block_scale.scale_vec::4X");
        else RDB_MMA_FP4("1", "mxf4nvf4.block_scale.scale_vec::4X");
    } else {
        if constexpr (PAIR) RDB_MMA_FP4("2", "mxf4.block_scale.scale_vec::2X");
        else RDB_MMA_FP4("1", "mxf4.block_scale.scale_vec::2X");
    }
#undef RDB_MMA_FP4
}

// A stage of scale tiles is contiguous in memory: one untiled copy.
__device__ __forceinline__ void bulk_load_scales(uint32_t dst_smem, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst_smem), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar) : "memory");
}

// 32 consecutive outputs of row m from column n on; vec: 16-byte stores are aligned.
__device__ __forceinline__ void store32(void* D, int type, size_t N, int m, int n, const float* v, float alpha, bool vec) {
    const size_t at = static_cast<size_t>(m) * N + n;
    const bool whole = vec && n + 32 <= N;
    if (type == RDB_TYPE_FP32) {
        float* p = reinterpret_cast<float*>(D) + at;
        if (whole) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(v[j] * alpha, v[j + 1] * alpha, v[j + 2] * alpha, v[j + 3] * alpha);
        } else {
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (n + j < N) p[j] = v[j] * alpha;
        }
        return;
    }
    uint16_t* p = reinterpret_cast<uint16_t*>(D) + at;
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x = v[j + 2 * i] * alpha, y = v[j + 2 * i + 1] * alpha;
            if (type == RDB_TYPE_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __half2 h = __floats2half2_rn(x, y);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        if (whole) {
            *reinterpret_cast<uint4*>(p + j) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (n + j + i < N) p[j + i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
        }
    }
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
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        if (type == RDB_TYPE_BF16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    uint16_t* p = reinterpret_cast<uint16_t*>(D) + at;
    if (vec && n + 4 <= N) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (n + j < N) p[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
}

}  // namespace fp4
}  // namespace rdb
