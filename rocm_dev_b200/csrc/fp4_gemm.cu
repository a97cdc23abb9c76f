// Products of microscaled 4-bit tensors for sm_100a:  D[M,N] = (A . B^T) * ta * tb, operands held as fp4.cuh describes.
//
// tcgen05.mma kind::mxf4 / kind::mxf4nvf4 multiplies 64 elements of K per step and applies the block scales itself, from
// TMEM; everything up to the fp32 accumulator is exact but the accumulation.  A pipeline stage is 256 elements of K: one
// 128-byte swizzle row of codes per operand row, and the scale tiles of that stretch, which lie contiguous in memory and
// go to shared memory with untiled copies and on to TMEM with tcgen05.cp.  Each ring slot owns TMEM columns for its
// scales, so they are free again exactly when the slot is.
//
// split_kernel: one output tile of 128 x R per cluster, the cluster's S CTAs each taking a slice of K - for products that
// are bound by streaming B (few rows of A) or that have too few tiles to fill the machine.  Roles per CTA as in the fp8
// skinny kernel: warp 0 loads, warp 1 issues the MMAs, then all warps move the accumulator to shared memory, and each
// rank sums its share of the columns over all ranks through distributed shared memory, in rank order: deterministic, no
// workspace, no atomics.
#include <atomic>

#include "fp4_mma.cuh"
#include "host_util.h"

RDB_DEFINE_WAIT_BUDGET_SETTER()

namespace rdb {
namespace fp4 {

constexpr int SMEM_LIMIT = 232448;         // 227 KiB opt-in maximum per CTA
constexpr int SM_SMEM = 228 * 1024;        // an SM's, for all its CTAs
constexpr int CTA_SMEM = 1024 + 160;       // what a CTA takes of it besides the dynamic part: the system's, and static
constexpr int MAX_STAGES = 8;
constexpr int SPLIT_THREADS = 256;
constexpr int A_OPERAND_SPAN = 128 * 128;  // bytes the MMA reads for its 128-row A operand, whatever was loaded

struct SplitParams {
    void* D;
    const uint8_t *sa, *sb;
    const float *ta, *tb;       // tensor scales, nullptr: 1
    int* status;
    int M, N, num_kb;
    int R, mbox;                // columns of the tile (a multiple of 64), rows of A that are loaded
    int b_tiles;                // 128-row scale tiles that R columns touch
    int sb_row_tiles;           // 128-row scale tiles of B in all
    int nstages, tmem_cols;
    int out_type, vec;
    int early_b;                // B may be requested before the preceding kernel has finished
};

template <int FMT>
__host__ __device__ constexpr int split_stage_bytes(int mbox, int R, int b_tiles) {
    return (mbox + R) * 128 + Format<FMT>::TILES * TILE_BYTES * (1 + b_tiles);
}

// Bound by the stream of B and by fill and drain around it: NVFP4 16 x 28672 x 4096 takes 14 to 15 us (66 MB, 10.4 at the
// copy rate; DRAM reads what the operands hold, once), 1 x 4096 x 4096 5.3 (1.5).
template <int FMT>
__global__ void __launch_bounds__(SPLIT_THREADS, 1)
split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const SplitParams p) {
    constexpr int TILES = Format<FMT>::TILES, SCALES = TILES * TILE_BYTES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t bars[2 * MAX_STAGES + 1];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_s;
    __shared__ Alpha alpha_s;
    volatile int* abort_flag = &abort_s;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = gridDim.x, rank = blockIdx.x, R = p.R, nstages = p.nstages;
    const int n0 = blockIdx.y * R, m0 = blockIdx.z * 128;
    const int rows = p.M - m0 < 128 ? p.M - m0 : 128;
    const int kb_begin = static_cast<int>(static_cast<long long>(p.num_kb) * rank / S);
    const int nkb = static_cast<int>(static_cast<long long>(p.num_kb) * (rank + 1) / S) - kb_begin;
    const int A_BYTES = p.mbox * 128, B_BYTES = R * 128;
    const int STAGE = split_stage_bytes<FMT>(p.mbox, R, p.b_tiles);
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + MAX_STAGES), done = smem_u32(bars + 2 * MAX_STAGES);
    const uint32_t stage0 = smem_u32(smem);

    if (threadIdx.x == 0) {
        prefetch_tensormap(&tmA);
        prefetch_tensormap(&tmB);
        for (int s = 0; s < nstages; s++) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        mbar_init(done, 1);
        abort_s = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_slot), p.tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            const uint64_t pol_b = gridDim.z > 1 ? l2_policy_evict_last() : l2_policy_evict_first(), pol_a = l2_policy_evict_last();
            const size_t sa_row = static_cast<size_t>(blockIdx.z) * p.num_kb * SCALES;
            auto load_b = [&](int i, uint32_t dst, uint32_t bar) {
                mbar_arrive_expect_tx(bar, STAGE);
                tma_load_2d(dst + A_BYTES, &tmB, (kb_begin + i) * 128, n0, bar, pol_b);
                for (int j = 0; j < p.b_tiles; j++) {
                    int rt = n0 / 128 + j;
                    if (rt >= p.sb_row_tiles) rt = p.sb_row_tiles - 1;       // columns past N: any scales do
                    bulk_load_scales(dst + A_BYTES + B_BYTES + SCALES * (1 + j),
                                     p.sb + (static_cast<size_t>(rt) * p.num_kb + kb_begin + i) * SCALES, SCALES, bar);
                }
            };
            auto load_a = [&](int i, uint32_t dst, uint32_t bar) {
                tma_load_2d(dst, &tmA, (kb_begin + i) * 128, m0, bar, pol_a);
                bulk_load_scales(dst + A_BYTES + B_BYTES, p.sa + sa_row + static_cast<size_t>(kb_begin + i) * SCALES, SCALES, bar);
            };
            const int pre = nkb < nstages ? nkb : nstages;
            if (!p.early_b) pdl_wait_prior();
            for (int i = 0; i < pre; i++) load_b(i, stage0 + i * STAGE, full0 + 8 * i);
            if (p.early_b) pdl_wait_prior();
            // the next kernel may start now that this one's predecessor has finished: one that fetches its weights early
            // then overlaps this kernel alone, never one further back that may have written them
            pdl_launch_dependents();
            for (int i = 0; i < pre; i++) load_a(i, stage0 + i * STAGE, full0 + 8 * i);
            for (int i = pre; i < nkb; i++) {
                const int s = i % nstages;
                if (!mbar_wait(empty0 + 8 * s, ((i / nstages) & 1) ^ 1)) { *abort_flag = 1; report_timeout(p.status); break; }
                load_b(i, stage0 + s * STAGE, full0 + 8 * s);
                load_a(i, stage0 + s * STAGE, full0 + 8 * s);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // all lanes; see fp4_mma.cuh
        pdl_wait_prior();                                // waits are limited: they count from when the data can come
        const uint32_t leader = elect_one();
        const int slot_cols = TILES * 4 * (1 + p.b_tiles);
        const int shift = (n0 & 127) / 32;               // a tile that starts inside a 128-row scale tile
        const uint32_t idesc0 = idesc_fp4<FMT>(128, R, 0), idesc2 = idesc_fp4<FMT>(128, R, 2);
        for (int i = 0; i < nkb; i++) {
            const int s = i % nstages;
            if (!mbar_wait(full0 + 8 * s, (i / nstages) & 1)) {
                if (leader) { *abort_flag = 1; report_timeout(p.status); }
                break;
            }
            tc_fence_after_sync();
            const uint32_t a = desc_lo_operand(stage0 + s * STAGE), b = a + (A_BYTES >> 4), sc = desc_lo_scales(stage0 + s * STAGE + A_BYTES + B_BYTES);
            const uint32_t tsa = tmem_base + R + s * slot_cols, tsb = tsa + 4 * TILES;
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                tmem_cp_scales<false>(leader, tsa + 4 * t, sc + t * (TILE_BYTES >> 4));
                tmem_cp_scales<false>(leader, tsb + 4 * t * p.b_tiles, sc + ((SCALES + t * TILE_BYTES) >> 4));
                if (p.b_tiles > 1) tmem_cp_scales<false>(leader, tsb + 4 * (t * p.b_tiles + 1), sc + ((2 * SCALES + t * TILE_BYTES) >> 4));
            }
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                const int t = ks * TILES / 4;
                tc_mma_fp4<FMT, false>(leader, tmem_base, a + ks * 2, b + ks * 2, TILES == 2 && (ks & 1) ? idesc2 : idesc0, tsa + 4 * t,
                                       tsb + 4 * t * p.b_tiles + shift, (i | ks) != 0);
            }
            commit(leader, empty0 + 8 * s);
        }
        commit(leader, done);                                // also after an abort
        __syncwarp();
    } else if (warp == 2) {
        if (lane == 0) {
            pdl_wait_prior();
            alpha_s = alpha_of(p.ta, p.tb);
        }
        __syncwarp();
    }

    // ---- the accumulator goes to shared memory, stg[row][R], over the drained ring.  A warp reads the TMEM lane quadrant
    // warp % 4 (32 rows), every second 32 columns of it.
    float* stg = reinterpret_cast<float*>(smem);
    const int pitch = R + 4;
    const int quad = warp & 3;
    pdl_wait_prior();                                        // D may belong to the preceding kernel; and the wait for `done` counts from here
    if (quad * 32 < rows) {
        bool ok = mbar_wait(done, 0);
        if (!ok) { *abort_flag = 1; report_timeout(p.status); }
        tc_fence_after_sync();
        if (ok && *abort_flag == 0) {
            float* row = stg + (quad * 32 + lane) * pitch;
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
#pragma unroll 1
            for (int c0 = warp >= 4 ? 32 : 0; c0 < R; c0 += 64) {
                float v[32];
                tmem_ld32(taddr + c0, v);
#pragma unroll
                for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(row + c0 + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            }
        }
        tc_fence_before_sync();
    }
    __syncthreads();
    const bool aborted = *abort_flag != 0;                   // every wait that can set it lies behind
    if (aborted) {
        for (int i = 0; i < 64; i++) __nanosleep(2000);      // MMAs and copies in flight land before their memory is given back
    }
    // TMEM goes back before this CTA waits for its peers: more CTAs may share an SM than its 512 columns serve, and one of
    // the peers may still wait for columns.  Two clusters that each held some and waited for the other's would hang.
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, p.tmem_cols);
    }
    if (S > 1) {
        cluster_arrive_release();
        cluster_wait_acquire();                              // every rank's partial sums are in place
    }
    const Alpha alpha = alpha_s;
    if (!aborted) {
        // columns in granules of four; rank r sums and stores [G r / S, G (r + 1) / S)
        const int G = R / 4, g0 = G * rank / S, ng = G * (rank + 1) / S - g0;
        for (int item = threadIdx.x; item < rows * ng; item += SPLIT_THREADS) {
            const int m = item / ng, c = (g0 + item - m * ng) * 4;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (n0 + c < p.N) {
                const float* mine = stg + m * pitch + c;
                if (S == 1) {
                    const float4 x = *reinterpret_cast<const float4*>(mine);
                    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
                } else {
                    const uint32_t at = smem_u32(mine);
                    float x[8][4];                           // all ranks' loads in flight together, then summed in order
#pragma unroll
                    for (int src = 0; src < 8; src++)
                        if (src < S)
                            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(x[src][0]), "=f"(x[src][1]), "=f"(x[src][2]), "=f"(x[src][3]) : "r"(mapa_smem(at, src)) : "memory");
#pragma unroll
                    for (int src = 0; src < 8; src++)
                        if (src < S) {
#pragma unroll
                            for (int j = 0; j < 4; j++) v[j] += x[src][j];
                        }
                }
                times_pre<4>(v, alpha);
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] *= alpha.mul;
                store4(p.D, p.out_type, p.N, m0 + m, n0 + c, v, p.vec);
            }
        }
    }
    if (S > 1) {                                             // no rank leaves while another still reads its memory
        __syncwarp();
        cluster_arrive_release();
        cluster_wait_acquire();
    }
}

// ------------------------------------------------------------- CTA pairs
// pair_kernel: persistent clusters of two CTAs compute 256 x 256 tiles with cta_group::2 MMAs.  CTA r of the pair loads
// rows [128 r, 128 r + 128) of the A tile and of the B tile, the scales of its A rows and those of ALL 256 B rows (each
// SM scales its own 128 x 256 half of the tile); the even CTA issues the scale copies and the MMAs for both.
// TMEM (512 columns): two accumulators of 256 columns that overlap by OVERLAP, then the scale slots.  The epilogue empties
// the shared columns first, so the next tile's MMAs wait for those alone.
namespace pairs {
constexpr int THREADS = 224;                    // warp 0: A loads, 1: MMA, 2-5: epilogue, 6: B loads
constexpr int ACC1 = 160, SCALE_COL = ACC1 + 256, GROUP_M = 16;
constexpr int OUT_BYTES = 32 * 128;             // 32 rows of 128 bytes: what one output copy stores
template <int FMT>
struct Cfg {
    static constexpr int SCALES = Format<FMT>::TILES * TILE_BYTES;
    static constexpr int STAGE = 2 * 128 * 128 + 3 * SCALES;
    static constexpr int STAGES = 5;
    static constexpr int SLOT = Format<FMT>::TILES * 12, SLOTS = (512 - SCALE_COL) / SLOT;      // 2 or 4
    static constexpr int OUT = 4 * 2 * OUT_BYTES;                            // two output buffers per epilogue warp
    static constexpr int SMEM = 1024 + STAGES * STAGE + OUT;
};
}  // namespace pairs

struct PairParams {
    void* D;
    const float *ta, *tb;
    int* status;
    int M, N, num_kb, tiles_m, tiles_n;
    int out_type, tma_out;      // tma_out: rows of D start on 16-byte boundaries
};

__device__ __forceinline__ void tile_coords(int tile, int tiles_m, int tiles_n, int& mb, int& nb) {
    const int per_group = pairs::GROUP_M * tiles_n;
    const int g = tile / per_group, r = tile - g * per_group;
    const int first = g * pairs::GROUP_M;
    const int gsize = tiles_m - first < pairs::GROUP_M ? tiles_m - first : pairs::GROUP_M;
    mb = first + r % gsize;
    nb = r / gsize;
}

// NVFP4 8192^3 takes 194 to 208 us in a burst and 215 to 223 sustained, where the board's power limit holds the clock down;
// 4096^3 30.5, with the tensor pipe busy 59 % of the active cycles (four waves on 64 of 74 pairs).
template <int FMT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pairs::THREADS, 1)
pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSA,
            const __grid_constant__ CUtensorMap tmSB, const __grid_constant__ CUtensorMap tmD, const PairParams p) {
    using C = pairs::Cfg<FMT>;
    constexpr int STAGES = C::STAGES, STAGE = C::STAGE, SCALES = C::SCALES, TILES = Format<FMT>::TILES, HALF = 128 * 128;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t bars[2 * STAGES + 2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_s;
    volatile int* abort_flag = &abort_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair_id = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
    const uint32_t acc_full = smem_u32(bars + 2 * STAGES), acc_free = smem_u32(bars + 2 * STAGES + 1);
    const uint32_t stage0 = smem_u32(smem);

    if (threadIdx.x == 0) {
        prefetch_tensormap(&tmA);
        prefetch_tensormap(&tmB);
        prefetch_tensormap(&tmSA);
        prefetch_tensormap(&tmSB);
        for (int s = 0; s < STAGES; s++) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_free, 8);                 // four epilogue warps in each CTA of the pair
        abort_s = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(&tmem_slot), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_arrive_release();                   // both CTAs' barriers and TMEM exist before either touches the other
    cluster_wait_acquire();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_slot;
    const int num_tiles = p.tiles_m * p.tiles_n;
    pdl_wait_prior();
    pdl_launch_dependents();

    if (warp == 0 || warp == 6) {
        if (lane == 0) {
            const bool is_a = warp == 0;
            const CUtensorMap* tm = is_a ? &tmA : &tmB;
            const CUtensorMap* ts = is_a ? &tmSA : &tmSB;
            const uint32_t off = is_a ? 0u : static_cast<uint32_t>(HALF), soff = 2 * HALF + (is_a ? 0 : SCALES);
            const uint64_t pol = l2_policy_evict_last();
            const uint32_t full_even0 = mapa_smem(full0, 0);
            int it = 0;
            bool ok = true;
            for (int tile = pair_id; tile < num_tiles && ok && *abort_flag == 0; tile += num_pairs) {
                int mb, nb;
                tile_coords(tile, p.tiles_m, p.tiles_n, mb, nb);
                const int row = (is_a ? mb : nb) * 256 + static_cast<int>(rank) * 128;
                const int plane = is_a ? mb * 2 + static_cast<int>(rank) : nb * 2;
                for (int kb = 0; kb < p.num_kb; kb++, it++) {
                    const int s = it % STAGES;
                    if (!mbar_wait(empty0 + 8 * s, ((it / STAGES) & 1) ^ 1)) { ok = false; break; }
                    if (is_a && rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, 2 * STAGE);
                    tma_load_2d_pair(stage0 + s * STAGE + off, tm, kb * 128, row, full_even0 + 8 * s, pol);
                    tma_load_3d_pair(stage0 + s * STAGE + soff, ts, 0, kb * (SCALES / 256), plane, full_even0 + 8 * s, pol);
                }
            }
            // every commit aimed at this CTA's `empty` barriers must land before the CTA may exit
            for (int i = 0; i < STAGES && ok && *abort_flag == 0; i++, it++) {
                const int s = it % STAGES;
                if (!mbar_wait(empty0 + 8 * s, ((it / STAGES) & 1) ^ 1)) ok = false;
            }
            if (!ok) { *abort_flag = 1; report_timeout(p.status); }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {                        // all lanes; see fp4_mma.cuh
            const uint32_t leader = elect_one();
            const uint32_t op0 = desc_lo_operand(stage0), sc0 = desc_lo_scales(stage0 + 2 * HALF);
            int it = 0, t = 0;
            bool ok = true;
            for (int tile = pair_id; tile < num_tiles && ok && *abort_flag == 0; tile += num_pairs, t++) {
                const uint32_t d = tmem_base + (t & 1) * pairs::ACC1;
                for (int kb = 0; kb < p.num_kb; kb++, it++) {
                    const int s = it % STAGES;
                    // the scale slot is free when the MMAs of SLOTS stages ago have finished
                    if (it >= C::SLOTS) {
                        const int old = it - C::SLOTS;
                        if (!mbar_wait(empty0 + 8 * (old % STAGES), (old / STAGES) & 1)) { ok = false; break; }
                    }
                    if (!mbar_wait(full0 + 8 * s, (it / STAGES) & 1)) { ok = false; break; }
                    tc_fence_after_sync();
                    const uint32_t a = op0 + s * (STAGE >> 4), b = a + (HALF >> 4), sc = sc0 + s * (STAGE >> 4);
                    const uint32_t tsa = tmem_base + pairs::SCALE_COL + (it % C::SLOTS) * C::SLOT, tsb = tsa + 4 * TILES;
#pragma unroll
                    for (int i = 0; i < TILES; i++) {
                        tmem_cp_scales<true>(leader, tsa + 4 * i, sc + i * (TILE_BYTES >> 4));
                        tmem_cp_scales<true>(leader, tsb + 8 * i, sc + ((SCALES + i * TILE_BYTES) >> 4));
                        tmem_cp_scales<true>(leader, tsb + 8 * i + 4, sc + ((2 * SCALES + i * TILE_BYTES) >> 4));
                    }
                    if (kb == 0 && t > 0) {
                        if (!mbar_wait_cluster(acc_free, (t - 1) & 1)) { ok = false; break; }
                        tc_fence_after_sync();
                    }
#pragma unroll
                    for (int ks = 0; ks < 4; ks++) {
                        const int i = ks * TILES / 4, id = TILES == 4 ? 0 : 2 * (ks & 1);
                        tc_mma_fp4<FMT, true>(leader, d, a + ks * 2, b + ks * 2, idesc_fp4<FMT>(256, 256, id), tsa + 4 * i, tsb + 8 * i, (kb | ks) != 0);
                    }
                    commit_both(leader, empty0 + 8 * s);
                    if (kb == p.num_kb - 1) commit_both(leader, acc_full);
                }
            }
            if (!ok && leader) { *abort_flag = 1; report_timeout(p.status); }
        }
        __syncwarp();
    } else {
        const int quad = warp & 3;
        const Alpha alpha = alpha_of(p.ta, p.tb);
        const uint32_t free_even = mapa_smem(acc_free, 0);
        uint8_t* out = smem + STAGES * STAGE + quad * 2 * pairs::OUT_BYTES;
        int turn = 0;
        // 32 columns of this warp's 32 rows: into shared memory in the layout of the copy's swizzle (128 or 64 bytes a
        // row, no bank conflicts), then one copy out.  A thread holds a row: its own stores would touch 32 lines each.
        auto put = [&](int m0, int n, float* v) {
            if (m0 >= p.M || n >= p.N) return;
            times_pre<32>(v, alpha);
            if (!p.tma_out) {                            // rows of D off 16 bytes: neighbouring lanes store neighbouring columns
                float* mine = reinterpret_cast<float*>(out) + lane * 33;
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 32; j++) mine[j] = v[j] * alpha.mul;
                __syncwarp();
                const int rows = p.M - m0 < 32 ? p.M - m0 : 32;
                if (n + lane < static_cast<int>(p.N)) {
#pragma unroll 8
                    for (int r = 0; r < rows; r++) store1(p.D, p.out_type, static_cast<size_t>(m0 + r) * p.N + n + lane, reinterpret_cast<float*>(out)[r * 33 + lane]);
                }
                return;
            }
            uint8_t* buf = out + (turn & 1) * pairs::OUT_BYTES;
            tma_store_wait_read<1>();                    // lane 0: the copy that last read this buffer is done with it
            __syncwarp();
            if (p.out_type == RDB_TYPE_FP32) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    *reinterpret_cast<float4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                        make_float4(v[4 * j] * alpha.mul, v[4 * j + 1] * alpha.mul, v[4 * j + 2] * alpha.mul, v[4 * j + 3] * alpha.mul);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = pack2(p.out_type, v[8 * j + 2 * i] * alpha.mul, v[8 * j + 2 * i + 1] * alpha.mul);
                    *reinterpret_cast<uint4*>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                tma_store_2d(&tmD, smem_u32(buf), n, m0);
                tma_store_commit();
            }
            turn++;
        };
        int t = 0;
        for (int tile = pair_id; tile < num_tiles; tile += num_pairs, t++) {
            int mb, nb;
            tile_coords(tile, p.tiles_m, p.tiles_n, mb, nb);
            if (!mbar_wait(acc_full, t & 1)) { *abort_flag = 1; report_timeout(p.status); }
            if (*abort_flag != 0) break;
            tc_fence_after_sync();
            const int row0 = mb * 256 + static_cast<int>(rank) * 128 + quad * 32;
            const uint32_t taddr = tmem_base + (t & 1) * pairs::ACC1 + (static_cast<uint32_t>(quad * 32) << 16);
            // columns shared with the other accumulator first: the last 96 of the first, the first 96 of the second
            float v[96];
            const int c0 = (t & 1) ? 0 : pairs::ACC1;
            tmem_ld64(taddr + c0, v);
            tmem_ld32(taddr + c0 + 64, v + 64);
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(free_even);
            const int n0 = nb * 256;
#pragma unroll
            for (int i = 0; i < 3; i++) put(row0, n0 + c0 + 32 * i, v + 32 * i);
            const int c1 = (t & 1) ? 96 : 0;
#pragma unroll 1
            for (int i = 0; i < 5; i++) {
                tmem_ld32(taddr + c1 + 32 * i, v);
                put(row0, n0 + c1 + 32 * i, v);
            }
        }
        tma_store_wait<0>();
    }

    if (*abort_flag != 0) {
        for (int i = 0; i < 64; i++) __nanosleep(2000);
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_arrive_release();                   // neither CTA frees TMEM or exits while the other may still signal it
    cluster_wait_acquire();
    if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

// ------------------------------------------------------------------ host
struct Product {
    const uint8_t *A, *sa, *B, *sb;
    const float *ta, *tb;
    void* D;
    int out_type, M, N, K;
};

struct SplitPlan {
    int R, S, stages, mbox, b_tiles, tmem_cols, smem;
};

static int ring_limit(int format, int mbox, int R, int b_tiles) {
    const int tiles = format == RDB_FP4_NVFP4 ? 4 : 2;
    const int stage = format == RDB_FP4_NVFP4 ? split_stage_bytes<RDB_FP4_NVFP4>(mbox, R, b_tiles) : split_stage_bytes<RDB_FP4_MXFP4>(mbox, R, b_tiles);
    int st = (512 - R) / (tiles * 4 * (1 + b_tiles));
    while (st > 1 && 1024 + st * stage + A_OPERAND_SPAN > SMEM_LIMIT - 1024) st--;
    return st < MAX_STAGES ? st : MAX_STAGES;
}

// The rest of a plan whose R and S are set: stages (at most stage_cap), TMEM columns, shared memory.
static void complete_plan(SplitPlan& pl, int format, int M, int K, int stage_cap) {
    const int num_kb = (K + STAGE_K - 1) / STAGE_K, tiles = format == RDB_FP4_NVFP4 ? 4 : 2, rows = M < 128 ? M : 128;
    pl.b_tiles = (pl.R + 127) / 128;
    pl.stages = ring_limit(format, pl.mbox, pl.R, pl.b_tiles);
    if (pl.stages > stage_cap) pl.stages = stage_cap;
    const int kb = (num_kb + pl.S - 1) / pl.S;
    if (pl.stages > kb) pl.stages = kb;
    pl.tmem_cols = 32;
    while (pl.tmem_cols < pl.R + pl.stages * tiles * 4 * (1 + pl.b_tiles)) pl.tmem_cols *= 2;
    const int stage = format == RDB_FP4_NVFP4 ? split_stage_bytes<RDB_FP4_NVFP4>(pl.mbox, pl.R, pl.b_tiles)
                                              : split_stage_bytes<RDB_FP4_MXFP4>(pl.mbox, pl.R, pl.b_tiles);
    // the ring, what the last stage's A operand reads beyond its rows, and the staging tile that reuses both
    int bytes = pl.stages * stage + A_OPERAND_SPAN;
    const int stg = (rows + 31) / 32 * 32 * (pl.R + 4) * 4;
    if (bytes < stg) bytes = stg;
    pl.smem = 1024 + bytes;
    // no more CTAs to an SM than its 512 columns serve: one more would only wait there for columns while another SM has room
    const int least = SM_SMEM / (512 / pl.tmem_cols + 1);
    if (pl.smem < least) pl.smem = least;
}

// Clusters of S CTAs that are resident at once on the current device with one CTA to an SM; 0 if that cannot be told.
// (The query answers for one CTA to an SM however small its shared memory is.)
static int query_resident(int S) {
    const int smem = SMEM_LIMIT - 1024;
    auto kernel = split_kernel<RDB_FP4_MXFP4>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) { cudaGetLastError(); return 0; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S);
    cfg.blockDim = dim3(SPLIT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) { cudaGetLastError(); return 0; }
    return n;
}

// The same for a plan with up to `per_sm` (1 or 2) CTAs to an SM, as far as shared memory and TMEM columns allow.  Two: twice
// as many at least.  More fit on the layout of SMs that answers kOne: up to kTwo[S] tiles of K = 14336 take one wave, a few
// more 50 to 70 % longer.  These last ones start late, when the launch before has left the very SMs they need, which a long
// K hides (six stages a CTA: 33 tiles 8.6 us cut in eight, 9.1 in six) and a short one does not (K = 4096, 32 tiles: 7.3 us
// in eight, 6.9 in six).
static int resident(const SplitPlan& pl, int per_sm, int num_kb) {
    static const int kOne[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15}, kTwo[9] = {0, 296, 148, 92, 71, 55, 44, 37, 33};
    static std::atomic<int> cache[kMaxDevices][9];                  // answer + 1
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
    std::atomic<int>& slot = cache[dev][pl.S];
    int n = slot.load(std::memory_order_relaxed);
    if (n == 0) slot.store(n = 1 + query_resident(pl.S), std::memory_order_relaxed);
    n--;
    if (per_sm == 1 || pl.tmem_cols > 256 || 2 * (pl.smem + CTA_SMEM) > SM_SMEM) return n;
    return num_kb >= 6 * pl.S && n == kOne[pl.S] ? kTwo[pl.S] : 2 * n;
}

// Tile width and K split; 0 hints mean free choice.  Times are device times on 148 SMs, weights from HBM.
static SplitPlan split_plan(int format, int M, int N, int K, int sm_count, int r_hint, int s_hint, int stages_hint) {
    const int num_kb = (K + STAGE_K - 1) / STAGE_K, m_tiles = (M + 127) / 128;
    SplitPlan best = {};
    best.mbox = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    auto tiles_of = [&](int R) { return static_cast<long long>((N + R - 1) / R) * m_tiles; };
    int stage_cap = MAX_STAGES;
    best.R = 128;
    best.S = 1;
    // K is cut at most `most` times, and no further than all clusters are resident at once: what is left over would be a
    // second wave (46 tiles of 32 x 128, K = 14336, MXFP4: 12.0 us cut in five, 19.6 in six, of which 44 are resident).
    auto widest = [&](int most, int per_sm) {
        for (int S = most < 8 ? most : 8; S >= 2; S--) {
            SplitPlan pl = best;
            pl.S = S;
            complete_plan(pl, format, M, K, stage_cap);
            if (tiles_of(pl.R) <= resident(pl, per_sm, num_kb)) return S;
        }
        return 1;
    };
    if (r_hint > 0 || s_hint > 0) {
        if (r_hint > 0) best.R = r_hint;
        if (s_hint > 0) best.S = s_hint < num_kb ? s_hint : num_kb;
    } else if (M <= 32) {
        // A stream over B.  128 columns and four stages leave room for a second CTA on every SM, which may belong to the
        // next launch: 28672 x 4096 at M = 16 takes 14.6 us, with one CTA of 256 columns 15.6.  (NVFP4 with 17 to 32 rows
        // lacks 320 bytes for that: one CTA to an SM, unless K is short.)  K is cut as often as the clusters are all
        // resident: 8192 x 8192 takes 18.5 us uncut, 9.5 cut in four, 15.9 cut in five.  Not below two stages a CTA (2048 x
        // 2048: 4.5 us in four, 4.9 in eight); a K too short for that in four, in up to four with one CTA to an SM (NVFP4,
        // 16 x 1024: 2048 rows of B take 3.8 us in four or two, 8192 rows 5.3 in four and 4.6 in two).
        if (N <= 64) best.R = 64;
        stage_cap = 4;
        best.S = num_kb < 8 ? widest(num_kb < 4 ? num_kb : 4, 1) : widest(num_kb / 2, 2);
    } else if (tiles_of(128) <= sm_count) {
        // One CTA to an SM: K is cut while the clusters are resident, down to four stages a CTA (128 x 4096 x 4096: 8.5 us in
        // four, 9.2 in two; 128 x 6144 x 4096, 48 tiles: 9.8 in two, 17.5 in three, of which 45 are
        // resident); a short K is not cut, tiles are narrower instead (1024^3: 5.5 us with 64 columns, 6.5 with 128).
        best.S = widest(num_kb / 4, 1);
        if (best.S <= 1 && num_kb <= 8 && tiles_of(64) <= sm_count) best.R = 64;
    } else {
        best.R = 256;       // 128 x 28672 x 4096: 19.4 us, with 128 columns in two waves 26
    }
    complete_plan(best, format, M, K, stages_hint > 0 && stages_hint < stage_cap ? stages_hint : stage_cap);
    return best;
}

template <int FMT>
static int launch_split(const Product& q, const SplitPlan& pl, unsigned flags, const DeviceInfo* info, cudaStream_t stream) {
    static bool attr_set[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return RDB_CUDA_ERROR;
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(split_kernel<FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT - 1024) != cudaSuccess) return RDB_CUDA_ERROR;
        attr_set[dev] = true;
    }
    CUtensorMap tmA, tmB;
    const uint64_t pitch = row_bytes(q.K);
    int r = make_tmap_2d(&tmA, q.A, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.M, pitch, pitch, 128, pl.mbox, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r != RDB_SUCCESS) return r;
    r = make_tmap_2d(&tmB, q.B, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.N, pitch, pitch, 128, pl.R, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r != RDB_SUCCESS) return r;
    SplitParams p;
    p.D = q.D;
    p.sa = q.sa; p.sb = q.sb; p.ta = q.ta; p.tb = q.tb;
    p.status = info->status_dev;
    p.M = q.M; p.N = q.N;
    p.num_kb = (q.K + STAGE_K - 1) / STAGE_K;
    p.R = pl.R; p.mbox = pl.mbox; p.b_tiles = pl.b_tiles;
    p.sb_row_tiles = (q.N + 127) / 128;
    p.nstages = pl.stages; p.tmem_cols = pl.tmem_cols;
    p.out_type = q.out_type;
    p.vec = q.N % 4 == 0 && (reinterpret_cast<uintptr_t>(q.D) & (q.out_type == RDB_TYPE_FP32 ? 15u : 7u)) == 0;
    p.early_b = (flags & RDB_SKINNY_OVERLAP_PRIOR_KERNEL) != 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(pl.S, (q.N + pl.R - 1) / pl.R, (q.M + 127) / 128);
    cfg.blockDim = dim3(SPLIT_THREADS);
    cfg.dynamicSmemBytes = pl.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = pl.S;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, split_kernel<FMT>, tmA, tmB, p) != cudaSuccess) { cudaGetLastError(); return RDB_CUDA_ERROR; }
    return RDB_SUCCESS;
}

template <int FMT>
static int launch_pair(const Product& q, int max_ctas, const DeviceInfo* info, cudaStream_t stream) {
    using C = pairs::Cfg<FMT>;
    static bool attr_set[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return RDB_CUDA_ERROR;
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(pair_kernel<FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return RDB_CUDA_ERROR;
        attr_set[dev] = true;
    }
    PairParams p;
    p.D = q.D;
    p.ta = q.ta; p.tb = q.tb;
    p.status = info->status_dev;
    p.M = q.M; p.N = q.N;
    p.num_kb = (q.K + STAGE_K - 1) / STAGE_K;
    p.tiles_m = (q.M + 255) / 256;
    p.tiles_n = (q.N + 255) / 256;
    p.out_type = q.out_type;
    const int out_size = q.out_type == RDB_TYPE_FP32 ? 4 : 2;
    p.tma_out = q.N * static_cast<size_t>(out_size) % 16 == 0 && aligned16(q.D);
    CUtensorMap tmA, tmB, tmSA, tmSB, tmD = {};
    const uint64_t pitch = row_bytes(q.K), scale_rows = static_cast<uint64_t>(p.num_kb) * C::SCALES / 256;
    int r = make_tmap_2d(&tmA, q.A, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.M, pitch, pitch, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r == RDB_SUCCESS) r = make_tmap_2d(&tmB, q.B, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.N, pitch, pitch, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r == RDB_SUCCESS) r = make_tmap_bytes256(&tmSA, q.sa, scale_rows, (q.M + 127) / 128, C::SCALES / 256, 1);
    if (r == RDB_SUCCESS) r = make_tmap_bytes256(&tmSB, q.sb, scale_rows, (q.N + 127) / 128, C::SCALES / 256, 2);
    if (r == RDB_SUCCESS && p.tma_out)
        r = make_tmap_2d(&tmD, q.D, q.out_type == RDB_TYPE_FP32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, out_size, q.M, q.N,
                         static_cast<uint64_t>(q.N) * out_size, 32, 32, out_size == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
    if (r != RDB_SUCCESS) return r;
    int num_pairs = p.tiles_m * p.tiles_n, cap = info->sm_count / 2;
    if (max_ctas > 0 && max_ctas / 2 < cap) cap = max_ctas / 2 > 0 ? max_ctas / 2 : 1;
    if (num_pairs > cap) num_pairs = (num_pairs + (num_pairs + cap - 1) / cap - 1) / ((num_pairs + cap - 1) / cap);    // same waves, fewest CTAs
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * num_pairs);
    cfg.blockDim = dim3(pairs::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, pair_kernel<FMT>, tmA, tmB, tmSA, tmSB, tmD, p) != cudaSuccess) { cudaGetLastError(); return RDB_CUDA_ERROR; }
    return RDB_SUCCESS;
}

static int check(const Product& q, int format) {
    if (q.M < 1 || q.N < 1 || q.K < 1) return RDB_BAD_SHAPE;
    if (format != RDB_FP4_MXFP4 && format != RDB_FP4_NVFP4) return RDB_INVALID_CONFIG;
    if (q.M > MAX_EXTENT || q.N > MAX_EXTENT || q.K > MAX_EXTENT) return RDB_SIZE_ABOVE_LIMIT;
    if (q.out_type != RDB_TYPE_BF16 && q.out_type != RDB_TYPE_FP16 && q.out_type != RDB_TYPE_FP32) return RDB_INVALID_CONFIG;
    if (!q.A || !q.sa || !q.B || !q.sb || !q.D) return RDB_INVALID_CONFIG;
    if (format == RDB_FP4_NVFP4 ? !q.ta || !q.tb : q.ta || q.tb) return RDB_INVALID_CONFIG;
    if (!aligned16(q.A) || !aligned16(q.sa) || !aligned16(q.B) || !aligned16(q.sb) ||
        reinterpret_cast<uintptr_t>(q.D) % (q.out_type == RDB_TYPE_FP32 ? 4 : 2) ||
        (reinterpret_cast<uintptr_t>(q.ta) & 3u) || (reinterpret_cast<uintptr_t>(q.tb) & 3u))
        return RDB_BAD_ALIGNMENT;
    return RDB_SUCCESS;
}

static bool split_fits(const SplitPlan& pl, const Product& q) {       // the grid's limits: 65535 tiles in y and z
    return (q.N + pl.R - 1) / pl.R <= 65535 && (q.M + 127) / 128 <= 65535;
}

static int run_pairs(const Product& q, int format, int max_ctas, DeviceInfo* info, cudaStream_t stream) {
    const long long tiles = static_cast<long long>((q.M + 255ll) / 256) * ((q.N + 255ll) / 256);
    if (tiles > (1ll << 30)) return RDB_SIZE_ABOVE_LIMIT;
    return format == RDB_FP4_NVFP4 ? launch_pair<RDB_FP4_NVFP4>(q, max_ctas, info, stream) : launch_pair<RDB_FP4_MXFP4>(q, max_ctas, info, stream);
}

static int run_split(const Product& q, int format, int r_hint, int s_hint, int stages_hint, unsigned flags, DeviceInfo* info, cudaStream_t stream) {
    const SplitPlan pl = split_plan(format, q.M, q.N, q.K, info->sm_count, r_hint, s_hint, stages_hint);
    if (!split_fits(pl, q)) return RDB_SIZE_ABOVE_LIMIT;
    return format == RDB_FP4_NVFP4 ? launch_split<RDB_FP4_NVFP4>(q, pl, flags, info, stream) : launch_split<RDB_FP4_MXFP4>(q, pl, flags, info, stream);
}

}  // namespace fp4
}  // namespace rdb

extern "C" {

int rdb_skinny_gemm_fp4_tuned(const uint8_t* A, const uint8_t* scales_a, const float* tensor_scale_a, const uint8_t* B,
                              const uint8_t* scales_b, const float* tensor_scale_b, void* D, int out_type, int M, int N, int K,
                              int format, int columns_per_tile, int split_k, int stages, unsigned flags, void* stream) {
    const rdb::fp4::Product q = {A, scales_a, B, scales_b, tensor_scale_a, tensor_scale_b, D, out_type, M, N, K};
    const int ok = rdb::fp4::check(q, format);
    if (ok != RDB_SUCCESS) return ok;
    if (M > 32) return RDB_M_ABOVE_WARPTILE_M;
    if (flags & ~RDB_SKINNY_OVERLAP_PRIOR_KERNEL) return RDB_INVALID_CONFIG;
    if (columns_per_tile < 0 || columns_per_tile > 256 || columns_per_tile % 64 != 0 || split_k < 0 || split_k > 8 || stages < 0) return RDB_INVALID_CONFIG;
    int err = 0;
    rdb::DeviceInfo* info = rdb::device_info(&err);
    if (!info) return err;
    auto st = static_cast<cudaStream_t>(stream);
    // more columns than the split kernel's grid can have tiles (8.4 million): pairs, whose tiles are walked
    if (columns_per_tile == 0 && split_k == 0 && stages == 0 && !rdb::fp4::split_fits(rdb::fp4::split_plan(format, M, N, K, info->sm_count, 0, 0, 0), q))
        return rdb::fp4::run_pairs(q, format, 0, info, st);
    return rdb::fp4::run_split(q, format, columns_per_tile, split_k, stages, flags, info, st);
}

int rdb_fp4_split_plan(int M, int N, int K, int format, int* columns_per_tile, int* split_k, int* stages, int* smem_bytes) {
    if (M < 1 || N < 1 || K < 1) return RDB_BAD_SHAPE;
    if (format != RDB_FP4_MXFP4 && format != RDB_FP4_NVFP4) return RDB_INVALID_CONFIG;
    if (M > rdb::fp4::MAX_EXTENT || N > rdb::fp4::MAX_EXTENT || K > rdb::fp4::MAX_EXTENT) return RDB_SIZE_ABOVE_LIMIT;
    if (!columns_per_tile || !split_k || !stages || !smem_bytes) return RDB_INVALID_CONFIG;
    int err = 0;
    rdb::DeviceInfo* info = rdb::device_info(&err);
    if (!info) return err;
    const rdb::fp4::SplitPlan pl = rdb::fp4::split_plan(format, M, N, K, info->sm_count, 0, 0, 0);
    *columns_per_tile = pl.R;
    *split_k = pl.S;
    *stages = pl.stages;
    *smem_bytes = pl.smem;
    return RDB_SUCCESS;
}

int rdb_skinny_gemm_fp4(const uint8_t* A, const uint8_t* scales_a, const float* tensor_scale_a, const uint8_t* B,
                        const uint8_t* scales_b, const float* tensor_scale_b, void* D, int out_type, int M, int N, int K, int format,
                        unsigned flags, void* stream) {
    return rdb_skinny_gemm_fp4_tuned(A, scales_a, tensor_scale_a, B, scales_b, tensor_scale_b, D, out_type, M, N, K, format, 0, 0, 0, flags, stream);
}

int rdb_dense_gemm_fp4_tuned(const uint8_t* A, const uint8_t* scales_a, const float* tensor_scale_a, const uint8_t* B,
                             const uint8_t* scales_b, const float* tensor_scale_b, void* D, int out_type, int M, int N, int K,
                             int format, int tiling, int max_ctas, void* stream) {
    const rdb::fp4::Product q = {A, scales_a, B, scales_b, tensor_scale_a, tensor_scale_b, D, out_type, M, N, K};
    const int ok = rdb::fp4::check(q, format);
    if (ok != RDB_SUCCESS) return ok;
    if (tiling < 0 || tiling > 2 || max_ctas < 0) return RDB_INVALID_CONFIG;
    int err = 0;
    rdb::DeviceInfo* info = rdb::device_info(&err);
    if (!info) return err;
    auto st = static_cast<cudaStream_t>(stream);
    if (tiling == 0) {
        // Pairs where their 256 x 256 tiles are enough for half of the machine and K is long, or there are more 128-row
        // tiles than SMs: 512 x 4096 x 4096 takes 11.0 us (12.3 with 128-row tiles), 256 x 4096 x 4096 10.9 (9.9), 1024^3
        // 6.8 (5.5).  Up to 128 rows a pair would multiply padding: 48 x 28672 x 4096 takes 20.9 us, 15.5 with 128 rows.
        const long long t128 = static_cast<long long>((M + 127ll) / 128) * ((N + 127ll) / 128);
        const bool pairs = M > 128 && (t128 > info->sm_count || (2 * t128 > info->sm_count && K > 8 * rdb::fp4::STAGE_K));
        // (Nor does the split kernel's grid hold every N.)
        tiling = pairs || !rdb::fp4::split_fits(rdb::fp4::split_plan(format, M, N, K, info->sm_count, 0, 0, 0), q) ? 2 : 1;
    }
    if (tiling == 2) return rdb::fp4::run_pairs(q, format, max_ctas, info, st);
    return rdb::fp4::run_split(q, format, 0, 0, 0, 0, info, st);
}

int rdb_dense_gemm_fp4(const uint8_t* A, const uint8_t* scales_a, const float* tensor_scale_a, const uint8_t* B, const uint8_t* scales_b,
                       const float* tensor_scale_b, void* D, int out_type, int M, int N, int K, int format, void* stream) {
    return rdb_dense_gemm_fp4_tuned(A, scales_a, tensor_scale_a, B, scales_b, tensor_scale_b, D, out_type, M, N, K, format, 0, 0, stream);
}

}  // extern "C"
