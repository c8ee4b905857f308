// Private part of gemm_i8_sm100.cu: the gradient product through a frozen int8 weight,
//
//   dx[m, k] = sum_n t[m, n] * W[n, k],   t = dz * sb (fp32),   W int8 [N, K] as the forward has it.
//
// W is int8 and a gradient needs more than eight bits, so each row of t is put into 16-bit fixed point relative to its
// largest magnitude and cut into two int8 digits: t = s * (256 hi + mid), s = top / 32639, off by at most 2^-16 of the row's
// top.  Both digits go through the int8 tensor cores with exact int32 sums, hi in one accumulator and mid in another (256 +
// 256 columns are the whole tensor memory), and dx = s * (256 sum_hi + sum_mid).  A digit pass costs what an int8 GEMM
// costs, the pair what a bf16 GEMM of that size costs, but W needs neither a bf16 copy nor a conversion on its way.
//
// Rows with outliers have a third digit (gradient_digits.cuh).  A tile with such a row takes a third pass: the drain warps
// turn the first two accumulators into 256 sum_hi + sum_mid, fp32, in the place of hi's, and the third digit is summed in
// the place of mid's.  Its other rows take nothing from it: a row's result does not depend on the rows beside it.  The whole
// backward pass of 2048 x 4096 x 7168 with GELU and bias: 154 us without such rows, 195 to 207 us with one in every tile.
//
// The sum runs over W's rows, so W is the operand whose memory runs along its N axis: its 128 x 128-byte boxes are used
// as they lie in memory (an MN-major operand); no transposed copy of the weight exists.
//
// Pairs of CTAs, tiles of 256 x 256, pipeline and barriers as in gemm_i8_pair_kernel; a tile walks the K blocks twice.
// With both accumulators taken by one tile, the drain does not overlap the next tile's MMAs (its loads do).  Short sums feel
// it: at N = 134, K = 7568 the kernel takes 24 us for 37 MB of dx.  4096 x 7168 over N = 4096: 174 us = 2.8 POPS of int8 work.
#ifndef W8A8_GEMM_I8_GRAD_KERNEL_CUH
#define W8A8_GEMM_I8_GRAD_KERNEL_CUH

#include <type_traits>

#include "gemm_i8_common.cuh"
#include "gemm_i8_epilogues.cuh"
#include "gemm_i8_fused_pair_kernel.cuh"
#include "gradient_digits.cuh"

namespace w8a8 {
namespace {

struct GradParams {
    const unsigned* row_size;  // [M] packed_size of the rows of t
    const uint8_t* wide;       // whether a block of 32 rows has a wide one; 8-byte aligned, zeros up to whole tiles of 256 rows
    __nv_bfloat16* dx;         // [M, K]
    int M, K;
    // the sum runs over `parts` ranges of part_rows rows of W (gates and ups of a gated weight); a digit row holds them at
    // columns that are multiples of part_blocks * 128, with zeros behind each
    int parts, part_rows, part_blocks;
    int group_m;
    // bias gradient: column sums of blocks of rows, added up by the drain warps while the first tile is multiplied
    const float* partial;      // [row_blocks][columns], or null
    int row_blocks;
    float* dbias;
    unsigned long long wait_limit_ns;
    int withhold_loads;        // as in Params
};

// Not zero if one of the rows [row0, row0 + ROWS) is in a block of 32 with a wide row; row0 is a multiple of ROWS.  One load:
// eight of them, one after another, added 4 us to every tile.
template <int ROWS>
__device__ __forceinline__ unsigned any_wide(const GradParams& p, int row0) {
    const uint8_t* first = p.wide + row0 / 32;
    if constexpr (ROWS == 256) {
        const uint2 q = __ldcg(reinterpret_cast<const uint2*>(first));
        return q.x | q.y;
    } else if constexpr (ROWS == 128) {
        return __ldcg(reinterpret_cast<const unsigned*>(first));
    } else if constexpr (ROWS == 64) {
        return __ldcg(reinterpret_cast<const unsigned short*>(first));
    } else {
        return __ldcg(reinterpret_cast<const unsigned char*>(first));
    }
}

// 32 columns per warp, a lane per column; the blocks' sums are added in sixteen interleaved chains (so that as many loads are
// under way), in an order that only the number of blocks fixes
__device__ __forceinline__ void sum_columns(const GradParams& p, int warp, int warps) {
    const int columns = p.parts * p.part_rows, lane = threadIdx.x & 31;
    for (int c = warp * 32 + lane; c < columns; c += warps * 32) {
        float s[16] = {};
#pragma unroll 1
        for (int b = 0; b < p.row_blocks; b += 16) {
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = b + j < p.row_blocks ? __ldcg(p.partial + (int64_t)(b + j) * columns + c) : 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] += v[j];
        }
#pragma unroll
        for (int h = 8; h > 0; h >>= 1) {
#pragma unroll
            for (int j = 0; j < h; ++j) s[j] += s[j + h];
        }
        p.dbias[c] = s[0];
    }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFusedThreads, 1)
gemm_i8_grad_kernel(const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmW, const GradParams p) {
    using L = FusedPairSmem;
    constexpr int STAGES = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kTmemSlotOff);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kAbortOff);
    const uint32_t tiles_base = ptx::smem_u32(smem);
    const uint32_t bar_base = ptx::smem_u32(bars);
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    const uint32_t acc_full_bar = bar_base + 8u * (2 * STAGES), acc_empty_bar = bar_base + 8u * (2 * STAGES + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_ctarank();

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        ptx::mbar_init(acc_full_bar, 1);
        ptx::mbar_init(acc_empty_bar, 2 * kFusedDrainWarps);
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
        ptx::prefetch_tensormap(&tmD);
        ptx::prefetch_tensormap(&tmW);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), 512);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();  // the peer's barriers exist before anything arrives on them
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    const int tiles_m = (p.M + 255) / 256, tiles_k = (p.K + 255) / 256;
    const int total = tiles_m * tiles_k;
    const PairTileOrder order{tiles_m, tiles_k, p.group_m};
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int blocks = p.parts * p.part_blocks;

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        if (!p.withhold_loads && ptx::elect_one()) {
            ptx::grid_dependency_wait();   // the digits come from the kernel before
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = pair; t < total && ok; t += npairs) {
                int mt, kt;
                order.at(t, mt, kt);
                const int digits = any_wide<256>(p, mt * 256) != 0 ? 3 : 2;
                for (int digit = 0; digit < digits && ok; ++digit) {
                    const int row0 = digit * p.M + mt * 256 + (int)rank * 128;   // rows past the digit belong to no output
                    for (int nb = 0; nb < blocks; ++nb) {
                        if (!ptx::mbar_wait_bounded(empty_bar(stage), phase ^ 1u, p.wait_limit_ns) || *abort_flag) {
                            report_wait_failure(kWaitEmptyStage);
                            *abort_flag = 1;
                            ok = false;
                            break;
                        }
                        const uint32_t a_dst = tiles_base + stage * L::kStageBytes;
                        const uint32_t leader_full = ptx::map_to_cta(full_bar(stage), 0);
                        if (rank == 0) ptx::mbar_arrive_expect_tx(full_bar(stage), 2 * L::kStageBytes);
                        ptx::tma_load_2d_pair(a_dst, &tmD, nb * BK, row0, leader_full);
                        const int part = nb >= p.part_blocks ? 1 : 0;
                        ptx::tma_load_2d_pair(a_dst + L::kABytes, &tmW, kt * 256 + (int)rank * 128,
                                              part * p.part_rows + (nb - part * p.part_blocks) * BK, leader_full);
                        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (even CTA only) ----------------
        if (rank == 0 && ptx::elect_one()) {
            ptx::grid_dependency_wait();   // `wide` comes from the kernel before
            constexpr uint32_t idesc = ptx::idesc_i8_b_mn(256, 256);
            int stage = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            auto wide_tile = [&](int t) {
                int mt, kt;
                order.at(t, mt, kt);
                return any_wide<256>(p, mt * 256);
            };
            unsigned wide = wide_tile(pair);
            for (int t = pair; t < total && ok; t += npairs) {
                const unsigned next_wide = wide_tile(min(t + npairs, total - 1));   // asked for well before it is needed
                for (int digit = 0; digit < (wide != 0 ? 3 : 2) && ok; ++digit) {
                    // the first digits need both accumulators drained, the third that they have become one
                    if (digit != 1) {
                        if (!ptx::mbar_wait_bounded(acc_empty_bar, acc_phase ^ 1u, p.wait_limit_ns) || *abort_flag) {
                            report_wait_failure(kWaitAccEmpty);
                            *abort_flag = 1;
                            ok = false;
                            break;
                        }
                        ptx::tc_fence_after_sync();
                    }
                    for (int nb = 0; nb < blocks; ++nb) {
                        if (!ptx::mbar_wait_bounded(full_bar(stage), phase, p.wait_limit_ns) || *abort_flag) {
                            report_wait_failure(kWaitFullStage);
                            *abort_flag = 1;
                            ok = false;
                            break;
                        }
                        ptx::tc_fence_after_sync();
                        const uint32_t a_src = tiles_base + stage * L::kStageBytes;
                        const uint64_t adesc = ptx::smem_desc_k_sw128(a_src);
                        const uint64_t bdesc = ptx::smem_desc_mn_sw128(a_src + L::kABytes);
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; ++k)
                            ptx::mma_i8_ss_pair(tmem_base + (digit == 0 ? 0 : 256), adesc + 2u * k, bdesc + (4096u >> 4) * k, idesc,
                                                (nb | k) != 0 ? 1u : 0u);
                        ptx::tc_commit_pair(empty_bar(stage), 0x3);
                        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    }
                    if (!ok) break;
                    if (digit != 0) {
                        ptx::tc_commit_pair(acc_full_bar, 0x3);
                        acc_phase ^= 1u;
                    }
                }
                wide = next_wide;
            }
        }
    } else {
        // ---------------- drain warps (both CTAs) ----------------
        ptx::grid_dependency_wait();
        if (p.partial != nullptr) sum_columns(p, blockIdx.x * kFusedDrainWarps + warp - 2, gridDim.x * kFusedDrainWarps);
        const int quarter = warp & 3, turn = (warp - 2) >> 2;
        uint32_t* stage = reinterpret_cast<uint32_t*>(smem + L::kTransposeOff + (warp - 2) * kBlockBytes);
        uint32_t acc_phase = 0;
        const bool vec = block_vector_ok(p.dx, p.K, p.K);
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        for (int t = pair; t < total; t += npairs) {
            int mt, kt;
            order.at(t, mt, kt);
            const int row0 = mt * 256 + (int)rank * 128 + quarter * 32, rows = min(32, p.M - row0);
            const unsigned size = lane < rows ? __ldcg(p.row_size + row0 + lane) : 0u;
            const float s = digit_scale(top_of_size(size));
            const bool wide = any_wide<256>(p, mt * 256) != 0;
            __syncwarp();
            auto accumulators_full = [&]() {
                if (!ptx::mbar_wait_bounded(acc_full_bar, acc_phase, p.wait_limit_ns) || *abort_flag) {
                    report_wait_failure(kWaitAccFull);
                    *abort_flag = 1;
                    return false;
                }
                ptx::tc_fence_after_sync();
                return true;
            };
            auto release_accumulators = [&]() {
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_cta(acc_empty_bar, 0));
                acc_phase ^= 1u;
            };
            if (!accumulators_full()) break;
            if (wide) {
#pragma unroll 1
                for (int cc = turn; cc < 8; cc += 2) {
                    uint32_t hi[32], mid[32];
                    __syncwarp();
                    ptx::tmem_ld_32x32b_x32(t_lane + cc * 32, hi);
                    ptx::tmem_ld_32x32b_x32(t_lane + 256 + cc * 32, mid);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) hi[j] = __float_as_uint(digit_sum((int)hi[j], (int)mid[j]));
                    ptx::tmem_st_32x32b_x32(t_lane + cc * 32, hi);
                }
                ptx::tmem_st_wait();
                release_accumulators();
                if (!accumulators_full()) break;
            }
            // separate loops for the two kinds of tile: one loop with the choice inside made every tile's drain half as
            // long again (2422 x 134 x 7568 47 -> 62 us)
            auto drain = [&](auto third) {
#pragma unroll 1
                for (int cc = turn; cc < 8; cc += 2) {
                    uint32_t hi[32], last[32];   // with the third digit: the sum of the first two, and the third
                    __syncwarp();
                    ptx::tmem_ld_32x32b_x32(t_lane + cc * 32, hi);
                    ptx::tmem_ld_32x32b_x32(t_lane + 256 + cc * 32, last);
                    ptx::tmem_ld_wait();
                    const int k = kt * 256 + cc * 32;
                    if (rows <= 0 || k >= p.K) continue;
                    auto value = [&](int j) {
                        float v;
                        if constexpr (decltype(third)::value) {
                            v = __uint_as_float(hi[j]);
                            if (is_wide(size)) v = wide_digit_sum(v, (int)last[j]);
                        } else {
                            v = digit_sum((int)hi[j], (int)last[j]);
                        }
                        return __fmul_rn(v, s);
                    };
                    Row32 out;
#pragma unroll
                    for (int j = 0; j < 16; ++j) out.w[j] = pack_bf16x2_rn(value(2 * j), value(2 * j + 1));
                    store_block(p.dx + (int64_t)row0 * p.K + k, p.K, out, {rows, p.K - k, vec}, stage, lane);
                }
            };
            if (wide) drain(std::true_type{});
            else drain(std::false_type{});
            release_accumulators();
        }
    }

    // ---------------- teardown ----------------
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();  // neither CTA leaves while the other may still touch its memory
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
}

// ------------------------------------------------------------------------------------
// The same product for few rows: operands swapped, as in gemm_i8_stream_kernel.  128 columns of W sit on the MMA's M axis
// (W is then the A operand, MN-major as above), ROWS rows of both digits side by side on its N axis, so W is read once
// for both digits and no tensor-core rows are spent on padding.  A cluster of S CTAs shares one tile and splits W's rows
// between its CTAs; the int32 partials [2 ROWS][128] meet in shared memory and are summed exactly.  More rows than ROWS
// are further blocks of clusters, which read W again.  A block with a wide row walks its share of W's rows once more for the
// third digit, into accumulator columns of its own.
// ------------------------------------------------------------------------------------
template <int ROWS>
struct GradStreamSmem {
    static constexpr int kWBytes = 128 * BK;
    static constexpr int kDigitBytes = ROWS * BK;   // one digit's rows
    static constexpr int kStageBytes = kWBytes + 2 * kDigitBytes;
    static constexpr int kRingBytes = 196 * 1024;
    static constexpr int kStages = kRingBytes / kStageBytes < 10 ? kRingBytes / kStageBytes : 10;
    static constexpr int kTilesBytes = kStages * kStageBytes;
    static constexpr int kColumns = (3 * ROWS + 31) / 32 * 32;   // accumulator columns, read 32 at a time
    static constexpr int kTmemColumns = kColumns <= 64 ? 64 : kColumns <= 128 ? 128 : kColumns <= 256 ? 256 : 512;
    static constexpr int kPartialBytes = kColumns * 128 * 4;
    static_assert(kPartialBytes <= kTilesBytes, "the partial tile reuses the stage ring");
    static constexpr int kScaleOff = kTilesBytes;   // the rows' digit scales, negative for wide rows
    static constexpr int kBarOff = kScaleOff + ROWS * 4;
    static constexpr int kNumBars = 2 * kStages + 1;
    static constexpr int kTmemSlotOff = kBarOff + kNumBars * 8;
    static constexpr int kAbortOff = kTmemSlotOff + 4;
    static constexpr int kWideOff = kAbortOff + 4;
    static constexpr int kTotal = kWideOff + 4;
    static constexpr int kDynamic = kTotal + 1024;
};

// dx of the rows [lo, hi) of the block: item = (row, four columns), consecutive threads on consecutive columns
template <int ROWS, int U, bool WIDE>
__device__ __forceinline__ void reduce_gradient(const GradParams& p, const uint32_t (&peer_base)[8], int S, int m0, int lo, int hi,
                                                int k0, const float* scale_s) {
    constexpr int D = WIDE ? 3 : 2;
    const int items = (hi - lo) * 32;
    const bool vec = (reinterpret_cast<uintptr_t>(p.dx) & 7) == 0;   // K is a multiple of 16
    for (int it0 = threadIdx.x; it0 < items; it0 += kThreads * U) {
        uint4 v[U][D][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = it0 + u * kThreads;
            if (it < items) {
#pragma unroll
                for (int d = 0; d < D; ++d) {
                    const uint32_t off = (uint32_t)((d * ROWS + lo + (it >> 5)) * 128 + (it & 31) * 4) * 4u;
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (r < S) v[u][d][r] = ptx::ld_shared_cluster_v4(peer_base[r] + off);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = it0 + u * kThreads;
            if (it >= items) break;
            const int c = lo + (it >> 5), k = k0 + (it & 31) * 4;
            if (k >= p.K) continue;
            int a[D][4] = {};
#pragma unroll
            for (int d = 0; d < D; ++d) {
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    if (r < S) {
                        a[d][0] += (int)v[u][d][r].x; a[d][1] += (int)v[u][d][r].y;
                        a[d][2] += (int)v[u][d][r].z; a[d][3] += (int)v[u][d][r].w;
                    }
                }
            }
            const float s = scale_s[c];
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                y[j] = digit_sum(a[0][j], a[1][j]);
                if (WIDE && s < 0.0f) y[j] = wide_digit_sum(y[j], a[D - 1][j]);
                y[j] = __fmul_rn(y[j], fabsf(s));
            }
            const uint32_t out_lo = pack_bf16x2_rn(y[0], y[1]), out_hi = pack_bf16x2_rn(y[2], y[3]);
            __nv_bfloat16* out = p.dx + (int64_t)(m0 + c) * p.K + k;
            if (vec) {
                *reinterpret_cast<uint2*>(out) = make_uint2(out_lo, out_hi);
            } else {
                uint16_t* o = reinterpret_cast<uint16_t*>(out);
                o[0] = (uint16_t)(out_lo & 0xffffu); o[1] = (uint16_t)(out_lo >> 16);
                o[2] = (uint16_t)(out_hi & 0xffffu); o[3] = (uint16_t)(out_hi >> 16);
            }
        }
    }
}

template <int ROWS>
__global__ void __launch_bounds__(kThreads, 1)
gemm_i8_grad_stream_kernel(const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmW, const GradParams p) {
    using L = GradStreamSmem<ROWS>;
    constexpr int STAGES = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kTmemSlotOff);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kAbortOff);
    volatile int* wide_s = reinterpret_cast<volatile int*>(smem + L::kWideOff);
    int* partial = reinterpret_cast<int*>(smem);  // [kColumns][128] once the ring has drained
    float* scale_s = reinterpret_cast<float*>(smem + L::kScaleOff);
    const uint32_t tiles_base = ptx::smem_u32(smem);
    const uint32_t bar_base = ptx::smem_u32(bars);
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    const uint32_t acc_full_bar = bar_base + 8u * (2 * STAGES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = (int)ptx::cluster_nctarank(), split = (int)ptx::cluster_ctarank();
    const int tiles_k = (p.K + 127) / 128, cluster = blockIdx.x / S, m_block = cluster / tiles_k;
    const int k0 = (cluster - m_block * tiles_k) * 128, m0 = m_block * ROWS;

    const int blocks = p.parts * p.part_blocks;
    const int nb0 = (int)((int64_t)blocks * split / S), nb1 = (int)((int64_t)blocks * (split + 1) / S);
    const int prologue = p.withhold_loads ? 0 : (nb1 - nb0) < STAGES ? (nb1 - nb0) : STAGES;
    auto load_weight = [&](uint32_t dst, int nb, uint32_t bar) {
        const int part = nb >= p.part_blocks ? 1 : 0;
        ptx::tma_load_2d(dst, &tmW, k0, part * p.part_rows + (nb - part * p.part_blocks) * BK, bar);
    };
    auto load_digits = [&](uint32_t dst, int nb, uint32_t bar) {   // rows past the block or the digit belong to no output
        ptx::tma_load_2d(dst, &tmD, nb * BK, m0, bar);
        ptx::tma_load_2d(dst + L::kDigitBytes, &tmD, nb * BK, p.M + m0, bar);
    };
    bool ok = true;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        ptx::mbar_init(acc_full_bar, 1);
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
        // the weight does not depend on the kernel before this one, the digits do
        for (int i = 0; i < prologue; ++i) {
            ptx::mbar_arrive_expect_tx(full_bar(i), L::kStageBytes);
            load_weight(tiles_base + i * L::kStageBytes, nb0 + i, full_bar(i));
        }
        ptx::grid_dependency_wait();
        const unsigned some_wide = any_wide<ROWS>(p, m0);
        for (int i = 0; i < prologue; ++i) load_digits(tiles_base + i * L::kStageBytes + L::kWBytes, nb0 + i, full_bar(i));
        *wide_s = some_wide != 0;   // its load is under way while the others are requested
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_slot), L::kTmemColumns);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    const bool wide = *wide_s != 0;
    const int passes = wide ? 2 : 1;   // both first digits at once, then the third

    if (warp == 0) {
        if (!p.withhold_loads && ptx::elect_one()) {
            int stage = prologue == STAGES ? 0 : prologue;
            uint32_t phase = prologue == STAGES ? 1u : 0u;
            for (int it = prologue; it < passes * (nb1 - nb0); ++it) {
                const bool third = it >= nb1 - nb0;
                const int nb = third ? it - (nb1 - nb0) + nb0 : nb0 + it;
                if (!ptx::mbar_wait_bounded(empty_bar(stage), phase ^ 1u, p.wait_limit_ns) || *abort_flag) {
                    report_wait_failure(kWaitEmptyStage);
                    *abort_flag = 1;
                    break;
                }
                const uint32_t dst = tiles_base + stage * L::kStageBytes;
                ptx::mbar_arrive_expect_tx(full_bar(stage), third ? L::kWBytes + L::kDigitBytes : L::kStageBytes);
                load_weight(dst, nb, full_bar(stage));
                if (third) ptx::tma_load_2d(dst + L::kWBytes, &tmD, nb * BK, 2 * p.M + m0, full_bar(stage));
                else load_digits(dst + L::kWBytes, nb, full_bar(stage));
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (ptx::elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool issued_all = true;
            for (int it = 0; it < passes * (nb1 - nb0); ++it) {
                if (!ptx::mbar_wait_bounded(full_bar(stage), phase, p.wait_limit_ns) || *abort_flag) {
                    report_wait_failure(kWaitFullStage);
                    *abort_flag = 1;
                    issued_all = false;
                    break;
                }
                ptx::tc_fence_after_sync();
                const bool third = it >= nb1 - nb0;
                const uint32_t d_tmem = tmem_base + (third ? 2 * ROWS : 0);
                const uint32_t idesc = third ? ptx::idesc_i8_a_mn(128, ROWS) : ptx::idesc_i8_a_mn(128, 2 * ROWS);
                const bool first = it == 0 || it == nb1 - nb0;
                const uint32_t src = tiles_base + stage * L::kStageBytes;
                const uint64_t adesc = ptx::smem_desc_mn_sw128(src);
                const uint64_t bdesc = ptx::smem_desc_k_sw128(src + L::kWBytes);
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k)
                    ptx::mma_i8_ss(d_tmem, adesc + (4096u >> 4) * k, bdesc + 2u * k, idesc, (!first || k != 0) ? 1u : 0u);
                ptx::tc_commit(empty_bar(stage));
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
            if (issued_all) ptx::tc_commit(acc_full_bar);
        }
    } else {
        // drain warps: scales and column sums first, then accumulator -> shared partial
        ptx::grid_dependency_wait();
        for (int i = threadIdx.x - 64; i < ROWS; i += kDrainThreads) {
            const unsigned size = m0 + i < p.M ? __ldcg(p.row_size + m0 + i) : 0u;
            const float s = digit_scale(top_of_size(size));
            scale_s[i] = is_wide(size) ? -s : s;
        }
        if (p.partial != nullptr) sum_columns(p, blockIdx.x * 4 + warp - 2, gridDim.x * 4);
        const int quarter = warp & 3, wcol = quarter * 32 + lane;  // column of W inside the tile = TMEM lane
        __syncwarp();
        if (nb1 > nb0) {
            if (!ptx::mbar_wait_bounded(acc_full_bar, 0, p.wait_limit_ns) || *abort_flag) {
                report_wait_failure(kWaitAccFull);
                *abort_flag = 1;
                ok = false;
            }
        }
        ptx::tc_fence_after_sync();
        __syncwarp();
        if (ok) {
            const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
            for (int cc = 0; cc < (wide ? L::kColumns : 2 * ROWS) / 32; ++cc) {
                uint32_t r[32];
                if (nb1 > nb0) {
                    ptx::tmem_ld_32x32b_x32(t_lane + cc * 32, r);
                    ptx::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = 0;  // a CTA without blocks contributes zero
                }
#pragma unroll
                for (int j = 0; j < 32; ++j) partial[(cc * 32 + j) * 128 + wcol] = (int)r[j];
            }
        }
    }

    // every CTA's partial is complete and visible to the cluster
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();
    ptx::grid_dependency_wait();

    {
        const int rows = min(ROWS, p.M - m0);
        const int lo = (int)((int64_t)rows * split / S), hi = (int)((int64_t)rows * (split + 1) / S);
        const uint32_t my_partial = ptx::smem_u32(partial);
        uint32_t peer_base[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) peer_base[r] = ptx::map_to_cta(my_partial, r < S ? r : 0);
        if (wide) reduce_gradient<ROWS, 1, true>(p, peer_base, S, m0, lo, hi, k0, scale_s);
        else if ((hi - lo) * 32 <= kThreads) reduce_gradient<ROWS, 1, false>(p, peer_base, S, m0, lo, hi, k0, scale_s);
        else reduce_gradient<ROWS, 2, false>(p, peer_base, S, m0, lo, hi, k0, scale_s);
    }

    // nobody leaves while a peer may still read its shared memory
    __syncthreads();
    ptx::cluster_sync();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, L::kTmemColumns);
    }
}

}  // namespace
}  // namespace w8a8

#endif  // W8A8_GEMM_I8_GRAD_KERNEL_CUH
