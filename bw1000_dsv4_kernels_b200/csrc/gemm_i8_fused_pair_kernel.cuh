// Private part of gemm_i8_sm100.cu: the CTA-pair kernel behind w8a8_linear, w8a8_gated and their gradients wherever
// the weight-streaming kernels are not faster (fused_few, stream_blocks_splits).  Pairs, pipeline and barriers are those of gemm_i8_pair_kernel; what differs:
//
//   * The tile is 256 rows by p.tile_n rows of B, chosen per launch (fused_tile_n): with one tile per pair at a time, a
//     problem of 224 tiles on 74 pairs takes four rounds for 3.03 rounds of work at a width of 256.
//   * A gated tile takes its B rows in two halves: the even CTA loads tile_n / 2 gate rows, the odd CTA the tile_n / 2 up
//     rows of the same outputs, so that accumulator columns [0, tile_n / 2) are gates, the others ups, and one thread
//     has both of an output.
//   * Eight drain warps per CTA instead of four, two per scheduler: the activations, the residual and the fp32 gradients
//     make the drain several times as long as that of the plain epilogue, and one warp per scheduler waits for its own
//     results most of the time (a GELU gradient tile took 40 us with four warps, its MMAs 16).  Warps w and w + 4 own the
//     same 32 rows and take the tile's 32-column chunks in turn.
//   * A chunk's residual or incoming gradient is requested one chunk ahead, the first before the accumulator is waited for.
//   * The activation is a template parameter and the chunk loop is not unrolled: with a choice of five activations inside
//     and four chunks unrolled, a tile ran through half a megabyte of instructions once and waited for their fetches.
#ifndef W8A8_GEMM_I8_FUSED_PAIR_KERNEL_CUH
#define W8A8_GEMM_I8_FUSED_PAIR_KERNEL_CUH

#include "gemm_i8_common.cuh"
#include "gemm_i8_epilogues.cuh"
#include "gemm_i8_pair_kernel.cuh"

namespace w8a8 {
namespace {

constexpr int kFusedDrainWarps = 8;
constexpr int kFusedThreads = 64 + 32 * kFusedDrainWarps;

struct FusedPairSmem {
    static constexpr int kStages = 6;
    static constexpr int kABytes = BM * BK;
    static constexpr int kBBytes = 128 * BK;       // at most: tile_n / 2 rows
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kTilesBytes = kStages * kStageBytes;
    static constexpr int kColsOff = kTilesBytes;                                     // per warp: scales and biases of its chunks
    static constexpr int kTransposeOff = kColsOff + kFusedDrainWarps * 2 * 128 * 4;  // per warp: a 32 x 32 bf16 block
    static constexpr int kBarOff = kTransposeOff + kFusedDrainWarps * kBlockBytes;
    static constexpr int kNumBars = 2 * kStages + 4;
    static constexpr int kTmemSlotOff = kBarOff + kNumBars * 8;
    static constexpr int kAbortOff = kTmemSlotOff + 4;
    static constexpr int kTotal = kAbortOff + 4;
    static constexpr int kDynamic = kTotal + 1024;
};

template <int EPI, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFusedThreads, 1)
gemm_i8_fused_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Params p) {
    using L = FusedPairSmem;
    constexpr int STAGES = L::kStages;
    constexpr bool kGated = is_gated(EPI);
    constexpr bool kGrad = EPI == kEpiLinearGrad || EPI == kEpiGatedGrad;
    constexpr int kChunks = kGated ? 2 : 4;    // at most this many chunks of a tile belong to one warp
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kTmemSlotOff);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kAbortOff);

    const uint32_t tiles_base = ptx::smem_u32(smem);
    const uint32_t bar_base = ptx::smem_u32(bars);
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto acc_full_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
    auto acc_empty_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };

    ptx::grid_launch_dependents();  // a kernel launched to overlap this one may start its set-up and weight loads
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_ctarank();
    constexpr uint32_t kTmemCols = 512;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(acc_full_bar(a), 1);
            ptx::mbar_init(acc_empty_bar(a), 2 * kFusedDrainWarps);  // drain warps of both CTAs
        }
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
        ptx::prefetch_tensormap(&tmA);
        ptx::prefetch_tensormap(&tmB);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), kTmemCols);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();  // the peer's barriers exist before anything arrives on them
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    const int half_n = p.tile_n >> 1;                      // B rows that each CTA loads
    const int out_n = kGated ? half_n : p.tile_n;          // output columns of a tile
    const int tiles_m = (p.M + 255) / 256;
    const int tiles_n = (p.N + out_n - 1) / out_n;
    const int total = tiles_m * tiles_n;
    const PairTileOrder order{tiles_m, tiles_n, p.pair_group_m};
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int k_blocks = (p.K + BK - 1) / BK;
    const uint32_t pair_stage_bytes = 2u * (uint32_t)(L::kABytes + half_n * BK);

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        if (!p.withhold_loads && ptx::elect_one()) {
            auto b_row = [&](int nt) {
                return kGated ? nt * half_n + (int)rank * p.inter : nt * p.tile_n + (int)rank * half_n;
            };
            // The first ring-full needs no free-stage wait; its weight tiles are requested before the dependency wait and
            // its activations after it (see gemm_i8_pair_kernel).
            struct Cursor {
                int t, kb;
            };
            auto advance = [&](Cursor& c) {
                if (++c.kb == k_blocks) {
                    c.kb = 0;
                    c.t += npairs;
                }
            };
            const Cursor c0{pair, 0};
            int first = 0;
            for (Cursor c = c0; first < STAGES && c.t < total; ++first, advance(c)) {
                int mt, nt;
                order.at(c.t, mt, nt);
                if (rank == 0) ptx::mbar_arrive_expect_tx(full_bar(first), pair_stage_bytes);
                ptx::tma_load_2d_pair(tiles_base + first * L::kStageBytes + L::kABytes, &tmB, c.kb * BK, b_row(nt),
                                      ptx::map_to_cta(full_bar(first), 0));
            }
            ptx::grid_dependency_wait();
            Cursor c = c0;
            for (int i = 0; i < first; ++i, advance(c)) {
                int mt, nt;
                order.at(c.t, mt, nt);
                ptx::tma_load_2d_pair(tiles_base + i * L::kStageBytes, &tmA, c.kb * BK, mt * 256 + (int)rank * 128,
                                      ptx::map_to_cta(full_bar(i), 0));
            }
            int stage = first == STAGES ? 0 : first;
            uint32_t phase = first == STAGES ? 1u : 0u;
            while (c.t < total) {
                int mt, nt;
                order.at(c.t, mt, nt);
                for (; c.kb < k_blocks; ++c.kb) {
                    if (!ptx::mbar_wait_bounded(empty_bar(stage), phase ^ 1u, p.wait_limit_ns) || *abort_flag) {
                        report_wait_failure(kWaitEmptyStage);
                        *abort_flag = 1;
                        c.t = total;  // leave both loops
                        break;
                    }
                    const uint32_t a_dst = tiles_base + stage * L::kStageBytes;
                    const uint32_t leader_full = ptx::map_to_cta(full_bar(stage), 0);
                    if (rank == 0) ptx::mbar_arrive_expect_tx(full_bar(stage), pair_stage_bytes);
                    ptx::tma_load_2d_pair(a_dst, &tmA, c.kb * BK, mt * 256 + (int)rank * 128, leader_full);
                    ptx::tma_load_2d_pair(a_dst + L::kABytes, &tmB, c.kb * BK, b_row(nt), leader_full);
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
                if (c.t < total) {
                    c.kb = 0;
                    c.t += npairs;
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (even CTA only) ----------------
        if (rank == 0 && ptx::elect_one()) {
            const uint32_t idesc = ptx::idesc_i8(256, p.tile_n);
            int stage = 0;
            uint32_t phase = 0;
            int acc = 0;
            uint32_t acc_phase = 0;
            bool ok = true;
            for (int t = pair; t < total && ok; t += npairs) {
                if (!ptx::mbar_wait_bounded(acc_empty_bar(acc), acc_phase ^ 1u, p.wait_limit_ns) || *abort_flag) {
                    report_wait_failure(kWaitAccEmpty);
                    *abort_flag = 1;
                    break;
                }
                ptx::tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + acc * 256;
                for (int kb = 0; kb < k_blocks; ++kb) {
                    if (!ptx::mbar_wait_bounded(full_bar(stage), phase, p.wait_limit_ns) || *abort_flag) {
                        report_wait_failure(kWaitFullStage);
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    const uint32_t a_src = tiles_base + stage * L::kStageBytes;
                    const uint64_t adesc = ptx::smem_desc_k_sw128(a_src);
                    const uint64_t bdesc = ptx::smem_desc_k_sw128(a_src + L::kABytes);
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; ++k)
                        ptx::mma_i8_ss_pair(d_tmem, adesc + 2u * k, bdesc + 2u * k, idesc, (kb | k) != 0 ? 1u : 0u);
                    ptx::tc_commit_pair(empty_bar(stage), 0x3);  // frees the stage in both CTAs
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
                if (!ok) break;
                ptx::tc_commit_pair(acc_full_bar(acc), 0x3);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
        }
    } else {
        // ---------------- drain warps (both CTAs) ----------------
        ptx::grid_dependency_wait();  // before reading activation scales, residual or gradient, or writing C
        const int quarter = warp & 3, turn = (warp - 2) >> 2;
        // this warp's columns: scales [128], biases [128]; a gated chunk has 32 gate and 32 up columns
        float* cols = reinterpret_cast<float*>(smem + L::kColsOff) + (warp - 2) * 256;
        uint32_t* stage = reinterpret_cast<uint32_t*>(smem + L::kTransposeOff + (warp - 2) * kBlockBytes);
        const int chunks = out_n / 32;
        const bool has_res = p.resid != nullptr;
        const bool in_vec = block_vector_ok(p.resid, p.ldr, p.N), out_vec = block_vector_ok(p.C, p.ldc, p.N);
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int t = pair; t < total; t += npairs) {
            int mt, nt;
            order.at(t, mt, nt);
            const int n0 = nt * out_n;
            const int row0 = mt * 256 + (int)rank * 128 + quarter * 32, rows = min(32, p.M - row0), row = row0 + lane;
            const bool row_ok = lane < rows;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int c = n0 + (turn + 2 * i) * 32 + lane, cu = p.inter + c;
                const bool ok = turn + 2 * i < chunks && c < p.N;
                if constexpr (kGated) {
                    cols[i * 64 + lane] = ok ? __ldg(p.sb + c) : 0.0f;
                    cols[i * 64 + 32 + lane] = ok ? __ldg(p.sb + cu) : 0.0f;
                    cols[128 + i * 64 + lane] = ok && p.bias != nullptr ? __bfloat162float(p.bias[c]) : kNoBias;
                    cols[128 + i * 64 + 32 + lane] = ok && p.bias != nullptr ? __bfloat162float(p.bias[cu]) : kNoBias;
                } else {
                    cols[i * 32 + lane] = ok ? __ldg(p.sb + c) : 0.0f;
                    cols[128 + i * 32 + lane] = ok && p.bias != nullptr ? __bfloat162float(p.bias[c]) : kNoBias;
                }
            }
            // residual or incoming gradient of the chunk at column n; zeros where there is none
            auto fetch = [&](int cc) {
                const int n = n0 + cc * 32;
                if (EPI == kEpiGated || (!kGrad && !has_res) || cc >= chunks || n >= p.N || rows <= 0) return Fetched{};
                return fetch_block(p.resid, p.ldr, p.M, p.N, p.resid + (int64_t)row0 * p.ldr + n, {rows, p.N - n, in_vec}, lane);
            };
            Fetched fetched = fetch(turn);
            const float sa = row_ok ? __ldg(p.sa + row) : 0.0f;
            __syncwarp();
            if (!ptx::mbar_wait_bounded(acc_full_bar(acc), acc_phase, p.wait_limit_ns) || *abort_flag) {
                report_wait_failure(kWaitAccFull);
                *abort_flag = 1;
                break;
            }
            ptx::tc_fence_after_sync();
            const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * 256;
            RowSize size = RowSize::none();
            const float* col = cols;
#pragma unroll 1
            for (int cc = turn; cc < chunks; cc += 2, col += kGated ? 64 : 32) {
                const int n = n0 + cc * 32;
                if (n >= p.N || rows <= 0) break;
                uint32_t r[32], u[kGated ? 32 : 1];
                __syncwarp();  // tcgen05.ld is warp-collective
                ptx::tmem_ld_32x32b_x32(t_lane + cc * 32, r);
                if constexpr (kGated) ptx::tmem_ld_32x32b_x32(t_lane + half_n + cc * 32, u);
                Row32 in = {};
                if (kGrad || (EPI == kEpiLinear && has_res)) in = arrange_block(fetched, {rows, p.N - n, in_vec}, stage, lane);
                fetched = fetch(cc + 2);
                ptx::tmem_ld_wait();
                if constexpr (!kGrad) {
                    Row32 out;
                    if constexpr (kGated) out = gated_values<ACT>(r, u, sa, {col}, {col + 128}, {col + 32}, {col + 160});
                    else out = linear_values<ACT>(r, sa, {col}, {col + 128}, has_res, in);
                    store_block(static_cast<__nv_bfloat16*>(p.C) + (int64_t)row0 * p.ldc + n, p.ldc, out,
                                {rows, p.N - n, out_vec}, stage, lane);
                } else {
                    // dz has room for whole chunks; columns at or beyond N get zeros (their gradient was read as zero)
                    float* dz = static_cast<float*>(p.C) + (int64_t)row0 * p.ldc + n;
                    if constexpr (kGated)
                        gated_gradients<ACT>(r, u, sa, {col}, {col + 128}, {col + 32}, {col + 160}, in, dz, dz + p.up_col,
                                             p.ldc, rows, stage, lane, size);
                    else
                        linear_gradients<ACT>(r, sa, {col}, {col + 128}, in, dz, p.ldc, rows, stage, lane, size);
                }
            }
            if constexpr (kGrad) {
                if (row_ok) p.row_sizes[(int64_t)row * p.size_slots + 2 * nt + turn] = size;
            }
            ptx::tc_fence_before_sync();  // the accumulator reads above are ordered before the release below
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_cta(acc_empty_bar(acc), 0));
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1u;
        }
    }

    // ---------------- teardown ----------------
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();  // neither CTA leaves while the other may still touch its memory
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

}  // namespace
}  // namespace w8a8

#endif  // W8A8_GEMM_I8_FUSED_PAIR_KERNEL_CUH
