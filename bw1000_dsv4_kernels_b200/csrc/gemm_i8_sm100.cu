// W8A8 GEMM for sm_100a: C = bf16((float(A * B^T) * sa) * sb), int8 operands, int32
// accumulation on the 5th-generation tensor cores.
//
//   * A [M,K] and B [N,K] are both K-contiguous, so both MMA operands are "K-major".
//   * One CTA per SM, persistent over output tiles of 128 x BN.  Warp 0 issues TMA tile
//     loads (128-byte swizzle, 128 bytes of K per stage) into a ring of shared-memory
//     stages; warp 1 issues tcgen05.mma.kind::i8 (M128 x BN x K32) from one thread, four
//     per stage, accumulating in tensor memory; warps 2-5 drain the finished accumulator
//     with tcgen05.ld, apply the two scales and store bf16.  Tensor memory holds two
//     accumulators so that the drain of tile i overlaps the MMAs of tile i+1.
//   * The grouped (MoE) form puts an expert's weight rows on the MMA's M axis and its tokens
//     on the N axis (gemm_i8_wt_kernel.cuh); its work list is derived inside the kernel from
//     expert_offsets or masked_m (device memory), so no host synchronisation and no scratch
//     buffer is needed.
//   * Its group-scaled form (one activation scale per 128 of K) cannot defer scaling to
//     the end: each 128-wide K block is one accumulator that the drain warps fold into
//     fp32 registers as y = fma(float(acc), sa[row, g], y).
//   * Every wait on an mbarrier is bounded; a wait that gives up records a code in a
//     device status word and the CTA leaves its loops and frees its tensor memory.
//
// Arithmetic of the epilogue follows hip_kernels/w8a8_gemm_v5.hip:123 and
// hip_kernels/w8a8_gemm_intmm_fused.hip:34: (float(acc) * sa[row]) * sb[col] -> bf16.
#include <cuda.h>
#include <cuda_runtime.h>
#include <atomic>
#include <cuda_bf16.h>
#include <cstdint>
#include <cstdio>
#include <mutex>

#include "launch_common.h"
#include "sm100_ptx.cuh"
#include "w8a8_arith.cuh"
#include "gemm_i8_common.cuh"
#include "gemm_i8_tile_kernel.cuh"
#include "gemm_i8_pair_kernel.cuh"
#include "gemm_i8_fused_pair_kernel.cuh"
#include "gemm_i8_stream_kernels.cuh"
#include "gemm_i8_wt_kernel.cuh"
#include "gemm_i8_grad_kernel.cuh"

namespace w8a8 {

// Option of the calling thread: launch the dense GEMMs (weight-streaming kernels for M <= 256, CTA-pair
// kernel above) so that they may overlap the kernel before them on the stream (programmatic dependent
// launch).  Off by default.  Per thread, so that one thread that captures a CUDA graph with the option
// on does not change what other threads launch meanwhile.
static thread_local int g_overlap_previous = 0;
void set_overlap_previous_kernel(int on) { g_overlap_previous = on ? 1 : 0; }
int overlap_previous_kernel() { return g_overlap_previous; }

namespace {

// ------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess &&
            qres == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(sym);
    });
    return fn;
}

// 2-D uint8 tensor [rows, K] (K contiguous), box = 128 bytes of K x box_rows rows,
// 128-byte swizzle, out-of-range elements read as zero.
// Encoded tensor maps are kept per thread in a small table keyed by everything that goes into them (a
// descriptor holds an address and a shape, nothing that can go stale): a serving loop launches the same few
// GEMMs over the same buffers, and the grouped GEMM alone needs eleven maps per launch.
struct TileMapKey {
    const void* base;
    uint64_t rows, K;
    uint32_t box_rows;
    bool operator==(const TileMapKey& o) const {
        return base == o.base && rows == o.rows && K == o.K && box_rows == o.box_rows;
    }
};
struct TileMapCache {
    static constexpr int kEntries = 64;
    TileMapKey key[kEntries];
    CUtensorMap map[kEntries];
    int used = 0, next = 0;
};

int make_tile_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t K, uint32_t box_rows) {
    static thread_local TileMapCache cache;
    const TileMapKey k{base, rows, K, box_rows};
    for (int i = 0; i < cache.used; ++i) {
        if (cache.key[i] == k) {
            *map = cache.map[i];
            return 0;
        }
    }
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return fail(DSV4_ERR_DRIVER, "w8a8_gemm: cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[2] = {K, rows};
    const cuuint64_t strides[1] = {K};
    const cuuint32_t box[2] = {BK, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box,
                          estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        static thread_local char msg[160];
        snprintf(msg, sizeof msg, "w8a8_gemm: cuTensorMapEncodeTiled failed with CUresult %d (rows=%llu K=%llu)",
                 (int)r, (unsigned long long)rows, (unsigned long long)K);
        return fail(DSV4_ERR_DRIVER, msg);
    }
    const int slot = cache.used < TileMapCache::kEntries ? cache.used++ : cache.next;
    cache.next = (slot + 1) % TileMapCache::kEntries;
    cache.key[slot] = k;
    cache.map[slot] = *map;
    return 0;
}

// The status word's mirror in mapped host memory: allocated (host memory only) and published to the
// device on the first GEMM launch on each device.  A kernel whose bounded wait gives up writes its
// code there as well, so a later launch can refuse to go on without synchronising anything.
volatile int* host_status_mirror() {
    static volatile int* mirror[64] = {};
    static std::mutex mu;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    if (mirror[dev] != nullptr) return mirror[dev];
    std::lock_guard<std::mutex> lock(mu);
    if (mirror[dev] != nullptr) return mirror[dev];
    // a stream under capture (any thread's) must not be disturbed by what follows, none of which is for the graph
    struct Relaxed {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
        ~Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
    } relaxed;
    int* host = nullptr;
    int* device_view = nullptr;
    if (cudaHostAlloc(reinterpret_cast<void**>(&host), sizeof(int), cudaHostAllocMapped) != cudaSuccess ||
        cudaHostGetDevicePointer(reinterpret_cast<void**>(&device_view), host, 0) != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    *host = 0;
    if (cudaMemcpyToSymbol(g_host_status_mirror, &device_view, sizeof device_view) != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    mirror[dev] = host;
    return mirror[dev];
}

template <int BN, int STAGES>
int launch_variant(const CUtensorMap& tmA, const CUtensorMap& tmB, const Params& p, int max_tiles,
                   cudaStream_t st) {
    using L = Smem<BN, STAGES>;
    static_assert(L::kDynamic <= 227 * 1024, "shared memory limit");
    static bool opted_in[64] = {};
    if (!opt_in_shared_memory(gemm_i8_kernel<BN, STAGES>, L::kDynamic, opted_in))
        return fail(DSV4_ERR_LAUNCH, "w8a8_gemm: cannot raise the dynamic shared memory limit");
    int grid = sm_count();
    if (grid <= 0) return fail(DSV4_ERR_LAUNCH, "w8a8_gemm: no CUDA device");
    if (max_tiles < grid) grid = max_tiles;
    if (grid < 1) grid = 1;
    gemm_i8_kernel<BN, STAGES><<<grid, kThreads, L::kDynamic, st>>>(tmA, tmB, p);
    return check_launch("w8a8_gemm");
}

// How many clusters of `size` (at most eight) CTAs of a kernel the device can run at once (one CTA per SM, a cluster inside one
// GPC); asked once per kernel, device and cluster size, of a kernel that has its shared memory opted in (the answer is
// none otherwise).
using ClusterCounts = int[64][9];
template <typename Kernel>
int active_clusters(Kernel kernel, int size, int smem, ClusterCounts& cached) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || size < 1 || size > 8) return 0;
    if (cached[dev][size] == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(size * 64), 1, 1);
        cfg.blockDim = dim3(kThreads, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)size;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            n = -1;
        }
        cached[dev][size] = n > 0 ? n : -1;
    }
    return cached[dev][size] > 0 ? cached[dev][size] : 0;
}
template <int NTOK, int EPI>
int launch_stream_variant(const CUtensorMap& tmW, const CUtensorMap& tmX, const Params& p, int n_tiles, int splits,
                          cudaStream_t st) {
    using L = StreamSmem<NTOK>;
    static_assert(L::kDynamic <= 227 * 1024, "shared memory limit");
    static bool opted_in[64] = {};
    if (!opt_in_shared_memory(gemm_i8_stream_kernel<NTOK, EPI>, L::kDynamic, opted_in))
        return fail(DSV4_ERR_LAUNCH, "w8a8_gemm: cannot raise the dynamic shared memory limit");
    // fused epilogues: no wider a split than lets all clusters run at once (17 x 3000 x 1024, 24 tiles: 9.7 us split over six
    // CTAs, 5.6 over five)
    if constexpr (EPI != kEpiPlain) {
        static ClusterCounts cached = {};
        while (splits > 1 && active_clusters(gemm_i8_stream_kernel<NTOK, EPI>, splits, L::kDynamic, cached) < n_tiles) --splits;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n_tiles * splits), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = L::kDynamic;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_previous_kernel() ? 2 : 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, gemm_i8_stream_kernel<NTOK, EPI>, tmW, tmX, p);
    if (err != cudaSuccess) {
        cudaGetLastError();  // clear the sticky launch error
        static thread_local char msg[160];
        snprintf(msg, sizeof msg, "w8a8_gemm (weight streaming): %s", cudaGetErrorString(err));
        return fail(DSV4_ERR_LAUNCH, msg);
    }
    return check_launch("w8a8_gemm (weight streaming)");
}

template <int EPI>
bool stream_pair_opted_in() {
    static bool opted_in[64] = {};
    return opt_in_shared_memory(gemm_i8_stream_pair_kernel<EPI>, StreamPairSmem::kDynamic, opted_in);
}
template <int EPI>
int stream_pair_active_clusters(int splits) {
    static ClusterCounts cached = {};
    return active_clusters(gemm_i8_stream_pair_kernel<EPI>, 2 * splits, StreamPairSmem::kDynamic, cached);
}

template <int EPI>
int launch_stream_pair(const CUtensorMap& tmW, const CUtensorMap& tmX, const Params& p, int n_tiles, int splits,
                       cudaStream_t st) {
    using L = StreamPairSmem;
    static_assert(L::kDynamic <= 227 * 1024, "shared memory limit");
    if (!stream_pair_opted_in<EPI>())
        return fail(DSV4_ERR_LAUNCH, "w8a8_gemm: cannot raise the dynamic shared memory limit");
    // a cluster must fit into one GPC: take the widest K split whose clusters all run in one wave
    while (splits > 1 && stream_pair_active_clusters<EPI>(splits) < n_tiles) --splits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n_tiles * 2 * splits), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = L::kDynamic;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)(2 * splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_previous_kernel() ? 2 : 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, gemm_i8_stream_pair_kernel<EPI>, tmW, tmX, p);
    if (err != cudaSuccess) {
        cudaGetLastError();  // clear the sticky launch error
        static thread_local char msg[160];
        snprintf(msg, sizeof msg, "w8a8_gemm (weight streaming, CTA pairs): %s", cudaGetErrorString(err));
        return fail(DSV4_ERR_LAUNCH, msg);
    }
    return check_launch("w8a8_gemm (weight streaming, CTA pairs)");
}

// Grouped GEMM, weights on the MMA's M axis: one CTA per SM walks the (expert, token chunk, weight tile) items.
template <bool GS, bool STAGED = false>
int launch_wt_variant(const CUtensorMap& tmW, const WtMaps& xmaps, const Params& p, cudaStream_t st) {
    using L = WtSmem<GS, STAGED>;
    static_assert(L::kDynamic <= 227 * 1024, "shared memory limit");
    static bool opted_in[64] = {};
    if (!opt_in_shared_memory(gemm_i8_wt_kernel<GS, STAGED>, L::kDynamic, opted_in))
        return fail(DSV4_ERR_LAUNCH, "grouped_gemm: cannot raise the dynamic shared memory limit");
    int grid = sm_count();
    if (grid <= 0) return fail(DSV4_ERR_LAUNCH, "grouped_gemm: no CUDA device");
    // at most this many items exist, whatever the segment lengths turn out to be
    const int64_t bound = ((int64_t)p.M / kWtChunk + p.E) * ((p.N + 127) / 128);
    if (bound < grid) grid = (int)bound;
    if (grid < 1) grid = 1;
    gemm_i8_wt_kernel<GS, STAGED><<<grid, GS ? 576 : 192, L::kDynamic, st>>>(tmW, xmaps, p);
    return check_launch("grouped_gemm");
}

// bf16 [rows, cols] view with row stride ldc elements: box = 64 columns x 128 rows, 128-byte swizzle
int make_store_map(CUtensorMap* map, void* base, uint64_t rows, uint64_t cols, uint64_t ldc) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return fail(DSV4_ERR_DRIVER, "w8a8_gemm: cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {ldc * 2};
    const cuuint32_t box[2] = {64, 128};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(DSV4_ERR_DRIVER, "w8a8_gemm_allgather: cuTensorMapEncodeTiled failed for an output map");
    return 0;
}

template <int STAGES, bool TMA_STORE>
int launch_pair_variant(const CUtensorMap& tmA, const CUtensorMap& tmB, const Params& p, const StoreMaps& smaps,
                        cudaStream_t st) {
    using L = PairSmem<STAGES, TMA_STORE>;
    static_assert(L::kDynamic <= 227 * 1024, "shared memory limit");
    static bool opted_in[64] = {};
    if (!opt_in_shared_memory(gemm_i8_pair_kernel<STAGES, TMA_STORE>, L::kDynamic, opted_in))
        return fail(DSV4_ERR_LAUNCH, "w8a8_gemm: cannot raise the dynamic shared memory limit");
    const int tiles = ((p.M + 255) / 256) * ((p.N + 255) / 256);
    int pairs = sm_count() / 2;
    if (pairs <= 0) return fail(DSV4_ERR_LAUNCH, "w8a8_gemm: no CUDA device");
    if (tiles < pairs) pairs = tiles;
    if (!overlap_previous_kernel()) {
        gemm_i8_pair_kernel<STAGES, TMA_STORE><<<2 * pairs, kThreads, L::kDynamic, st>>>(tmA, tmB, p, smaps);
        return check_launch("w8a8_gemm");
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * pairs), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = L::kDynamic;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, gemm_i8_pair_kernel<STAGES, TMA_STORE>, tmA, tmB, p, smaps);
    if (err != cudaSuccess) {
        cudaGetLastError();  // clear the sticky launch error
        static thread_local char msg[160];
        snprintf(msg, sizeof msg, "w8a8_gemm (CTA pairs): %s", cudaGetErrorString(err));
        return fail(DSV4_ERR_LAUNCH, msg);
    }
    return check_launch("w8a8_gemm");
}

// Width of the fused pair kernel's tiles (rows of B, a multiple of `unit`).  256 wherever that gives every pair a tile: a
// narrower tile moves more operand bytes per MMA, and under the power cap a partly empty last round costs less than its
// share (224 tiles at 256 on 74 pairs 203 us, 199 at 224, 208 at 160, 270 at 128).  Problems of fewer tiles take the
// widest tile that still spreads them over the pairs (40 x 256 columns of a gated 333 x 1024 x 1040: 12.2 us at 256, 9.4
// at 64).
int fused_tile_n(int tiles_m, int rows, int unit, int pairs) {
    int w = 256;
    while (w > 64 && (int64_t)tiles_m * ((rows + w - unit - 1) / (w - unit)) <= pairs) w -= unit;
    return w;
}

template <int EPI, int ACT>
int launch_fused_pair(const GemmArgs& a, Params p, cudaStream_t st) {
    using L = FusedPairSmem;
    static_assert(L::kDynamic <= 227 * 1024, "shared memory limit");
    static bool opted_in[64] = {};
    if (!opt_in_shared_memory(gemm_i8_fused_pair_kernel<EPI, ACT>, L::kDynamic, opted_in))
        return fail(DSV4_ERR_LAUNCH, "w8a8_linear: cannot raise the dynamic shared memory limit");
    int pairs = sm_count() / 2;
    if (pairs <= 0) return fail(DSV4_ERR_LAUNCH, "w8a8_linear: no CUDA device");
    const int w_rows = is_gated(EPI) ? 2 * a.N : a.N, tiles_m = (a.M + 255) / 256;
    p.tile_n = fused_tile_n(tiles_m, w_rows, is_gated(EPI) ? 64 : 32, pairs);
    const int out_n = is_gated(EPI) ? p.tile_n / 2 : p.tile_n;
    p.size_slots = 2 * ((a.N + out_n - 1) / out_n);   // a tile's chunks go to two warps per row in turn
    if (a.size_slots != nullptr) *a.size_slots = p.size_slots;
    CUtensorMap tmA, tmB;
    if (int rc = make_tile_map(&tmA, a.A, (uint64_t)a.M, (uint64_t)a.K, BM)) return rc;
    if (int rc = make_tile_map(&tmB, a.B, (uint64_t)w_rows, (uint64_t)a.K, (uint32_t)(p.tile_n / 2))) return rc;
    const int64_t tiles = (int64_t)tiles_m * ((a.N + out_n - 1) / out_n);
    if (tiles > INT32_MAX) return fail(DSV4_ERR_ARG, "w8a8_linear: too many tiles");
    if (tiles < pairs) pairs = (int)tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * pairs), 1, 1);
    cfg.blockDim = dim3(kFusedThreads, 1, 1);
    cfg.dynamicSmemBytes = L::kDynamic;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_previous_kernel() ? 1 : 0;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, gemm_i8_fused_pair_kernel<EPI, ACT>, tmA, tmB, p);
    if (err != cudaSuccess) {
        cudaGetLastError();  // clear the sticky launch error
        static thread_local char msg[160];
        snprintf(msg, sizeof msg, "w8a8_linear (CTA pairs): %s", cudaGetErrorString(err));
        return fail(DSV4_ERR_LAUNCH, msg);
    }
    return check_launch("w8a8_linear");
}

// The CTA-pair streaming kernel over `blocks` blocks of tokens of about the same length
int stream_block_tokens(int M, int blocks) { return ((M + blocks - 1) / blocks + 31) / 32 * 32; }
template <int EPI>
int launch_stream_blocks(const GemmArgs& a, Params p, int blocks, int pair_tiles, int splits, cudaStream_t st) {
    const int w_rows = is_gated(EPI) ? 2 * a.N : a.N;
    p.block_m = EPI == kEpiPlain ? 256 : stream_block_tokens(a.M, blocks);
    CUtensorMap tmW, tmX;
    if (int rc = make_tile_map(&tmW, a.B, (uint64_t)w_rows, (uint64_t)a.K, is_gated(EPI) ? 64 : 128)) return rc;
    if (int rc = make_tile_map(&tmX, a.A, (uint64_t)a.M, (uint64_t)a.K, (uint32_t)(p.block_m / 2))) return rc;  // a CTA's half of the tokens
    return launch_stream_pair<EPI>(tmW, tmX, p, pair_tiles * blocks, splits, st);
}

// Whether a K split over `splits` CTAs or pairs pays for a block of so many tokens: a K block costs 0.3 us, the split saves
// (1 - 1 / splits) of them, and the sum of the partials through shared memory, with its epilogue, costs 6 to 9 us more for 256
// tokens than the tile kernel's drain.
bool split_pays(int tokens, int splits, int k_blocks) { return k_blocks * (splits - 1) >= tokens / 8 * splits; }

// Half as many tiles as there are pairs of SMs (37 on a B200): with so few, a tile's K is worth splitting
int few_tiles() { return sm_count() / 4; }

// Whether few tokens with a fused epilogue go to the weight-streaming kernel rather than the tiles of 256 tokens, whose drain
// is faster and whose tiles are as narrow as 64 outputs.  Measured (tiles / streaming, with bias, GELU, residual): 128 x 4096
// x 1024 5.6 / 9.0 us, x 7168 14.7 / 14.8; 128 x 18432 x 4096 28.2 / 29.2; 65 x 18432 x 4096 27.2 / 24.0; 65 x 4096 x 1024
// 6.2 / 7.6; 59 x 3000 x 64 6.6 / 9.0, x 512 7.3 / 6.6; 33 x 18432 x 1024 14.4 / 9.7; 256 x 400 x 4096 12.4 / 8.3 (blocks of 32).
bool fused_few(int M, int ntok, int w_rows, int n_tiles, int splits, int k_blocks) {
    const bool few = n_tiles <= few_tiles();
    if (M <= 64) return M <= 32 || k_blocks > 2 || !few;
    if (M > 128 && w_rows >= 256 && ntok > 64) return false;
    return few ? split_pays(min(M, ntok), splits, k_blocks) : M <= 96;
}

// K split of more tokens over the streaming kernel's pairs, or 0 where the tile kernel is faster.  Measured (tiles / this
// one): 600 x 1000 x 8192 with bias, GELU, residual 24.3 / 16.8 us, x 2048 10.3 / 13.4; gated 300 x 2048 x 7168 20.4 / 17.5,
// 400 x 500 x 4096 12.0 / 12.4; 200 x 2000 x 2048 9.0 / 12.8.
template <int EPI>
int stream_blocks_splits(int M, int pair_tiles, int blocks, int k_blocks) {
    const int64_t clusters = (int64_t)pair_tiles * blocks;
    if (clusters > few_tiles() || !stream_pair_opted_in<EPI>()) return 0;
    for (int s = k_blocks < 4 ? k_blocks : 4; s > 1; --s)
        if (stream_pair_active_clusters<EPI>(s) >= clusters) return split_pays(stream_block_tokens(M, blocks), s, k_blocks) ? s : 0;
    return 0;
}

// Dense problems: the kernel by the number of tokens and tiles.  A gated weight [2 N, K] gives N outputs, and each weight
// tile takes half its rows from the gates and half from the ups, so its N counts twice.
template <int EPI>
int gemm_i8_dense(const GemmArgs& a, Params p, int bn, cudaStream_t st) {
    constexpr bool kGated = is_gated(EPI);
    const int sms = sm_count();
    const int w_rows = kGated ? 2 * a.N : a.N;
    CUtensorMap tmA, tmB;
    const int k_blocks = (a.K + BK - 1) / BK;
    p.size_slots = kGated ? (a.N + 63) / 64 : (a.N + 127) / 128;   // the streaming kernels' tiles; launch_fused_pair has its own
    if (a.size_slots != nullptr) *a.size_slots = p.size_slots;
    // Few tokens: stream the weight once, tokens on the MMA's N axis, K split over a cluster
    if (a.M <= 256 && a.npeers == 0) {
        if (EPI == kEpiPlain && a.M > 128 && a.N >= 256) {
            // 129..256 tokens: CTA pairs halve the token traffic per SM
            const int pair_tiles = (a.N + 255) / 256;
            int psplits = sms / (2 * pair_tiles);
            if (psplits > 4) psplits = 4;
            if (psplits > k_blocks) psplits = k_blocks;
            if (psplits < 1) psplits = 1;
            return launch_stream_blocks<EPI>(a, p, 1, pair_tiles, psplits, st);
        }
        const int n_tiles = kGated ? (a.N + 63) / 64 : (a.N + 127) / 128;
        int splits = sms / n_tiles;
        if (splits > 8) splits = 8;
        if (splits > k_blocks) splits = k_blocks;
        if (splits < 1) splits = 1;
        // fused epilogues: blocks of at most 128 tokens, several clusters of them for more
        int ntok = a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 64 ? 64 : a.M <= 128 || EPI != kEpiPlain ? 128 : 256;
        int tiles = n_tiles;
        if constexpr (EPI != kEpiPlain) {
            if (a.M > 128) tiles *= 2;
            // blocks of fewer tokens while the clusters would fill less than half the SMs (200 x 200 x 8192 12.7 -> 7.3 us,
            // 90 x 60 x 2048 7.6 -> 5.5; 17 x 1000 x 4096 5.9 -> 6.2 with 16, hence not below 32)
            while (ntok > 32 && tiles * splits * 2 <= sms) {
                ntok /= 2;
                tiles = n_tiles * ((a.M + ntok - 1) / ntok);
            }
        }
        if (EPI == kEpiPlain || fused_few(a.M, ntok, w_rows, n_tiles, splits, k_blocks)) {
            int rc4 = make_tile_map(&tmA, a.B, (uint64_t)w_rows, (uint64_t)a.K, kGated ? 64 : 128);   // weights
            if (rc4) return rc4;
            rc4 = make_tile_map(&tmB, a.A, (uint64_t)a.M, (uint64_t)a.K, (uint32_t)ntok);  // tokens
            if (rc4) return rc4;
            switch (ntok) {
                case 16: return launch_stream_variant<16, EPI>(tmA, tmB, p, tiles, splits, st);
                case 32: return launch_stream_variant<32, EPI>(tmA, tmB, p, tiles, splits, st);
                case 64: return launch_stream_variant<64, EPI>(tmA, tmB, p, tiles, splits, st);
                case 128: return launch_stream_variant<128, EPI>(tmA, tmB, p, tiles, splits, st);
                default:
                    if constexpr (EPI == kEpiPlain) return launch_stream_variant<256, EPI>(tmA, tmB, p, tiles, splits, st);
                    return fail(DSV4_ERR_ARG, "w8a8_linear: more tokens than a block has");   // ntok is one of those above
            }
        }
    }
    if constexpr (EPI != kEpiPlain) {
        // More tokens, few tiles, long K: CTA pairs over blocks of tokens; otherwise tiles of 256 tokens
        const int pair_tiles = kGated ? (a.N + 127) / 128 : (a.N + 255) / 256;
        const int blocks = (a.M + 255) / 256;
        const int splits = stream_blocks_splits<EPI>(a.M, pair_tiles, blocks, k_blocks);
        if (splits > 0) return launch_stream_blocks<EPI>(a, p, blocks, pair_tiles, splits, st);
        switch (a.act) {
            case kActRelu: return launch_fused_pair<EPI, kActRelu>(a, p, st);
            case kActGelu: return launch_fused_pair<EPI, kActGelu>(a, p, st);
            case kActGeluTanh: return launch_fused_pair<EPI, kActGeluTanh>(a, p, st);
            case kActSilu: return launch_fused_pair<EPI, kActSilu>(a, p, st);
            default:   // the entry points refuse a gated projection without an activation, and a gradient of none needs no z
                if constexpr (EPI == kEpiLinear) return launch_fused_pair<EPI, kActNone>(a, p, st);
                return fail(DSV4_ERR_ARG, "w8a8_linear: unknown activation");
        }
    }
    // Dense problems with more than one 128-row tile go to the CTA-pair kernel
    if (a.M > 128 && (int64_t)((a.M + 255) / 256) * ((a.N + 255) / 256) >= sms / 4) {
        int rc2 = make_tile_map(&tmA, a.A, (uint64_t)a.M, (uint64_t)a.K, BM);
        if (rc2) return rc2;
        rc2 = make_tile_map(&tmB, a.B, (uint64_t)w_rows, (uint64_t)a.K, 128);
        if (rc2) return rc2;
        StoreMaps smaps;
        smaps.count = 0;
        if (a.npeers > 0) {
            // fused all-gather: tile stores through tensor maps of this rank's slab and of every peer's
            rc2 = make_store_map(&smaps.m[0], a.C, (uint64_t)a.M, (uint64_t)a.N, (uint64_t)p.ldc);
            if (rc2) return rc2;
            for (int d = 0; d < a.npeers; ++d) {
                rc2 = make_store_map(&smaps.m[1 + d], a.peerC[d], (uint64_t)a.M, (uint64_t)a.N, (uint64_t)p.ldc);
                if (rc2) return rc2;
            }
            smaps.count = 1 + a.npeers;
            return launch_pair_variant<4, true>(tmA, tmB, p, smaps, st);
        }
        return launch_pair_variant<6, false>(tmA, tmB, p, smaps, st);
    }
    int rc = make_tile_map(&tmA, a.A, (uint64_t)a.M, (uint64_t)a.K, BM);
    if (rc) return rc;
    rc = make_tile_map(&tmB, a.B, (uint64_t)w_rows, (uint64_t)a.K, (uint32_t)bn);
    if (rc) return rc;
    const int max_tiles = ((a.M + BM - 1) / BM) * ((a.N + bn - 1) / bn);
    switch (bn) {
        case 256: return launch_variant<256, 4>(tmA, tmB, p, max_tiles, st);
        case 128: return launch_variant<128, 6>(tmA, tmB, p, max_tiles, st);
        case 64: return launch_variant<64, 8>(tmA, tmB, p, max_tiles, st);
        default: return launch_variant<32, 10>(tmA, tmB, p, max_tiles, st);
    }
}

}  // namespace

int refuse_after_failed_wait() {
    volatile int* mirror = host_status_mirror();
    const int site = mirror != nullptr ? *mirror : 0;
    if (site == 0) return 0;
    *mirror = 0;
    static thread_local char msg[160];
    snprintf(msg, sizeof msg, "w8a8_gemm: an earlier kernel on this device gave up a bounded wait (site %d); "
             "nothing was launched; dsv4_device_status reads and clears the device's word", site);
    return fail(DSV4_ERR_DEVICE_WAIT, msg);
}

int gemm_i8(const GemmArgs& a, cudaStream_t st) {
    const bool grouped = a.offsets != nullptr || a.masked_m != nullptr;
    if (a.M < 0 || a.N < 0 || a.K < 0) return fail(DSV4_ERR_ARG, "w8a8_gemm: negative size");
    if (a.M == 0 || a.N == 0) return 0;
    if (a.K == 0) return fail(DSV4_ERR_ARG, "w8a8_gemm: K must be positive");
    if (a.A == nullptr || a.B == nullptr || (a.C == nullptr && a.row_ptr == nullptr))
        return fail(DSV4_ERR_ARG, "w8a8_gemm: null pointer");
    if (a.row_ptr != nullptr && (!grouped || a.sa_groups != 1 || a.out_i32 || a.npeers != 0))
        return fail(DSV4_ERR_ARG, "grouped_gemm_scatter: row destinations exist only for the grouped GEMM with per-token scales");
    if (!a.out_i32 && (a.sa == nullptr || a.sb == nullptr)) return fail(DSV4_ERR_ARG, "w8a8_gemm: null scale pointer");
    if (a.K % 16 != 0) return fail(DSV4_ERR_ARG, "w8a8_gemm: K must be a multiple of 16 (TMA row stride)");
    if ((reinterpret_cast<uintptr_t>(a.A) & 15) || (reinterpret_cast<uintptr_t>(a.B) & 15))
        return fail(DSV4_ERR_ARG, "w8a8_gemm: A and B must be 16-byte aligned");
    if (grouped && (a.E <= 0 || a.E > kMaxExperts)) return fail(DSV4_ERR_ARG, "grouped_gemm: E must be in 1..1024");
    if (a.sa_groups != 1) {
        if (!grouped) return fail(DSV4_ERR_ARG, "w8a8_gemm: group scales exist only for the grouped GEMM");
        if (a.out_i32) return fail(DSV4_ERR_ARG, "w8a8_gemm: raw accumulators exist only for per-token scaling");
        if (a.K % 128 != 0 || a.sa_groups != a.K / 128)
            return fail(DSV4_ERR_ARG, "grouped_gemm: group scales need K % 128 == 0 and sa_groups == K / 128");
    }

    if (int rc = refuse_after_failed_wait()) return rc;

    Params p;
    p.wait_limit_ns = a.test_wait_limit_ns ? a.test_wait_limit_ns : ptx::kWaitLimitNs;
    p.withhold_loads = a.test_withhold_loads;
    p.sa = a.sa; p.sb = a.sb; p.C = a.C; p.offsets = a.offsets;
    p.masked_m = a.masked_m; p.max_m = a.max_m;
    p.row_ptr = a.row_ptr;
    p.M = a.M; p.N = a.N; p.K = a.K; p.E = grouped ? a.E : 1;
    p.ldc = a.ldc > 0 ? a.ldc : a.N;
    p.sa_groups = a.sa_groups; p.out_i32 = a.out_i32;
    if (p.ldc < a.N) return fail(DSV4_ERR_ARG, "w8a8_gemm: ldc smaller than N");
    p.bias = static_cast<const __nv_bfloat16*>(a.bias);
    p.resid = static_cast<const __nv_bfloat16*>(a.resid);
    p.ldr = a.ldr; p.act = a.act; p.inter = a.N; p.row_sizes = static_cast<RowSize*>(a.row_sizes);
    p.up_col = a.up_col; p.tile_n = 256;
    if (a.epilogue != kEpiPlain && (grouped || a.out_i32 || a.npeers != 0))
        return fail(DSV4_ERR_ARG, "w8a8_linear: the fused epilogues exist for the dense GEMM with bf16 output");
    {
        // groups of m-tiles whose rows of A (256 x K bytes each) take at most 32 MB, all about equally large
        const int tiles_m = (a.M + 255) / 256;
        const int64_t tile_bytes = (int64_t)256 * a.K;
        int gm_max = (int)((int64_t)32 * 1024 * 1024 / (tile_bytes > 0 ? tile_bytes : 1));
        if (gm_max < 1) gm_max = 1;
        const int groups = (tiles_m + gm_max - 1) / gm_max;
        p.pair_group_m = groups > 0 ? (tiles_m + groups - 1) / groups : 1;
        if (p.pair_group_m < 1) p.pair_group_m = 1;
    }
    p.npeers = 0;
    for (int d = 0; d < 7; ++d) p.peerC[d] = nullptr;
    if (a.npeers > 0) {
        if (a.npeers > 7 || grouped || a.out_i32 || a.sa_groups != 1)
            return fail(DSV4_ERR_ARG, "w8a8_gemm_allgather: at most 7 peers, dense per-token-scaled bf16 output only");
        if (a.N % 32 != 0 || p.ldc % 8 != 0 || (reinterpret_cast<uintptr_t>(a.C) & 15))
            return fail(DSV4_ERR_ARG, "w8a8_gemm_allgather: N % 32 == 0, ldc % 8 == 0 and 16-byte aligned outputs required");
        for (int d = 0; d < a.npeers; ++d) {
            if (a.peerC[d] == nullptr || (reinterpret_cast<uintptr_t>(a.peerC[d]) & 15))
                return fail(DSV4_ERR_ARG, "w8a8_gemm_allgather: null or misaligned peer pointer");
            p.peerC[d] = a.peerC[d];
        }
        p.npeers = a.npeers;
    }

    const uint64_t b_rows = grouped ? (uint64_t)a.E * a.N : (uint64_t)a.N;
    const int sms = sm_count();
    const int tiles_m_bound = (a.M + BM - 1) / BM;

    // Tile width: 256 columns when that already gives every SM a tile, otherwise narrower
    // tiles so that a short, weight-streaming problem spreads over more SMs.
    int bn = 256;
    if ((int64_t)tiles_m_bound * ((a.N + 255) / 256) < sms) bn = 128;
    if (bn == 128 && (int64_t)tiles_m_bound * ((a.N + 127) / 128) < sms) bn = 64;
    if (bn == 64 && (int64_t)tiles_m_bound * ((a.N + 63) / 64) < sms) bn = 32;

    if (grouped) {
        CUtensorMap tmB;
        if (a.masked_m != nullptr && (a.offsets != nullptr || a.max_m <= 0 || (int64_t)a.E * a.max_m != a.M))
            return fail(DSV4_ERR_ARG, "grouped_gemm_masked: needs max_m > 0, M == E * max_m and no expert_offsets");
        if (a.out_i32) return fail(DSV4_ERR_ARG, "grouped_gemm: raw accumulators exist only for the dense GEMM");
        int rcw = make_tile_map(&tmB, a.B, b_rows, (uint64_t)a.K, 128);
        if (rcw) return rcw;
        WtMaps xmaps;
        for (int i = 0; i < kWtMaps; ++i) {
            rcw = make_tile_map(&xmaps.x[i], a.A, (uint64_t)a.M, (uint64_t)a.K, (uint32_t)(16 * (i + 1)));
            if (rcw) return rcw;
        }
        // Per-token scales: with a short K (the MoE down projection: 16 K blocks per item) the item's tile leaves
        // through shared memory in 256-byte row segments, which beats the sixth pipeline stage that the staging
        // tile displaces (0.72 against 0.79 ms on 256 experts of 128 rows, N = 7168, K = 2048); with a long K the
        // deeper pipeline wins (338 against 331 us on 64 experts, N = 4096, K = 7168).  Row destinations always
        // take the staged form.
        const bool short_k = (a.K + BK - 1) / BK <= 32 && p.ldc % 8 == 0 && (reinterpret_cast<uintptr_t>(a.C) & 15) == 0;
        if (a.sa_groups == 1 && (a.row_ptr != nullptr || short_k)) return launch_wt_variant<false, true>(tmB, xmaps, p, st);
        return a.sa_groups != 1 ? launch_wt_variant<true>(tmB, xmaps, p, st) : launch_wt_variant<false>(tmB, xmaps, p, st);
    }
    switch (a.epilogue) {
        case kEpiLinear: return gemm_i8_dense<kEpiLinear>(a, p, bn, st);
        case kEpiGated: return gemm_i8_dense<kEpiGated>(a, p, bn, st);
        case kEpiLinearGrad: return gemm_i8_dense<kEpiLinearGrad>(a, p, bn, st);
        case kEpiGatedGrad: return gemm_i8_dense<kEpiGatedGrad>(a, p, bn, st);
        default: return gemm_i8_dense<kEpiPlain>(a, p, bn, st);
    }
}

namespace {

// The gradient product of few rows.  The sum is split over as many CTAs (at most eight) as still let all clusters run at
// once.
//
// Returns without a launch where the kernel for many rows is faster (`launched` says so): clusters that do not run at once,
// or a sum so short that the rows' share of it is not worth joining the partials.  A block of 128 rows of W costs a pair of
// CTAs 0.75 us there (two digits), a CTA here up to 0.55 us, shared by S of them.  Measured (there / here, whole backward
// pass): gated 16 x 2048 x 7168 34.7 / 19.6 us, 64 x 9000 x 5008 69 / 38, 200 x 4096 x 7168 49 / 47, 600 x 8192 x 512 73 / 47,
// gated 700 x 300 x 1024 21.3 / 22.0.
template <int ROWS>
int launch_grad_stream(const GradientArgs& a, const GradParams& p, cudaStream_t st, bool& launched) {
    using L = GradStreamSmem<ROWS>;
    launched = false;
    static_assert(L::kDynamic <= 227 * 1024, "shared memory limit");
    static bool opted_in[64] = {};
    static ClusterCounts cached = {};
    if (!opt_in_shared_memory(gemm_i8_grad_stream_kernel<ROWS>, L::kDynamic, opted_in))
        return fail(DSV4_ERR_LAUNCH, "w8a8 backward: cannot raise the dynamic shared memory limit");
    const int64_t clusters = (int64_t)((a.K + 127) / 128) * ((a.M + ROWS - 1) / ROWS);
    const int blocks = a.parts * p.part_blocks;
    int splits = blocks < 8 ? blocks : 8;
    while (splits > 0 && active_clusters(gemm_i8_grad_stream_kernel<ROWS>, splits, L::kDynamic, cached) < clusters) --splits;
    if (blocks * (3 * splits - 2) < 20 * splits || splits == 0) return 0;
    launched = true;
    CUtensorMap tmD, tmW;
    if (int rc = make_tile_map(&tmD, a.digits, (uint64_t)3 * a.M, (uint64_t)a.parts * a.part_pitch, ROWS)) return rc;
    if (int rc = make_tile_map(&tmW, a.W, (uint64_t)a.parts * a.part_rows, (uint64_t)a.K, 128)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * splits), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = L::kDynamic;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, gemm_i8_grad_stream_kernel<ROWS>, tmD, tmW, p) != cudaSuccess) {
        cudaGetLastError();  // clear the sticky launch error
        return fail(DSV4_ERR_LAUNCH, "w8a8 backward: launch of the gradient product");
    }
    return check_launch("w8a8 backward");
}

}  // namespace

// dx = dz_scaled W for digits that split_gradient_kernel wrote (see gemm_i8_grad_kernel.cuh)
int gemm_i8_gradient(const GradientArgs& a, cudaStream_t st) {
    using L = FusedPairSmem;
    static bool opted_in[64] = {};
    if (!opt_in_shared_memory(gemm_i8_grad_kernel, L::kDynamic, opted_in))
        return fail(DSV4_ERR_LAUNCH, "w8a8 backward: cannot raise the dynamic shared memory limit");
    GradParams p = {};
    p.row_size = a.row_size;
    p.wide = a.wide;
    p.dx = static_cast<__nv_bfloat16*>(a.dx);
    p.M = a.M; p.K = a.K;
    p.parts = a.parts; p.part_rows = a.part_rows; p.part_blocks = a.part_pitch / BK;
    p.wait_limit_ns = a.test_wait_limit_ns ? a.test_wait_limit_ns : ptx::kWaitLimitNs;
    p.withhold_loads = a.test_withhold_loads;
    const int pitch = a.parts * a.part_pitch;
    // groups of m-tiles whose two digits take at most 32 MB, as in gemm_i8
    const int tiles_m = (a.M + 255) / 256;
    int gm_max = (int)((int64_t)32 * 1024 * 1024 / ((int64_t)512 * pitch));
    if (gm_max < 1) gm_max = 1;
    const int groups = (tiles_m + gm_max - 1) / gm_max;
    p.group_m = (tiles_m + groups - 1) / groups;
    p.partial = a.partial;
    p.row_blocks = a.row_blocks;
    p.dbias = a.dbias;
    // rows of a block: as few as still fill half the SMs with clusters of eight, since a CTA's load is its digits' (83 rows,
    // gated 15696 x 96: 49 us with 128, 42 with 16; 128 rows, 4096 x 512: 26 and 22)
    int rows = a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 64 ? 64 : 128;
    while (rows > 16 && (int64_t)((a.K + 127) / 128) * ((a.M + rows - 1) / rows) * 16 <= sm_count()) rows /= 2;
    bool launched;
    const int rc = rows == 16   ? launch_grad_stream<16>(a, p, st, launched)
                   : rows == 32 ? launch_grad_stream<32>(a, p, st, launched)
                   : rows == 64 ? launch_grad_stream<64>(a, p, st, launched)
                                : launch_grad_stream<128>(a, p, st, launched);
    if (rc != 0 || launched) return rc;
    CUtensorMap tmD, tmW;
    if (int rc = make_tile_map(&tmD, a.digits, (uint64_t)3 * a.M, (uint64_t)pitch, BM)) return rc;
    if (int rc = make_tile_map(&tmW, a.W, (uint64_t)a.parts * a.part_rows, (uint64_t)a.K, 128)) return rc;
    const int64_t tiles = (int64_t)tiles_m * ((a.K + 255) / 256);
    int pairs = sm_count() / 2;
    if (pairs <= 0) return fail(DSV4_ERR_LAUNCH, "w8a8 backward: no CUDA device");
    if (tiles > INT32_MAX) return fail(DSV4_ERR_ARG, "w8a8 backward: too many tiles");
    if (tiles < pairs) pairs = (int)tiles;
    return launch_after(gemm_i8_grad_kernel, dim3(2 * pairs), dim3(kFusedThreads), L::kDynamic, st, "w8a8 backward", tmD, tmW, p);
}

// ------------------------------------------------------------------------------------
// int32 [M,N] -> bf16 with the two scales (hip_kernels/w8a8_gemm_intmm_fused.hip:22-36)
// ------------------------------------------------------------------------------------
namespace {
__global__ void __launch_bounds__(256) scale_convert_kernel(const int* __restrict__ acc,
                                                            const float* __restrict__ sa,
                                                            const float* __restrict__ sb,
                                                            __nv_bfloat16* __restrict__ out, int M, int N) {
    const int64_t total = (int64_t)M * N;
    for (int64_t f = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; f < total;
         f += (int64_t)gridDim.x * blockDim.x) {
        const int row = (int)(f / N), col = (int)(f % N);
        out[f] = __float2bfloat16_rn(__fmul_rn(__fmul_rn(__int2float_rn(acc[f]), sa[row]), sb[col]));
    }
}
}  // namespace

int scale_convert(const void* acc, const void* sa, const void* sb, void* out, int M, int N, cudaStream_t st) {
    if (M == 0 || N == 0) return 0;
    int64_t blocks = ((int64_t)M * N + 255) / 256;
    if (blocks > (1 << 20)) blocks = 1 << 20;
    scale_convert_kernel<<<(int)blocks, 256, 0, st>>>(static_cast<const int*>(acc), static_cast<const float*>(sa),
                                                      static_cast<const float*>(sb),
                                                      static_cast<__nv_bfloat16*>(out), M, N);
    return check_launch("scale_convert");
}

int read_device_status(cudaStream_t st, int* out) {
    if (cudaStreamSynchronize(st) != cudaSuccess) return fail(DSV4_ERR_LAUNCH, "device_status: stream synchronise failed");
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_device_status, sizeof(int)) != cudaSuccess)
        return fail(DSV4_ERR_LAUNCH, "device_status: cannot read the status word");
    if (v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_device_status, &zero, sizeof(int));
        if (volatile int* mirror = host_status_mirror()) *mirror = 0;
    }
    if (v == 0) {
        const int rc = read_row_status(&v);
        if (rc) return rc;
    }
    if (out) *out = v;
    return 0;
}

}  // namespace w8a8
