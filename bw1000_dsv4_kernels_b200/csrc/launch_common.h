// Status codes and error reporting shared by the launchers behind the C-ABI.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

#include "../../include/dsv4_w8a8.h"

namespace w8a8 {

// Records `msg` as the calling thread's last error and returns `code`.
int fail(int code, const char* msg);
// cudaGetLastError() after a launch; records "<what>: <cuda error string>" on failure.
int check_launch(const char* what);

#ifdef __CUDACC__
// SMs of the current device; 0 without one
inline int sm_count() {
    static thread_local int cached_dev = -1, cached = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev != cached_dev) {
        cudaDeviceGetAttribute(&cached, cudaDevAttrMultiProcessorCount, dev);
        cached_dev = dev;
    }
    return cached;
}

// More than 48 KB of dynamic shared memory needs an opt-in per kernel and per device; done on the
// first launch of each kernel on each device.
template <typename Kernel>
bool opt_in_shared_memory(Kernel kernel, int bytes, bool (&done)[64]) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && done[dev]) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        cudaGetLastError();  // clear the sticky error
        return false;
    }
    if (dev >= 0 && dev < 64) done[dev] = true;
    return true;
}

// Launches a kernel that may start while the one before it on the stream still runs (programmatic dependent launch); it
// has to wait (griddepcontrol.wait) before it touches anything that kernel, or one before it, reads or writes.
template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const char* what, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    if (err != cudaSuccess) {
        cudaGetLastError();  // clear the sticky launch error
        return fail(DSV4_ERR_LAUNCH, what);
    }
    return check_launch(what);
}
#endif

// ---- launchers implemented in rowwise_quant.cu -----------------------------------
int ptq(const void* x, void* q, void* s, int M, int K, int64_t ldx, cudaStream_t st);
int ptgq(const void* x, void* q, void* s, int M, int K, int gs, cudaStream_t st);
int add_rmsnorm_quant(void* res, const void* x, const void* w, void* q, void* s, int M, int K,
                      float eps, cudaStream_t st);
int rmsnorm(void* x, int M, int K, float eps, cudaStream_t st);
// masked_m / max_m: masked expert layout (rows are E blocks of max_m rows, the first masked_m[e] of block e valid)
int silu_mul_quant(const void* g, const void* u, const int* mask, const int* valid_rows, void* q, void* s,
                   int M, int N, int64_t ldg, int64_t ldu, cudaStream_t st, const int* masked_m = nullptr,
                   int max_m = 0);
int silu_mul(const void* g, const void* u, void* out, int M, int N, int64_t ldg, int64_t ldu,
             cudaStream_t st);

// ---- launchers implemented in gemm_i8_sm100.cu ------------------------------------
struct GemmArgs {
    const void* A;        // int8 [M or R, K]
    const void* B;        // int8 [N, K] or [E, N, K]
    const float* sa;      // [M] per token, or [M, K/128] when sa_groups > 1
    const float* sb;      // [N] or [E, N]; may be null only when out_i32
    void* C;              // bf16 [M, N] or int32 [M, N]
    const int* offsets;   // null for a dense GEMM, else expert_offsets[E+1]
    const int* masked_m = nullptr;  // masked layout instead of offsets: A, C are [E, max_m, .], masked_m[E] on the device
    int max_m = 0;
    int M, N, K, E;
    int64_t ldc;          // row stride of C in elements; 0 = N
    int sa_groups;        // 1 = per-token scale; K/128 = one scale per 128 of K
    int out_i32;          // 1 = write raw int32 accumulators
    void* const* row_ptr = nullptr;  // grouped GEMM, per-token scales: device array, one destination row per result row (C unused)
    void* peerC[7];       // fused all-gather: the other ranks' mapped output slabs
    int npeers;           // 0 = none
    // fused epilogue (enum Epilogue in gemm_i8_common.cuh): 1 linear, 2 gated (B is [2 N, K], gates first)
    int epilogue = 0;
    const void* bias = nullptr;    // bf16, one per row of B
    const void* resid = nullptr;   // bf16 [M, N] with row stride ldr
    int64_t ldr = 0;
    int act = 0;                   // enum Activation in activations.cuh
    void* row_sizes = nullptr;     // gradient epilogues (3 linear, 4 gated; resid is the incoming gradient, C is fp32): RowSize
    int* size_slots = nullptr;     // where to say how many slots each row of row_sizes has (two per 64 rows of B at most)
    int up_col = 0;                // gated gradient: first column of the ups in C
    // Test hook, zero through every public entry point: the tile producers of the launch issue no
    // loads and every bounded wait gives up after test_wait_limit_ns, so the kernel's give-up path runs.
    int test_withhold_loads = 0;
    unsigned long long test_wait_limit_ns = 0;
};
int gemm_i8(const GemmArgs& a, cudaStream_t st);
// Before the launches of an operator whose kernels wait on barriers: if one launched earlier on this device gave up such a
// wait, says so once (DSV4_ERR_DEVICE_WAIT).  The device's word has its mirror in host memory from the first call on.
int refuse_after_failed_wait();
struct GradientArgs {
    const void* digits;         // int8 [3][M][parts * part_pitch]: hi, mid, and lo for wide rows only
    const unsigned* row_size;   // [M] packed_size (gradient_digits.cuh)
    const unsigned char* wide;  // per block of 32 rows: whether it has a wide row; 8-byte aligned, zeros up to a multiple of eight
    const void* W;              // int8 [parts * part_rows, K]
    void* dx;                   // bf16 [M, K]
    int M, K, parts, part_rows, part_pitch;   // part_pitch: multiple of 128, zeros behind part_rows
    const float* partial;       // null, or [row_blocks][parts * part_rows]: column sums of blocks of rows
    int row_blocks;
    float* dbias;               // their sums
    int test_withhold_loads = 0;                   // as in GemmArgs
    unsigned long long test_wait_limit_ns = 0;
};
int gemm_i8_gradient(const GradientArgs& a, cudaStream_t st);
int scale_convert(const void* acc, const void* sa, const void* sb, void* out, int M, int N,
                  cudaStream_t st);

// ---- launchers implemented in moe_segments.cu -------------------------------------
int moe_segments(const int* topk_ids, int T, int topk, int E, int expert_lo, int* offsets, int* src_row,
                 int* dst_slot, cudaStream_t st);
int gather_rows(const void* src, const int* src_row, void* dst, int R, int row_bytes,
                const float* src_scale, float* dst_scale, int scales_per_row, const int* valid_rows,
                cudaStream_t st);
int moe_topk(const float* logits, int T, int E, int k, int* ids, float* weights, cudaStream_t st);
int moe_combine(const void* z, const int* dst_slot, const float* w, void* out, int T, int topk, int H,
                int out_f32, cudaStream_t st);
void set_overlap_previous_kernel(int on);
int overlap_previous_kernel();
int moe_combine_exchange(const void* const* z_ranks, const int* const* slot_ranks, const int* topk_ids,
                         const float* topk_w, void* const* out_ranks, int G, int experts_per_rank, int t0, int t1,
                         int topk, int H, cudaStream_t st);
int moe_push_rows(const int* dst_slot, int T, int topk, int tokens_per_rank, void* const* inbox_ranks, int G, int H,
                  void** row_ptr, cudaStream_t st);

// ---- launchers implemented in layernorm.cu ------------------------------------------
// res null: no residual; q null: bf16 output y
int layernorm(void* res, const void* x, const void* w, const void* b, void* y, void* q, void* s, void* mean, void* rstd,
              int M, int K, float eps, cudaStream_t st);
int64_t layernorm_backward_workspace(int M, int K);
int layernorm_backward(const void* dy, const void* x, const void* mean, const void* rstd, const void* w, const void* dres,
                       void* dx, void* dw, void* db, void* workspace, int M, int K, cudaStream_t st);

// ---- launchers implemented in w8a8_backward.cu ----------------------------------------
struct BackwardArgs {
    const void* dy;        // bf16 [M, N], or [M, N / 2] when gated; row stride ldy
    int64_t ldy;
    const void* A;         // int8 [M, K]: the forward's codes
    const void* B;         // int8 [N, K]
    const float* sa;
    const float* sb;
    const void* bias;      // bf16 [N] or null
    int act;
    bool gated;
    void* dx;              // bf16 [M, K]
    float* dbias;          // fp32 [N] or null
    int M, N, K;
    int test_withhold_loads = 0;                   // of the gradient product, as in GemmArgs
    unsigned long long test_wait_limit_ns = 0;
};
int64_t w8a8_backward_workspace(int M, int N, bool gated, bool recompute, bool dbias);
int w8a8_backward(const BackwardArgs& a, void* workspace, cudaStream_t st);

int read_device_status(cudaStream_t st, int* out);
int read_row_status(int* out);  // status word of the row kernels (after the stream was synchronised)

}  // namespace w8a8
