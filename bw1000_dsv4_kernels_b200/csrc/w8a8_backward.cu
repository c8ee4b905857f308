// Backward pass of the fused W8A8 linear and of the gated projection, through the frozen int8 weight:
//
//   dz    = dy * act'(z)   (gated: dg = dh * zu * act'(zg), du = dh * act(zg)), z computed again from the forward's codes
//   dx    = (dz * sb) W                      the gradient of the dequantised activations
//   dbias = sum over rows of dz              fp32
//
// Three steps: the forward's GEMM with a gradient epilogue writes dz in fp32 and, per row and tile, the largest |dz * sb|
// (gemm_i8_epilogues.cuh); split_gradient_kernel puts dz * sb into two int8 digits per element and sums the columns;
// gemm_i8_grad_kernel, or gemm_i8_grad_stream_kernel for few rows, multiplies the digits with W and adds the column sums up.
// The codes and scales of the forward are all that has to be kept for it.  Each kernel is launched to start while the one
// before it drains.  Without an activation dz is dy itself: the first step is a pass over dy for the rows' largest
// magnitudes.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "activations.cuh"
#include "gradient_digits.cuh"
#include "launch_common.h"
#include "sm100_ptx.cuh"
#include "w8a8_arith.cuh"

namespace w8a8 {
namespace {

__device__ __forceinline__ unsigned top_bits(unsigned top, float v) { return max(top, __float_as_uint(v) & 0x7fffffffu); }

// eight consecutive gradients of one row as fp32; those at or beyond `left` are zero.  What the kernel before wrote is read
// past L1: this kernel may have started before that one ended.
__device__ __forceinline__ void load8(const float* p, int left, bool vec, float (&v)[8]) {
    if (vec && left >= 8) {
        const float4 a = __ldcg(reinterpret_cast<const float4*>(p)), b = __ldcg(reinterpret_cast<const float4*>(p + 4));
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < left ? __ldcg(p + j) : 0.0f;
    }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int left, bool vec, float (&v)[8]) {
    if (vec && left >= 8) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        v[0] = bf16lo_to_f32(q.x); v[1] = bf16hi_to_f32(q.x); v[2] = bf16lo_to_f32(q.y); v[3] = bf16hi_to_f32(q.y);
        v[4] = bf16lo_to_f32(q.z); v[5] = bf16hi_to_f32(q.z); v[6] = bf16lo_to_f32(q.w); v[7] = bf16hi_to_f32(q.w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < left ? __bfloat162float(p[j]) : 0.0f;
    }
}

// row_top[row] = largest |dy * sb| of the row, as float bits: one CTA per row
__global__ void __launch_bounds__(256) row_top_kernel(const __nv_bfloat16* dy, int64_t ldy, const float* __restrict__ sb, int N,
                                                      bool vec, unsigned* row_top) {
    __shared__ unsigned part[8];
    ptx::grid_launch_dependents();
    const __nv_bfloat16* row = dy + (int64_t)blockIdx.x * ldy;
    unsigned top = 0;
    for (int c = threadIdx.x * 8; c < N; c += 256 * 8) {
        float v[8];
        load8(row + c, N - c, vec, v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < N) top = top_bits(top, v[j] * __ldg(sb + c + j));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < 8; ++w) top = max(top, part[w]);
        row_top[blockIdx.x] = top;
    }
}

// The columns of dz and of the digits: `parts` ranges (gates and ups, or one) of part_rows columns each, at multiples of
// part_pitch (a multiple of 128, so that a K block of the gradient product never straddles two ranges).
struct Columns {
    int parts, part_rows, part_pitch;
    __host__ __device__ int pitch() const { return parts * part_pitch; }
};

// tops[row][slots] -> each row's largest magnitude, by every warp that needs it; row_top, where it is wanted, gets it once.
// dz -> digits int8 [2][M][pitch] (hi, then lo; zeros behind each range), and with SUM the column sums of every block of
// kSplitRows rows.  A warp takes 256 columns of every eighth row of the block, all its rows' loads at once.
constexpr int kSplitRows = 32;
constexpr int kSplitWarps = 8;
template <typename T, bool SUM>
__global__ void __launch_bounds__(32 * kSplitWarps) split_gradient_kernel(const T* dz, int64_t ld, const float* __restrict__ sb,
                                                                          const unsigned* tops, int slots, unsigned* row_top, int M,
                                                                          Columns cols, bool vec, int8_t* digits,
                                                                          float* partial) {
    __shared__ float sums[SUM ? kSplitWarps : 1][SUM ? 264 : 1];
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();   // dz and the rows' tops come from the kernel before
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // one grid dimension for blocks of rows and of columns: there can be more than 65535 of the first
    const int pitch = cols.pitch(), col_blocks = (pitch + 255) / 256;
    const int row_block = blockIdx.x / col_blocks, col_block = blockIdx.x - row_block * col_blocks;
    const int c = col_block * 256 + lane * 8;              // column with padding
    const int part = c >= cols.part_pitch ? 1 : 0, local = c - part * cols.part_pitch;
    const int left = c < pitch ? cols.part_rows - local : 0, w_row = part * cols.part_rows + local;
    const int64_t plane = (int64_t)M * pitch;
    const int r0 = row_block * kSplitRows + warp;
    constexpr int kRows = kSplitRows / kSplitWarps;
    float v[kRows][8], inv[kRows], scale[8], sum[8] = {};
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = r0 + i * kSplitWarps;
        const bool ok = r < M;
        load8(dz + (int64_t)(ok ? r : 0) * ld + c, ok ? left : 0, vec, v[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) scale[j] = j < left ? __ldg(sb + w_row + j) : 0.0f;
    // the rows' largest magnitudes, all rows' loads at once
    unsigned top[kRows] = {};
#pragma unroll 1
    for (int s = lane; s < slots; s += 32) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = r0 + i * kSplitWarps;
            if (r < M) top[i] = max(top[i], __ldcg(tops + (int64_t)r * slots + s));
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = r0 + i * kSplitWarps;
        top[i] = __reduce_max_sync(0xffffffffu, top[i]);
        inv[i] = r < M ? digit_inverse(__uint_as_float(top[i])) : 0.0f;
        if (row_top != nullptr && col_block == 0 && lane == 0 && r < M) row_top[r] = top[i];
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = r0 + i * kSplitWarps;
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int d[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (SUM) sum[4 * h + j] += v[i][4 * h + j];
                d[j] = digits_of(v[i][4 * h + j] * scale[4 * h + j], inv[i]);
            }
            hi[h] = pack_i8x4(digit_hi(d[0]), digit_hi(d[1]), digit_hi(d[2]), digit_hi(d[3]));
            lo[h] = pack_i8x4(digit_lo(d[0]), digit_lo(d[1]), digit_lo(d[2]), digit_lo(d[3]));
        }
        if (r < M && c < pitch) {
            int8_t* out = digits + (int64_t)r * pitch + c;
            *reinterpret_cast<uint2*>(out) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(out + plane) = make_uint2(lo[0], lo[1]);
        }
    }
    if constexpr (SUM) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[warp][lane * 8 + j] = sum[j];
        __syncthreads();
        const int col = col_block * 256 + threadIdx.x, p2 = col >= cols.part_pitch ? 1 : 0, l2 = col - p2 * cols.part_pitch;
        if (col < pitch && l2 < cols.part_rows) {
            float t = 0.0f;
#pragma unroll
            for (int w = 0; w < kSplitWarps; ++w) t += sums[w][threadIdx.x];
            partial[(int64_t)row_block * cols.parts * cols.part_rows + p2 * cols.part_rows + l2] = t;
        }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Layout {
    Columns cols;
    int row_blocks;
    int64_t digits, dz, tops, row_top, partial, total;   // offsets and size in bytes
};
Layout layout(int M, int N, bool gated, bool recompute, bool dbias) {
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    Layout l;
    l.cols.parts = gated ? 2 : 1;
    l.cols.part_rows = N / l.cols.parts;
    l.cols.part_pitch = (l.cols.part_rows + 127) / 128 * 128;
    l.row_blocks = (M + kSplitRows - 1) / kSplitRows;
    const int64_t pitch = l.cols.pitch();
    l.digits = 0;
    l.dz = l.digits + up(2 * (int64_t)M * pitch);
    l.tops = l.dz + (recompute ? up(4 * (int64_t)M * pitch) : 0);
    // the narrowest tile has 64 rows of W and two slots
    l.row_top = l.tops + (recompute ? up(4 * (int64_t)M * 2 * ((N + 63) / 64)) : 0);
    l.partial = l.row_top + up(4 * (int64_t)M);
    l.total = l.partial + (dbias ? up(4 * (int64_t)l.row_blocks * N) : 0);
    return l;
}

template <typename T>
int split(const T* dz, int64_t ld, const BackwardArgs& a, const Layout& l, const unsigned* tops, int slots, unsigned* row_top,
          int8_t* digits, float* partial, cudaStream_t st) {
    const bool vec = (ld * sizeof(T)) % 16 == 0 && aligned16(dz);
    const int64_t blocks = (int64_t)((l.cols.pitch() + 255) / 256) * l.row_blocks;
    if (blocks > INT32_MAX) return fail(DSV4_ERR_ARG, "w8a8 backward: too many rows");
    auto kernel = a.dbias != nullptr ? split_gradient_kernel<T, true> : split_gradient_kernel<T, false>;
    return launch_after(kernel, dim3((unsigned)blocks), dim3(32 * kSplitWarps), 0, st, "w8a8 backward", dz, ld, a.sb, tops, slots,
                        row_top, a.M, l.cols, vec, digits, partial);
}

}  // namespace

int64_t w8a8_backward_workspace(int M, int N, bool gated, bool recompute, bool dbias) {
    return layout(M, N, gated, recompute, dbias).total;
}

int w8a8_backward(const BackwardArgs& a, void* workspace, cudaStream_t st) {
    const bool recompute = a.act != kActNone;
    const Layout l = layout(a.M, a.N, a.gated, recompute, a.dbias != nullptr);
    char* ws = static_cast<char*>(workspace);
    int8_t* digits = reinterpret_cast<int8_t*>(ws + l.digits);
    unsigned* row_top = reinterpret_cast<unsigned*>(ws + l.row_top);
    float* partial = reinterpret_cast<float*>(ws + l.partial);
    const __nv_bfloat16* dy = static_cast<const __nv_bfloat16*>(a.dy);
    if (recompute) {
        float* dz = reinterpret_cast<float*>(ws + l.dz);
        GemmArgs g{};
        g.A = a.A; g.B = a.B; g.sa = a.sa; g.sb = a.sb; g.C = dz;
        g.M = a.M; g.N = l.cols.part_rows; g.K = a.K; g.E = 1; g.ldc = l.cols.pitch(); g.sa_groups = 1;
        g.epilogue = a.gated ? 4 : 3; g.bias = a.bias; g.resid = a.dy; g.ldr = a.ldy; g.act = a.act;
        g.up_col = l.cols.part_pitch;
        unsigned* tops = reinterpret_cast<unsigned*>(ws + l.tops);
        int slots = 0;
        g.row_top = tops;
        g.top_slots = &slots;
        if (int rc = gemm_i8(g, st)) return rc;
        if (int rc = split(dz, (int64_t)l.cols.pitch(), a, l, tops, slots, row_top, digits, partial, st)) return rc;
    } else {
        row_top_kernel<<<a.M, 256, 0, st>>>(dy, a.ldy, a.sb, a.N, a.ldy % 8 == 0 && aligned16(dy), row_top);
        if (int rc = check_launch("w8a8 backward")) return rc;
        if (int rc = split(dy, a.ldy, a, l, row_top, 1, nullptr, digits, partial, st)) return rc;
    }
    GradientArgs d;
    d.digits = digits; d.row_top = row_top; d.W = a.B; d.dx = a.dx;
    d.M = a.M; d.K = a.K; d.parts = l.cols.parts; d.part_rows = l.cols.part_rows; d.part_pitch = l.cols.part_pitch;
    d.partial = a.dbias != nullptr ? partial : nullptr; d.row_blocks = l.row_blocks; d.dbias = a.dbias;
    return gemm_i8_gradient(d, st);
}

}  // namespace w8a8
