// Backward pass of the fused W8A8 linear and of the gated projection, through the frozen int8 weight:
//
//   dz    = dy * act'(z)   (gated: dg = dh * zu * act'(zg), du = dh * act(zg)), z computed again from the forward's codes
//   dx    = (dz * sb) W                      the gradient of the dequantised activations
//   dbias = sum over rows of dz              fp32
//
// Three steps: the forward's GEMM with a gradient epilogue writes dz in fp32 and, per row and tile, the size of dz * sb
// (gemm_i8_epilogues.cuh); split_gradient_kernel puts dz * sb into two int8 digits per element, three in rows that need them
// (gradient_digits.cuh), and sums the columns; gemm_i8_grad_kernel, or gemm_i8_grad_stream_kernel for few rows, multiplies
// the digits with W and adds the column sums up.  The codes and scales of the forward are all that has to be kept for it.
// Each kernel is launched to start while the one before it drains.  Without an activation dz is dy itself: the first step
// is a pass over dy for the rows' sizes.
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

// sizes[row] = size of the row's dy * sb: one CTA per row
__global__ void __launch_bounds__(256) row_size_kernel(const __nv_bfloat16* dy, int64_t ldy, const float* __restrict__ sb, int N,
                                                       bool vec, RowSize* sizes) {
    __shared__ RowSize part[8];
    ptx::grid_launch_dependents();
    const __nv_bfloat16* row = dy + (int64_t)blockIdx.x * ldy;
    RowSize size = RowSize::none();
    for (int c = threadIdx.x * 8; c < N; c += 256 * 8) {
        float v[8];
        load8(row + c, N - c, vec, v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < N) size.add(v[j] * __ldg(sb + c + j));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) size.add_lane(o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = size;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < 8; ++w) size.add(part[w]);
        sizes[blockIdx.x] = size;
    }
}

// The columns of dz and of the digits: `parts` ranges (gates and ups, or one) of part_rows columns each, at multiples of
// part_pitch (a multiple of 128, so that a K block of the gradient product never straddles two ranges).
struct Columns {
    int parts, part_rows, part_pitch;
    __host__ __device__ int pitch() const { return parts * part_pitch; }
};

// sizes[row][slots] -> each row's size, by every warp that needs it (the same bits in each: one order of the sum); row_size
// gets it once, and wide[block of kSplitRows rows] whether one of them is wide (zeros behind the last, up to a multiple of
// eight).
// dz -> digits int8 [3][M][pitch] (hi, mid, lo; zeros behind each range; lo only in wide rows), and with SUM the column sums of
// every block of rows.  A warp takes 256 columns of every eighth row of the block, all its rows' loads at once.
constexpr int kSplitRows = 32;
constexpr int kSplitWarps = 8;
template <typename T, bool SUM>
__global__ void __launch_bounds__(32 * kSplitWarps, 4) split_gradient_kernel(const T* dz, int64_t ld, const float* __restrict__ sb,
                                                                          const RowSize* sizes, int slots, unsigned* row_size,
                                                                          uint8_t* wide, float share, int M, Columns cols, bool vec,
                                                                          int8_t* digits, float* partial) {
    __shared__ float sums[SUM ? kSplitWarps : 1][SUM ? 264 : 1];
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();   // dz and the rows' sizes come from the kernel before
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
    float v[kRows][8], scale[8], sum[8] = {};
    // the rows' sizes, all rows' loads at once, in front of dz (behind it: 2 us more, 6.9 against 5.2 us at 128 x 4096 and 14.2
    // against 12.1 at 2048 x 4096)
    RowSize size[kRows];
    bool three[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) size[i] = RowSize::none();
#pragma unroll 1
    for (int s = lane; s < slots; s += 32) {
        uint2 got[kRows];   // rows behind the last read the last one's
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            got[i] = __ldcg(reinterpret_cast<const uint2*>(sizes + (int64_t)min(r0 + i * kSplitWarps, M - 1) * slots + s));
#pragma unroll
        for (int i = 0; i < kRows; ++i) size[i].add(RowSize{got[i].x, __uint_as_float(got[i].y)});
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = r0 + i * kSplitWarps;
        const bool ok = r < M;
        load8(dz + (int64_t)(ok ? r : 0) * ld + c, ok ? left : 0, vec, v[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) scale[j] = j < left ? __ldg(sb + w_row + j) : 0.0f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = r0 + i * kSplitWarps;
        size[i].top = __reduce_max_sync(0xffffffffu, size[i].top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) size[i].roots = __fadd_rn(size[i].roots, __shfl_xor_sync(0xffffffffu, size[i].roots, o));
        three[i] = r < M && size[i].wide(share);
        if (col_block == 0 && lane == 0 && r < M) row_size[r] = packed_size(size[i].top, three[i]);
    }
    if (col_block == 0) {   // the whole CTA
        bool any = false;
#pragma unroll
        for (int i = 0; i < kRows; ++i) any |= three[i];
        const int some = __syncthreads_or(any);
        if (threadIdx.x == 0) {
            wide[row_block] = some != 0;
            if ((row_block + 1) * kSplitRows >= M)
                for (int i = row_block + 1; i & 7; ++i) wide[i] = 0;
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = r0 + i * kSplitWarps;
        const RowDigits row = RowDigits::make(size[i].top, three[i]);
        uint32_t hi[2], mid[2], lo[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            unsigned d[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (SUM) sum[4 * h + j] += v[i][4 * h + j];
                d[j] = row.of(v[i][4 * h + j] * scale[4 * h + j]);
            }
            hi[h] = pack_digit<2>(d);
            mid[h] = pack_digit<1>(d);
            lo[h] = pack_digit<0>(d);
        }
        if (r < M && c < pitch) {
            int8_t* out = digits + (int64_t)r * pitch + c;
            *reinterpret_cast<uint2*>(out) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(out + plane) = make_uint2(mid[0], mid[1]);
            if (three[i]) *reinterpret_cast<uint2*>(out + 2 * plane) = make_uint2(lo[0], lo[1]);
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
    int64_t digits, dz, sizes, row_size, wide, partial, total;   // offsets and size in bytes
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
    l.dz = l.digits + up(3 * (int64_t)M * pitch);
    l.sizes = l.dz + (recompute ? up(4 * (int64_t)M * pitch) : 0);
    // the narrowest tile has 64 rows of W and two slots
    l.row_size = l.sizes + up((int64_t)sizeof(RowSize) * M * (recompute ? 2 * ((N + 63) / 64) : 1));
    l.wide = l.row_size + up(4 * (int64_t)M);
    l.partial = l.wide + up(l.row_blocks);
    l.total = l.partial + (dbias ? up(4 * (int64_t)l.row_blocks * N) : 0);
    return l;
}

template <typename T>
int split(const T* dz, int64_t ld, const BackwardArgs& a, const Layout& l, const RowSize* sizes, int slots, unsigned* row_size,
          uint8_t* wide, int8_t* digits, float* partial, cudaStream_t st) {
    const bool vec = (ld * sizeof(T)) % 16 == 0 && aligned16(dz);
    const int64_t blocks = (int64_t)((l.cols.pitch() + 255) / 256) * l.row_blocks;
    if (blocks > INT32_MAX) return fail(DSV4_ERR_ARG, "w8a8 backward: too many rows");
    auto kernel = a.dbias != nullptr ? split_gradient_kernel<T, true> : split_gradient_kernel<T, false>;
    return launch_after(kernel, dim3((unsigned)blocks), dim3(32 * kSplitWarps), 0, st, "w8a8 backward", dz, ld, a.sb, sizes, slots,
                        row_size, wide, kWideRoot / (float)a.N, a.M, l.cols, vec, digits, partial);
}

}  // namespace

int64_t w8a8_backward_workspace(int M, int N, bool gated, bool recompute, bool dbias) {
    return layout(M, N, gated, recompute, dbias).total;
}

int w8a8_backward(const BackwardArgs& a, void* workspace, cudaStream_t st) {
    if (int rc = refuse_after_failed_wait()) return rc;
    const bool recompute = a.act != kActNone;
    const Layout l = layout(a.M, a.N, a.gated, recompute, a.dbias != nullptr);
    char* ws = static_cast<char*>(workspace);
    int8_t* digits = reinterpret_cast<int8_t*>(ws + l.digits);
    RowSize* sizes = reinterpret_cast<RowSize*>(ws + l.sizes);
    unsigned* row_size = reinterpret_cast<unsigned*>(ws + l.row_size);
    uint8_t* wide = reinterpret_cast<uint8_t*>(ws + l.wide);
    float* partial = reinterpret_cast<float*>(ws + l.partial);
    const __nv_bfloat16* dy = static_cast<const __nv_bfloat16*>(a.dy);
    if (recompute) {
        float* dz = reinterpret_cast<float*>(ws + l.dz);
        GemmArgs g{};
        g.A = a.A; g.B = a.B; g.sa = a.sa; g.sb = a.sb; g.C = dz;
        g.M = a.M; g.N = l.cols.part_rows; g.K = a.K; g.E = 1; g.ldc = l.cols.pitch(); g.sa_groups = 1;
        g.epilogue = a.gated ? 4 : 3; g.bias = a.bias; g.resid = a.dy; g.ldr = a.ldy; g.act = a.act;
        g.up_col = l.cols.part_pitch;
        int slots = 0;
        g.row_sizes = sizes;
        g.size_slots = &slots;
        if (int rc = gemm_i8(g, st)) return rc;
        if (int rc = split(dz, (int64_t)l.cols.pitch(), a, l, sizes, slots, row_size, wide, digits, partial, st)) return rc;
    } else {
        row_size_kernel<<<a.M, 256, 0, st>>>(dy, a.ldy, a.sb, a.N, a.ldy % 8 == 0 && aligned16(dy), sizes);
        if (int rc = check_launch("w8a8 backward")) return rc;
        if (int rc = split(dy, a.ldy, a, l, sizes, 1, row_size, wide, digits, partial, st)) return rc;
    }
    GradientArgs d;
    d.digits = digits; d.row_size = row_size; d.wide = wide; d.W = a.B; d.dx = a.dx;
    d.M = a.M; d.K = a.K; d.parts = l.cols.parts; d.part_rows = l.cols.part_rows; d.part_pitch = l.cols.part_pitch;
    d.partial = a.dbias != nullptr ? partial : nullptr; d.row_blocks = l.row_blocks; d.dbias = a.dbias;
    d.test_withhold_loads = a.test_withhold_loads; d.test_wait_limit_ns = a.test_wait_limit_ns;
    return gemm_i8_gradient(d, st);
}

}  // namespace w8a8
