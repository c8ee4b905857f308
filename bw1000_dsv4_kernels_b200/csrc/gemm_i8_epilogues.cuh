// Private part of gemm_i8_sm100.cu: epilogues of the int8 GEMM kernels beyond the plain scaling.
//
//   linear       z = (acc * sa) * sb + bias;  y = act(z) + residual            -> bf16
//   gated        the tile holds a block of gate columns and the same block of up columns (two loads of weight rows, I
//                rows apart), so one thread has g and u of the same output: h = act(zg) * zu   -> bf16
//   gradients    z is computed again from the same codes and scales: dz = dy * act'(z), or dg = dh * zu * act'(zg) and
//                du = dh * act(zg), stored in fp32, together with each row's size (largest |dz * sb| and their sum: the
//                scale and the number of digits of the fixed-point form in which the gradient product takes it)
//
// Without bias, activation and residual, linear gives the bits of the plain epilogue.
#ifndef W8A8_GEMM_I8_EPILOGUES_CUH
#define W8A8_GEMM_I8_EPILOGUES_CUH

#include "activations.cuh"
#include "gemm_i8_common.cuh"

namespace w8a8 {
namespace {

// 32 consecutive bf16 of one row, packed in pairs; elements at or beyond `n_left` are zero
struct Row32 {
    uint32_t w[16];
};
// rows of `n` elements come in whole 16-byte pieces at 16-byte aligned addresses
__device__ __forceinline__ bool block_vector_ok(const void* base, int64_t ld, int n) {
    return ld % 8 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0 && n % 8 == 0;
}

// z of two columns.  A missing bias is -0, which leaves every product as it is: the bits of the plain epilogue.
constexpr float kNoBias = -0.0f;
__device__ __forceinline__ float2 scaled2(uint32_t acc0, uint32_t acc1, float sa, float2 sb, float2 bias) {
    const float2 f = make_float2(__int2float_rn((int)acc0), __int2float_rn((int)acc1));
    return __ffma2_rn(__fmul2_rn(f, splat2(sa)), sb, bias);
}

// A warp's block of 32 rows x 64 bytes (32 bf16 or 16 fp32), one row per lane in registers.  Stored from there directly, an
// instruction touches 32 rows, half a 32-byte sector in each; the block goes through the warp's shared memory instead,
// and every instruction moves 64 contiguous bytes of eight rows (16-byte aligned rows) or of one row (odd widths and
// addresses, an element per lane).  2048 x 36864 x 7168 with bias and residual: 459 us
// directly, 396 us this way (the plain GEMM, which stores directly, 405 to 423 us).
constexpr int kStagePitch = 20;                        // words per row: 16, and 4 that keep 16-byte accesses off each other's banks
constexpr int kBlockBytes = 32 * kStagePitch * 4;
struct RowBlock {
    int rows;     // valid rows of the block (lane r owns row r)
    int cols;     // valid columns; those beyond are not touched, and read as zero
    bool vec;     // rows are 16-byte aligned and `cols` comes in whole 16-byte pieces
};
__device__ __forceinline__ void stage_row(uint32_t* stage, int lane, const uint4 (&v)[4]) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(stage + lane * kStagePitch + 4 * j) = v[j];
    __syncwarp();
}
// 16-byte pieces: `pieces` (1..4) valid ones per row
__device__ __forceinline__ void store_pieces(char* block, int64_t ld_bytes, const uint4 (&v)[4], int rows, int pieces,
                                             uint32_t* stage, int lane) {
    stage_row(stage, lane, v);
    const int piece = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 8 * i + (lane >> 2);
        if (row < rows && piece < pieces)
            *reinterpret_cast<uint4*>(block + row * ld_bytes + 16 * piece) =
                *reinterpret_cast<const uint4*>(stage + row * kStagePitch + 4 * piece);
    }
}
// Loading takes two steps, so that the requests can be out long before the block is needed: fetch_block issues them into
// registers as the memory is laid out, arrange_block turns those into one row per lane.  Rows that are not 16-byte
// aligned come as the 16-byte granules that cover them, at most five for 64 bytes, and each lane shifts its row into place;
// element by element, 2048 x 7167 x 1024 with bias, GELU and residual took 113 us instead of 61 (50 at 7168).  Only the
// first and the last granule of the array can reach out of it; what they hold of it is fetched by elements.
struct Fetched {
    uint32_t w[20];
    int skew;     // bytes from the first granule to this lane's row
};
// `array` has m rows of n elements, `block` begins at one of them
__device__ __forceinline__ Fetched fetch_block(const __nv_bfloat16* array, int64_t ld, int m, int n, const __nv_bfloat16* block,
                                               const RowBlock& b, int lane) {
    Fetched f = {};
    if (b.vec) {
        const int piece = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 8 * i + (lane >> 2);
            if (row < b.rows && 8 * piece < b.cols) {
                const uint4 q = *reinterpret_cast<const uint4*>(block + row * ld + 8 * piece);
                f.w[4 * i] = q.x; f.w[4 * i + 1] = q.y; f.w[4 * i + 2] = q.z; f.w[4 * i + 3] = q.w;
            }
        }
        return f;
    }
    const char *lo = reinterpret_cast<const char*>(array), *hi = reinterpret_cast<const char*>(array + (m - 1) * ld + n);
    const int bytes = 2 * min(b.cols, 32);
    f.skew = (int)(reinterpret_cast<uintptr_t>(block + lane * ld) & 15);
    // granule i of this lane, or null where no row needs it
    auto granule = [&](int i) -> const char* {
        const int g = 32 * i + lane, row = g / 5, piece = g - 5 * row;
        const char* src = reinterpret_cast<const char*>(block + row * ld);
        const int skew = (int)(reinterpret_cast<uintptr_t>(src) & 15);
        return row < b.rows && 16 * piece < skew + bytes ? src + 16 * piece - skew : nullptr;
    };
    unsigned edges = 0;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        const char* src = granule(i);
        if (src == nullptr) continue;
        if (src >= lo && src + 16 <= hi) {
            const uint4 q = *reinterpret_cast<const uint4*>(src);
            f.w[4 * i] = q.x; f.w[4 * i + 1] = q.y; f.w[4 * i + 2] = q.z; f.w[4 * i + 3] = q.w;
        } else {
            edges |= 1u << i;
        }
    }
#pragma unroll 1
    for (int k = 0; edges >> k; ++k) {   // one of a lane's granules, but for arrays a few elements wide
        if (!((edges >> k) & 1)) continue;
        const char* src = granule(k);
        uint32_t e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const char* at = src + 4 * j;
            const uint32_t l = at >= lo && at < hi ? *reinterpret_cast<const uint16_t*>(at) : 0u;
            const uint32_t h = at + 2 >= lo && at + 2 < hi ? *reinterpret_cast<const uint16_t*>(at + 2) : 0u;
            e[j] = l | (h << 16);
        }
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            if (i == k) {
#pragma unroll
                for (int j = 0; j < 4; ++j) f.w[4 * i + j] = e[j];
            }
        }
    }
    return f;
}
__device__ __forceinline__ Row32 arrange_block(const Fetched& f, const RowBlock& b, uint32_t* stage, int lane) {
    __syncwarp();
    if (b.vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(stage + (8 * i + (lane >> 2)) * kStagePitch + 4 * (lane & 3)) =
                make_uint4(f.w[4 * i], f.w[4 * i + 1], f.w[4 * i + 2], f.w[4 * i + 3]);
    } else {
        static_assert(kStagePitch == 20, "five granules are a staged row");
#pragma unroll
        for (int i = 0; i < 5; ++i)
            *reinterpret_cast<uint4*>(stage + (32 * i + lane) * 4) =
                make_uint4(f.w[4 * i], f.w[4 * i + 1], f.w[4 * i + 2], f.w[4 * i + 3]);
    }
    __syncwarp();
    Row32 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint4 q = *reinterpret_cast<const uint4*>(stage + lane * kStagePitch + 4 * j);
        r.w[4 * j] = q.x; r.w[4 * j + 1] = q.y; r.w[4 * j + 2] = q.z; r.w[4 * j + 3] = q.w;
    }
    if (!b.vec) {
        // 80 bytes of the lane's row, shifted by `skew`: four-word, then two-byte steps
        const uint4 q = *reinterpret_cast<const uint4*>(stage + lane * kStagePitch + 16);
        uint32_t w[20];
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = r.w[j];
        w[16] = q.x; w[17] = q.y; w[18] = q.z; w[19] = q.w;
        const bool by2 = f.skew & 8, by1 = f.skew & 4;
#pragma unroll
        for (int j = 0; j < 18; ++j) w[j] = by2 ? w[j + 2] : w[j];
#pragma unroll
        for (int j = 0; j < 17; ++j) w[j] = by1 ? w[j + 1] : w[j];
        const uint32_t half = (f.skew & 2) * 8;
#pragma unroll
        for (int j = 0; j < 16; ++j) r.w[j] = __funnelshift_r(w[j], w[j + 1], half);
        if (b.cols < 32) {   // what follows the row is not zero
#pragma unroll
            for (int j = 0; j < 16; ++j) r.w[j] &= 2 * j + 1 < b.cols ? 0xffffffffu : 2 * j < b.cols ? 0xffffu : 0u;
        }
    }
    return r;
}
__device__ __forceinline__ void store_block(__nv_bfloat16* block, int64_t ld, const Row32& r, const RowBlock& b, uint32_t* stage,
                                            int lane) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = make_uint4(r.w[4 * j], r.w[4 * j + 1], r.w[4 * j + 2], r.w[4 * j + 3]);
    if (b.vec) {
        store_pieces(reinterpret_cast<char*>(block), 2 * ld, v, b.rows, (b.cols + 7) >> 3, stage, lane);
        return;
    }
    stage_row(stage, lane, v);
    const uint16_t* s16 = reinterpret_cast<const uint16_t*>(stage);
    uint16_t* dst = reinterpret_cast<uint16_t*>(block) + lane;
    if (lane < b.cols) {
#pragma unroll 8
        for (int i = 0; i < 32; ++i)
            if (i < b.rows) dst[i * ld] = s16[i * (2 * kStagePitch) + lane];
    }
}

// 32 columns of scales or biases in this warp's shared memory (16-byte aligned), four at a time: the tensor cores take
// nearly all of the shared memory's bandwidth for their operands, and one access per column and row made the GEMM 12 %
// slower than its plain form.
struct Cols32 {
    const float* p;
    __device__ __forceinline__ float4 four(int j) const { return *reinterpret_cast<const float4*>(p + 4 * j); }
};
__device__ __forceinline__ float2 two(const float4& v, int k) { return k == 0 ? make_float2(v.x, v.y) : make_float2(v.z, v.w); }

// y of 32 columns from the accumulators of one row
template <int ACT>
__device__ __forceinline__ Row32 linear_values(const uint32_t (&r)[32], float sa, Cols32 sb, Cols32 bias, bool has_res,
                                               const Row32& res) {
    Row32 out;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 s4 = sb.four(j), b4 = bias.four(j);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int e = 4 * j + 2 * k;
            float2 y = act_value2<ACT>(scaled2(r[e], r[e + 1], sa, two(s4, k), two(b4, k)));
            if (has_res) {
                const float2 add = bf16x2_to_f32x2(res.w[e >> 1]);
                y = make_float2(__fadd_rn(y.x, add.x), __fadd_rn(y.y, add.y));
            }
            out.w[e >> 1] = pack_bf16x2_rn(y.x, y.y);
        }
    }
    return out;
}

// h of 32 outputs from the accumulators of their gates and ups
template <int ACT>
__device__ __forceinline__ Row32 gated_values(const uint32_t (&g)[32], const uint32_t (&u)[32], float sa, Cols32 sg, Cols32 bg,
                                              Cols32 su, Cols32 bu) {
    Row32 out;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 sg4 = sg.four(j), bg4 = bg.four(j), su4 = su.four(j), bu4 = bu.four(j);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int e = 4 * j + 2 * k;
            const float2 h = __fmul2_rn(act_value2<ACT>(scaled2(g[e], g[e + 1], sa, two(sg4, k), two(bg4, k))),
                                        scaled2(u[e], u[e + 1], sa, two(su4, k), two(bu4, k)));
            out.w[e >> 1] = pack_bf16x2_rn(h.x, h.y);
        }
    }
    return out;
}

__device__ __forceinline__ uint4 bits4(const float2& a, const float2& b) {
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
}

// dz of 32 columns -> the warp's block of dz (fp32, rows 16-byte aligned with room for whole chunks); dz * sb is added to the
// row's size
template <int ACT>
__device__ __forceinline__ void linear_gradients(const uint32_t (&r)[32], float sa, Cols32 sb, Cols32 bias, const Row32& dy,
                                                     float* block, int64_t ld, int rows, uint32_t* stage, int lane, RowSize& size) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint4 out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = 4 * half + i;
            const float4 s4 = sb.four(j), b4 = bias.four(j);
            float2 v[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int e = 4 * j + 2 * k;
                float2 slope;
                act_value_slope2<ACT>(scaled2(r[e], r[e + 1], sa, two(s4, k), two(b4, k)), slope);
                v[k] = __fmul2_rn(bf16x2_to_f32x2(dy.w[e >> 1]), slope);
                size.add(__fmul2_rn(v[k], two(s4, k)));
            }
            out[i] = bits4(v[0], v[1]);
        }
        store_pieces(reinterpret_cast<char*>(block + 16 * half), 4 * ld, out, rows, 4, stage, lane);
    }
}

// dg and du of 32 outputs
template <int ACT>
__device__ __forceinline__ void gated_gradients(const uint32_t (&g)[32], const uint32_t (&u)[32], float sa, Cols32 sg,
                                                    Cols32 bg, Cols32 su, Cols32 bu, const Row32& dh, float* block_g,
                                                    float* block_u, int64_t ld, int rows, uint32_t* stage, int lane, RowSize& size) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint4 out_g[4], out_u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = 4 * half + i;
            const float4 sg4 = sg.four(j), bg4 = bg.four(j), su4 = su.four(j), bu4 = bu.four(j);
            float2 vg[2], vu[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int e = 4 * j + 2 * k;
                float2 slope;
                const float2 value = act_value_slope2<ACT>(scaled2(g[e], g[e + 1], sa, two(sg4, k), two(bg4, k)), slope);
                const float2 d = bf16x2_to_f32x2(dh.w[e >> 1]);
                vg[k] = __fmul2_rn(__fmul2_rn(d, scaled2(u[e], u[e + 1], sa, two(su4, k), two(bu4, k))), slope);
                vu[k] = __fmul2_rn(d, value);
                size.add(__fmul2_rn(vg[k], two(sg4, k)));
                size.add(__fmul2_rn(vu[k], two(su4, k)));
            }
            out_g[i] = bits4(vg[0], vg[1]);
            out_u[i] = bits4(vu[0], vu[1]);
        }
        store_pieces(reinterpret_cast<char*>(block_g + 16 * half), 4 * ld, out_g, rows, 4, stage, lane);
        store_pieces(reinterpret_cast<char*>(block_u + 16 * half), 4 * ld, out_u, rows, 4, stage, lane);
    }
}

// Split-K epilogues of the weight-streaming kernels (see reduce_partials_and_store): the item's partials come through
// distributed shared memory, its residual from HBM at the same time.
__device__ __forceinline__ void store4(const Params& p, int row, int n, const float2& a, const float2& b, bool vec) {
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.C) + (int64_t)row * p.ldc + n;
    const uint32_t lo = pack_bf16x2_rn(a.x, a.y), hi = pack_bf16x2_rn(b.x, b.y);
    if (vec && n + 4 <= p.N) {
        *reinterpret_cast<uint2*>(out) = make_uint2(lo, hi);
    } else {
        const uint16_t h4[4] = {(uint16_t)(lo & 0xffffu), (uint16_t)(lo >> 16), (uint16_t)(hi & 0xffffu), (uint16_t)(hi >> 16)};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < p.N) reinterpret_cast<uint16_t*>(out)[j] = h4[j];
    }
}

// Gated: rows [0, 64) of the weight tile are gates, [64, 128) the ups of the same outputs; 16 groups of four outputs
// per token instead of 32.  Tokens count from m0, the first of the CTA's block of tokens.
template <int MAXS, int U, int EPI>
__device__ __forceinline__ void reduce_partials_fused(const Params& p, const uint32_t (&peer_base)[MAXS], int S, int m0, int cols_lo,
                                                      int cols_hi, int n0, int tid, int nthreads, const float* sa_s,
                                                      const float* sb_s, const float* bias_s) {
    constexpr bool kGated = is_gated(EPI), kGrad = EPI == kEpiLinearGrad || EPI == kEpiGatedGrad;
    constexpr bool kReads = EPI != kEpiGated;   // a residual, or the incoming gradient
    constexpr int kGroups = kGated ? 16 : 32, kShift = kGated ? 4 : 5, kHalves = kGated ? 2 : 1;
    const bool vec_store = (p.ldc % 4 == 0) && ((reinterpret_cast<uintptr_t>(p.C) & 7) == 0);
    const bool res_vec = (p.ldr % 4 == 0) && ((reinterpret_cast<uintptr_t>(p.resid) & 7) == 0);
    const int items = (cols_hi - cols_lo) * kGroups;
    // a warp's lanes stay together: the gradients' sizes are exchanged between them
    for (int it0 = tid; (it0 & ~31) < items; it0 += nthreads * U) {
        uint4 v[U][kHalves][MAXS];
        uint2 res[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = it0 + u * nthreads;
            res[u] = make_uint2(0u, 0u);
            if (it < items) {
                const int c = cols_lo + (it >> kShift), g = it & (kGroups - 1);
                if (kReads && p.resid != nullptr) {
                    const int n = n0 + g * 4;
                    const __nv_bfloat16* rp = p.resid + (int64_t)(m0 + c) * p.ldr + n;
                    if (res_vec && n + 4 <= p.N) {
                        res[u] = *reinterpret_cast<const uint2*>(rp);
                    } else {
                        uint32_t e[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) e[j] = n + j < p.N ? reinterpret_cast<const uint16_t*>(rp)[j] : 0u;
                        res[u] = make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
                    }
                }
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    const uint32_t off = (uint32_t)(c * 128 + h * 64 + g * 4) * 4u;
#pragma unroll
                    for (int r = 0; r < MAXS; ++r)
                        if (r < S) v[u][h][r] = ptx::ld_shared_cluster_v4(peer_base[r] + off);
                }
            }
        }
        float2 z[U][kHalves][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = it0 + u * nthreads;
            const bool ok = it < items;
            const int c = ok ? cols_lo + (it >> kShift) : 0, g = it & (kGroups - 1);
            const float sa = sa_s[c];
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                int a[4] = {0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < MAXS; ++r) {
                    if (ok && r < S) {
                        a[0] += (int)v[u][h][r].x; a[1] += (int)v[u][h][r].y; a[2] += (int)v[u][h][r].z; a[3] += (int)v[u][h][r].w;
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int col = h * 64 + g * 4 + 2 * j;
                    z[u][h][j] = scaled2((uint32_t)a[2 * j], (uint32_t)a[2 * j + 1], sa, make_float2(sb_s[col], sb_s[col + 1]),
                                         make_float2(bias_s[col], bias_s[col + 1]));
                }
            }
        }
        // one choice of the activation for all items: a tile's epilogue runs once, so its instructions are fetched cold
        with_act(p.act, [&](auto act) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (kGrad) {
                        const float2 d = bf16x2_to_f32x2(j == 0 ? res[u].x : res[u].y);
                        float2 slope;
                        const float2 value = act_value_slope2<decltype(act)::value>(z[u][0][j], slope);
                        if constexpr (kGated) {
                            z[u][0][j] = __fmul2_rn(__fmul2_rn(d, z[u][kHalves - 1][j]), slope);
                            z[u][kHalves - 1][j] = __fmul2_rn(d, value);
                        } else {
                            z[u][0][j] = __fmul2_rn(d, slope);
                        }
                    } else {
                        z[u][0][j] = act_value2<decltype(act)::value>(z[u][0][j]);
                        if constexpr (kGated) z[u][0][j] = __fmul2_rn(z[u][0][j], z[u][kHalves - 1][j]);
                    }
                }
            }
        });
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = it0 + u * nthreads;
            const int c = cols_lo + (it >> kShift), g = it & (kGroups - 1), n = n0 + g * 4;
            const bool ok = it < items && n < p.N;
            if constexpr (kGrad) {
                // dz rows have room for whole tiles: four columns are stored, those at or beyond N with zeros
                RowSize size = RowSize::none();
                if (ok) {
                    float* dz = static_cast<float*>(p.C) + (int64_t)(m0 + c) * p.ldc + n;
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) {
                        *reinterpret_cast<uint4*>(dz + h * p.up_col) = bits4(z[u][h][0], z[u][h][1]);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int col = h * 64 + g * 4 + 2 * j;
                            size.add(__fmul2_rn(z[u][h][j], make_float2(sb_s[col], sb_s[col + 1])));
                        }
                    }
                }
#pragma unroll
                for (int o = kGroups >> 1; o > 0; o >>= 1) size.add_lane(o);
                if (g == 0 && it < items && n0 < p.N)
                    p.row_sizes[(int64_t)(m0 + c) * p.size_slots + n0 / (kGated ? 64 : 128)] = size;
            } else if (ok) {
                if (kReads && p.resid != nullptr) {
                    const float2 r0 = bf16x2_to_f32x2(res[u].x), r1 = bf16x2_to_f32x2(res[u].y);
                    z[u][0][0] = make_float2(__fadd_rn(z[u][0][0].x, r0.x), __fadd_rn(z[u][0][0].y, r0.y));
                    z[u][0][1] = make_float2(__fadd_rn(z[u][0][1].x, r1.x), __fadd_rn(z[u][0][1].y, r1.y));
                }
                store4(p, m0 + c, n, z[u][0][0], z[u][0][1], vec_store);
            }
        }
    }
}

// With no more items than threads (few tokens) one item per thread: the loop body for U of them would be fetched, cold, to
// do nothing, which cost 1.4 us of a 9 us kernel.
template <int MAXS, int U, int EPI>
__device__ __forceinline__ void reduce_partials_fused_sized(const Params& p, const uint32_t (&peer_base)[MAXS], int S, int m0,
                                                            int cols_lo, int cols_hi, int n0, int tid, int nthreads,
                                                            const float* scales) {
    if ((cols_hi - cols_lo) * (is_gated(EPI) ? 16 : 32) <= nthreads)
        reduce_partials_fused<MAXS, 1, EPI>(p, peer_base, S, m0, cols_lo, cols_hi, n0, tid, nthreads, scales, scales + 256, scales + 384);
    else
        reduce_partials_fused<MAXS, U, EPI>(p, peer_base, S, m0, cols_lo, cols_hi, n0, tid, nthreads, scales, scales + 256, scales + 384);
}

}  // namespace
}  // namespace w8a8

#endif  // W8A8_GEMM_I8_EPILOGUES_CUH
