// Private part of gemm_i8_sm100.cu: epilogues of the int8 GEMM kernels beyond the plain scaling.
//
//   linear       z = (acc * sa) * sb + bias;  y = act(z) + residual            -> bf16
//   gated        the tile holds a block of gate columns and the same block of up columns (two loads of weight rows, I
//                rows apart), so one thread has g and u of the same output: h = act(zg) * zu   -> bf16
//   gradients    z is computed again from the same codes and scales: dz = dy * act'(z), or dg = dh * zu * act'(zg) and
//                du = dh * act(zg), stored in fp32, together with each row's largest |dz * sb| (the scale of the
//                fixed-point form in which the gradient product takes it)
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
__device__ __forceinline__ void load_row32(Row32& r, const __nv_bfloat16* p, int n_left, bool vec) {
    if (vec && n_left >= 32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint4 q = *reinterpret_cast<const uint4*>(p + 8 * j);
            r.w[4 * j] = q.x; r.w[4 * j + 1] = q.y; r.w[4 * j + 2] = q.z; r.w[4 * j + 3] = q.w;
        }
    } else {
        const uint16_t* s = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint32_t lo = 2 * j < n_left ? s[2 * j] : 0u, hi = 2 * j + 1 < n_left ? s[2 * j + 1] : 0u;
            r.w[j] = lo | (hi << 16);
        }
    }
}
__device__ __forceinline__ float row32_at(const Row32& r, int j) {
    return (j & 1) ? bf16hi_to_f32(r.w[j >> 1]) : bf16lo_to_f32(r.w[j >> 1]);
}
__device__ __forceinline__ void store_row32(__nv_bfloat16* p, const Row32& r, int n_left, bool vec) {
    if (vec && n_left >= 32) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4*>(p + 8 * j) = make_uint4(r.w[4 * j], r.w[4 * j + 1], r.w[4 * j + 2], r.w[4 * j + 3]);
    } else {
        uint16_t* s = reinterpret_cast<uint16_t*>(p);
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < n_left) s[j] = (uint16_t)((j & 1) ? r.w[j >> 1] >> 16 : r.w[j >> 1] & 0xffffu);
    }
}

__device__ __forceinline__ bool row_vector_ok(const void* base, int64_t ld) {
    return (ld % 8 == 0) && ((reinterpret_cast<uintptr_t>(base) & 15) == 0);
}

__device__ __forceinline__ float scaled(uint32_t acc, float sa, float sb, float bias) {
    return __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn((int)acc), sa), sb), bias);
}

// A warp's 32 x 32 block of a bf16 array, one row per lane.  Rows that are 16-byte aligned move as four 16-byte accesses
// per lane.  Otherwise (odd widths, odd addresses) an access per element and lane would touch 32 lines each, 32 times;
// the block goes through the warp's shared memory instead, where lane = column makes each row one access.
constexpr int kStagePitch = 17;                        // words per row: 16 plus one against bank conflicts
constexpr int kBlockBytes = 32 * kStagePitch * 4;
struct RowBlock {
    int rows;     // valid rows of the block (lane r owns row r)
    int cols;     // valid columns
    bool vec;     // rows are 16-byte aligned
};
__device__ __forceinline__ Row32 load_block(const __nv_bfloat16* block, int64_t ld, const RowBlock& b, uint32_t* stage, int lane) {
    Row32 r = {};
    if (b.vec && b.cols >= 32) {
        if (lane < b.rows) load_row32(r, block + lane * ld, 32, true);
        return r;
    }
    __syncwarp();
    uint16_t* s16 = reinterpret_cast<uint16_t*>(stage);
    const uint16_t* src = reinterpret_cast<const uint16_t*>(block) + lane;
#pragma unroll 8
    for (int i = 0; i < 32; ++i)
        s16[i * (2 * kStagePitch) + lane] = i < b.rows && lane < b.cols ? src[i * ld] : (uint16_t)0;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) r.w[j] = stage[lane * kStagePitch + j];
    return r;
}
__device__ __forceinline__ void store_block(__nv_bfloat16* block, int64_t ld, const Row32& r, const RowBlock& b, uint32_t* stage,
                                            int lane) {
    if (b.vec && b.cols >= 32) {
        if (lane < b.rows) store_row32(block + lane * ld, r, 32, true);
        return;
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) stage[lane * kStagePitch + j] = r.w[j];
    __syncwarp();
    const uint16_t* s16 = reinterpret_cast<const uint16_t*>(stage);
    uint16_t* dst = reinterpret_cast<uint16_t*>(block) + lane;
    if (lane < b.cols) {
#pragma unroll 8
        for (int i = 0; i < 32; ++i)
            if (i < b.rows) dst[i * ld] = s16[i * (2 * kStagePitch) + lane];
    }
}

// larger magnitude, as bits: unlike fmaxf it keeps a NaN, which then reaches the whole row of the result
__device__ __forceinline__ unsigned top_bits(unsigned top, float v) { return max(top, __float_as_uint(v) & 0x7fffffffu); }

// 32 columns of scales or biases in this warp's shared memory (16-byte aligned), four at a time: the tensor cores take
// nearly all of the shared memory's bandwidth for their operands, and one access per column and row made the GEMM 12 %
// slower than its plain form.
struct Cols32 {
    const float* p;
    __device__ __forceinline__ float4 four(int j) const { return *reinterpret_cast<const float4*>(p + 4 * j); }
};
__device__ __forceinline__ float at(const float4& v, int k) { return k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w; }

// Column scales and biases of a tile -> a warp's shared copy (one CTA per tile kernel)
__device__ __forceinline__ void stage_columns(const Params& p, float* sbs, float* bias_s, int lane, int count, int first) {
    for (int j = lane; j < count; j += 32) {
        const int c = first + j;
        sbs[j] = c < p.N ? __ldg(p.sb + c) : 0.0f;
        bias_s[j] = c < p.N && p.bias != nullptr ? __bfloat162float(p.bias[c]) : 0.0f;
    }
}

// y of 32 columns from the accumulators of one row
template <int ACT>
__device__ __forceinline__ Row32 linear_values(const uint32_t (&r)[32], float sa, Cols32 sb, Cols32 bias, bool has_res,
                                               const Row32& res) {
    Row32 out;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 s4 = sb.four(j), b4 = bias.four(j);
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = 4 * j + k;
            y[k] = act_value<ACT>(scaled(r[e], sa, at(s4, k), at(b4, k)));
            if (has_res) y[k] = __fadd_rn(y[k], row32_at(res, e));
        }
        out.w[2 * j] = pack_bf16x2_rn(y[0], y[1]);
        out.w[2 * j + 1] = pack_bf16x2_rn(y[2], y[3]);
    }
    return out;
}

// One finished accumulator of NCOLS columns (one CTA per tile kernel): this thread owns tile row `row`.
template <int NCOLS>
__device__ __forceinline__ void drain_linear(const Params& p, uint32_t t_lane, const float* sbs, const float* bias_s, int row,
                                             bool row_ok, int n0, bool vec_ok) {
    const float sa = row_ok ? __ldg(p.sa + row) : 0.0f;
    const bool has_res = p.resid != nullptr && row_ok;
    const bool res_vec = row_vector_ok(p.resid, p.ldr);
#pragma unroll 1
    for (int cc = 0; cc < NCOLS / 32; ++cc) {
        const int n = n0 + cc * 32;
        Row32 res = {};
        if (has_res && n < p.N) load_row32(res, p.resid + (int64_t)row * p.ldr + n, p.N - n, res_vec);
        uint32_t r[32];
        __syncwarp();  // tcgen05.ld is warp-collective: reconverge after the stores
        ptx::tmem_ld_32x32b_x32(t_lane + cc * 32, r);
        ptx::tmem_ld_wait();
        if (row_ok && n < p.N) {
            Row32 out;
            with_act(p.act, [&](auto a) {
                out = linear_values<decltype(a)::value>(r, sa, {sbs + cc * 32}, {bias_s + cc * 32}, has_res, res);
            });
            store_row32(static_cast<__nv_bfloat16*>(p.C) + (int64_t)row * p.ldc + n, out, p.N - n, vec_ok);
        }
    }
}

// h of 32 outputs from the accumulators of their gates and ups
template <int ACT>
__device__ __forceinline__ Row32 gated_values(const uint32_t (&g)[32], const uint32_t (&u)[32], float sa, Cols32 sg, Cols32 bg,
                                              Cols32 su, Cols32 bu) {
    Row32 out;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 sg4 = sg.four(j), bg4 = bg.four(j), su4 = su.four(j), bu4 = bu.four(j);
        float h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = 4 * j + k;
            h[k] = act_value<ACT>(scaled(g[e], sa, at(sg4, k), at(bg4, k))) * scaled(u[e], sa, at(su4, k), at(bu4, k));
        }
        out.w[2 * j] = pack_bf16x2_rn(h[0], h[1]);
        out.w[2 * j + 1] = pack_bf16x2_rn(h[2], h[3]);
    }
    return out;
}

__device__ __forceinline__ void store4f(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// dz of 32 columns -> dz (16-byte aligned); returns the largest |dz * sb| as bits, together with `top`
template <int ACT>
__device__ __forceinline__ unsigned linear_gradients(const uint32_t (&r)[32], float sa, Cols32 sb, Cols32 bias, const Row32& dy,
                                                     float* dz, bool store, unsigned top) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 s4 = sb.four(j), b4 = bias.four(j);
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = 4 * j + k;
            v[k] = row32_at(dy, e) * act_value_slope<ACT>(scaled(r[e], sa, at(s4, k), at(b4, k))).y;
            top = top_bits(top, v[k] * at(s4, k));
        }
        if (store) store4f(dz + 4 * j, v);
    }
    return top;
}

// dg and du of 32 outputs
template <int ACT>
__device__ __forceinline__ unsigned gated_gradients(const uint32_t (&g)[32], const uint32_t (&u)[32], float sa, Cols32 sg,
                                                    Cols32 bg, Cols32 su, Cols32 bu, const Row32& dh, float* dg, float* du,
                                                    bool store, unsigned top) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 sg4 = sg.four(j), bg4 = bg.four(j), su4 = su.four(j), bu4 = bu.four(j);
        float vg[4], vu[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = 4 * j + k;
            const float2 vs = act_value_slope<ACT>(scaled(g[e], sa, at(sg4, k), at(bg4, k)));
            const float d = row32_at(dh, e);
            vg[k] = d * scaled(u[e], sa, at(su4, k), at(bu4, k)) * vs.y;
            vu[k] = d * vs.x;
            top = top_bits(top_bits(top, vg[k] * at(sg4, k)), vu[k] * at(su4, k));
        }
        if (store) {
            store4f(dg + 4 * j, vg);
            store4f(du + 4 * j, vu);
        }
    }
    return top;
}

// Split-K epilogues of the weight-streaming kernels (see reduce_partials_and_store): the item's partials come through
// distributed shared memory, its residual from HBM at the same time.
__device__ __forceinline__ void store4(const Params& p, int row, int n, const float (&v)[4], bool vec) {
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.C) + (int64_t)row * p.ldc + n;
    const uint32_t lo = pack_bf16x2_rn(v[0], v[1]), hi = pack_bf16x2_rn(v[2], v[3]);
    if (vec && n + 4 <= p.N) {
        *reinterpret_cast<uint2*>(out) = make_uint2(lo, hi);
    } else {
        const uint16_t h4[4] = {(uint16_t)(lo & 0xffffu), (uint16_t)(lo >> 16), (uint16_t)(hi & 0xffffu), (uint16_t)(hi >> 16)};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < p.N) reinterpret_cast<uint16_t*>(out)[j] = h4[j];
    }
}

// GATED: rows [0, 64) of the weight tile are gates, [64, 128) the ups of the same outputs; 16 groups of four outputs
// per token instead of 32.
template <int MAXS, int U, bool GATED>
__device__ __forceinline__ void reduce_partials_fused(const Params& p, const uint32_t (&peer_base)[MAXS], int S, int cols_lo,
                                                      int cols_hi, int n0, int tid, int nthreads, const float* sa_s,
                                                      const float* sb_s, const float* bias_s) {
    constexpr int kGroups = GATED ? 16 : 32, kShift = GATED ? 4 : 5, kHalves = GATED ? 2 : 1;
    const bool vec_store = (p.ldc % 4 == 0) && ((reinterpret_cast<uintptr_t>(p.C) & 7) == 0);
    const bool res_vec = (p.ldr % 4 == 0) && ((reinterpret_cast<uintptr_t>(p.resid) & 7) == 0);
    const int items = (cols_hi - cols_lo) * kGroups;
    for (int it0 = tid; it0 < items; it0 += nthreads * U) {
        uint4 v[U][kHalves][MAXS];
        uint2 res[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = it0 + u * nthreads;
            res[u] = make_uint2(0u, 0u);
            if (it < items) {
                const int c = cols_lo + (it >> kShift), g = it & (kGroups - 1);
                if (!GATED && p.resid != nullptr) {
                    const int n = n0 + g * 4;
                    const __nv_bfloat16* rp = p.resid + (int64_t)c * p.ldr + n;
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
        float z[U][kHalves][4];
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
                for (int j = 0; j < 4; ++j)
                    z[u][h][j] = scaled((uint32_t)a[j], sa, sb_s[h * 64 + g * 4 + j], bias_s[h * 64 + g * 4 + j]);
            }
        }
        // one choice of the activation for all items: a tile's epilogue runs once, so its instructions are fetched cold
        with_act(p.act, [&](auto act) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    z[u][0][j] = act_value<decltype(act)::value>(z[u][0][j]);
                    if constexpr (GATED) z[u][0][j] *= z[u][kHalves - 1][j];
                }
            }
        });
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = it0 + u * nthreads;
            if (it >= items) break;
            const int c = cols_lo + (it >> kShift), n = n0 + (it & (kGroups - 1)) * 4;
            if (n >= p.N) continue;
            if (!GATED && p.resid != nullptr) {
                z[u][0][0] = __fadd_rn(z[u][0][0], bf16lo_to_f32(res[u].x));
                z[u][0][1] = __fadd_rn(z[u][0][1], bf16hi_to_f32(res[u].x));
                z[u][0][2] = __fadd_rn(z[u][0][2], bf16lo_to_f32(res[u].y));
                z[u][0][3] = __fadd_rn(z[u][0][3], bf16hi_to_f32(res[u].y));
            }
            store4(p, c, n, z[u][0], vec_store);
        }
    }
}

// With no more items than threads (few tokens) one item per thread: the loop body for U of them would be fetched, cold, to
// do nothing, which cost 1.4 us of a 9 us kernel.
template <int MAXS, int U, bool GATED>
__device__ __forceinline__ void reduce_partials_fused_sized(const Params& p, const uint32_t (&peer_base)[MAXS], int S, int cols_lo,
                                                            int cols_hi, int n0, int tid, int nthreads, const float* scales) {
    if ((cols_hi - cols_lo) * (GATED ? 16 : 32) <= nthreads)
        reduce_partials_fused<MAXS, 1, GATED>(p, peer_base, S, cols_lo, cols_hi, n0, tid, nthreads, scales, scales + 256, scales + 384);
    else
        reduce_partials_fused<MAXS, U, GATED>(p, peer_base, S, cols_lo, cols_hi, n0, tid, nthreads, scales, scales + 256, scales + 384);
}

}  // namespace
}  // namespace w8a8

#endif  // W8A8_GEMM_I8_EPILOGUES_CUH
