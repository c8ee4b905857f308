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

// Column scales and biases of a tile -> this warp's shared copy.  Columns [0, half) of the tile come from output column
// n0 on, columns [half, 2 half) from `second` on (a gated tile's up rows, or simply the next columns).
__device__ __forceinline__ void stage_columns(const Params& p, float* sbs, float* bias_s, int lane, int half, int first,
                                              int second, int first_end, int second_end) {
    for (int j = lane; j < 2 * half; j += 32) {
        const int c = j < half ? first + j : second + (j - half);
        const bool ok = c < (j < half ? first_end : second_end);
        sbs[j] = ok ? __ldg(p.sb + c) : 0.0f;
        bias_s[j] = ok && p.bias != nullptr ? __bfloat162float(p.bias[c]) : 0.0f;
    }
}

// One finished accumulator of NCOLS columns: this thread owns tile row `row`.  The residual of the next 32 columns is
// requested before the current ones are worked on.
template <int NCOLS>
__device__ __forceinline__ void drain_linear(const Params& p, uint32_t t_lane, const float* sbs, const float* bias_s, int row,
                                             bool row_ok, int n0, bool vec_ok) {
    const float sa = row_ok ? __ldg(p.sa + row) : 0.0f;
    const bool has_res = p.resid != nullptr && row_ok;
    const bool res_vec = row_vector_ok(p.resid, p.ldr);
    const __nv_bfloat16* rrow = p.resid + (int64_t)row * p.ldr;
    Row32 res = {};
    if (has_res && n0 < p.N) load_row32(res, rrow + n0, p.N - n0, res_vec);
#pragma unroll 1
    for (int cc = 0; cc < NCOLS / 32; ++cc) {
        uint32_t r[32];
        __syncwarp();  // tcgen05.ld is warp-collective: reconverge after the stores
        ptx::tmem_ld_32x32b_x32(t_lane + cc * 32, r);
        const int n = n0 + cc * 32;
        Row32 next = {};
        if (has_res && cc + 1 < NCOLS / 32 && n + 32 < p.N) load_row32(next, rrow + n + 32, p.N - n - 32, res_vec);
        ptx::tmem_ld_wait();
        if (row_ok && n < p.N) {
            Row32 out;
            with_act(p.act, [&](auto a) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    float y[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int e = 2 * j + h;
                        y[h] = act_value<decltype(a)::value>(scaled(r[e], sa, sbs[cc * 32 + e], bias_s[cc * 32 + e]));
                        if (has_res) y[h] = __fadd_rn(y[h], row32_at(res, e));
                    }
                    out.w[j] = pack_bf16x2_rn(y[0], y[1]);
                }
            });
            store_row32(static_cast<__nv_bfloat16*>(p.C) + (int64_t)row * p.ldc + n, out, p.N - n, vec_ok);
        }
        res = next;
    }
}

// A gated tile: accumulator columns [0, 128) are gates, [128, 256) the ups of the same 128 outputs.
__device__ __forceinline__ void drain_gated(const Params& p, uint32_t t_lane, const float* sbs, const float* bias_s, int row,
                                            bool row_ok, int n0, bool vec_ok) {
    const float sa = row_ok ? __ldg(p.sa + row) : 0.0f;
#pragma unroll 1
    for (int cc = 0; cc < 4; ++cc) {
        uint32_t g[32], u[32];
        __syncwarp();
        ptx::tmem_ld_32x32b_x32(t_lane + cc * 32, g);
        ptx::tmem_ld_32x32b_x32(t_lane + 128 + cc * 32, u);
        ptx::tmem_ld_wait();
        const int n = n0 + cc * 32;
        if (!row_ok || n >= p.N) continue;
        Row32 out;
        with_act(p.act, [&](auto a) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                float h[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int e = 2 * j + k, c = cc * 32 + e;
                    h[k] = act_value<decltype(a)::value>(scaled(g[e], sa, sbs[c], bias_s[c])) *
                           scaled(u[e], sa, sbs[128 + c], bias_s[128 + c]);
                }
                out.w[j] = pack_bf16x2_rn(h[0], h[1]);
            }
        });
        store_row32(static_cast<__nv_bfloat16*>(p.C) + (int64_t)row * p.ldc + n, out, p.N - n, vec_ok);
    }
}

__device__ __forceinline__ void store_f32x2(float* p, float a, float b, int n_left, bool vec) {
    if (vec) {   // n_left is even then
        if (n_left >= 2) *reinterpret_cast<float2*>(p) = make_float2(a, b);
    } else {
        if (n_left >= 1) p[0] = a;
        if (n_left >= 2) p[1] = b;
    }
}
// larger magnitude, as bits: unlike fmaxf it keeps a NaN, which then reaches the whole row of the result
__device__ __forceinline__ unsigned top_bits(unsigned top, float v) { return max(top, __float_as_uint(v) & 0x7fffffffu); }

template <int NCOLS>
__device__ __forceinline__ void drain_linear_grad(const Params& p, uint32_t t_lane, const float* sbs, const float* bias_s,
                                                  int row, bool row_ok, int n0) {
    const float sa = row_ok ? __ldg(p.sa + row) : 0.0f;
    const bool dy_vec = row_vector_ok(p.resid, p.ldr), z_vec = p.ldc % 4 == 0;
    unsigned top = 0;
#pragma unroll 1
    for (int cc = 0; cc < NCOLS / 32; ++cc) {
        uint32_t r[32];
        const int n = n0 + cc * 32, left = p.N - n;
        Row32 dy = {};
        if (row_ok && left > 0) load_row32(dy, p.resid + (int64_t)row * p.ldr + n, left, dy_vec);
        __syncwarp();
        ptx::tmem_ld_32x32b_x32(t_lane + cc * 32, r);
        ptx::tmem_ld_wait();
        if (!row_ok || left <= 0) continue;
        float* out = static_cast<float*>(p.C) + (int64_t)row * p.ldc + n;
        with_act(p.act, [&](auto a) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                float dz[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int e = j + k, c = cc * 32 + e;
                    dz[k] = row32_at(dy, e) * act_value_slope<decltype(a)::value>(scaled(r[e], sa, sbs[c], bias_s[c])).y;
                    if (e < left) top = top_bits(top, dz[k] * sbs[c]);
                }
                store_f32x2(out + j, dz[0], dz[1], left - j, z_vec);
            }
        });
    }
    if (row_ok && top != 0) atomicMax(p.row_top + row, top);
}

__device__ __forceinline__ void drain_gated_grad(const Params& p, uint32_t t_lane, const float* sbs, const float* bias_s,
                                                 int row, bool row_ok, int n0) {
    const float sa = row_ok ? __ldg(p.sa + row) : 0.0f;
    const bool dh_vec = row_vector_ok(p.resid, p.ldr), z_vec = p.ldc % 4 == 0 && p.inter % 2 == 0;
    unsigned top = 0;
#pragma unroll 1
    for (int cc = 0; cc < 4; ++cc) {
        uint32_t g[32], u[32];
        const int n = n0 + cc * 32, left = p.N - n;
        Row32 dh = {};
        if (row_ok && left > 0) load_row32(dh, p.resid + (int64_t)row * p.ldr + n, left, dh_vec);
        __syncwarp();
        ptx::tmem_ld_32x32b_x32(t_lane + cc * 32, g);
        ptx::tmem_ld_32x32b_x32(t_lane + 128 + cc * 32, u);
        ptx::tmem_ld_wait();
        if (!row_ok || left <= 0) continue;
        float* out_g = static_cast<float*>(p.C) + (int64_t)row * p.ldc + n;
        float* out_u = out_g + p.inter;
        with_act(p.act, [&](auto a) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                float dg[2], du[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int e = j + k, c = cc * 32 + e;
                    const float2 vs = act_value_slope<decltype(a)::value>(scaled(g[e], sa, sbs[c], bias_s[c]));
                    const float zu = scaled(u[e], sa, sbs[128 + c], bias_s[128 + c]), d = row32_at(dh, e);
                    dg[k] = d * zu * vs.y;
                    du[k] = d * vs.x;
                    if (e < left) top = top_bits(top_bits(top, dg[k] * sbs[c]), du[k] * sbs[128 + c]);
                }
                store_f32x2(out_g + j, dg[0], dg[1], left - j, z_vec);
                store_f32x2(out_u + j, du[0], du[1], left - j, z_vec);
            }
        });
    }
    if (row_ok && top != 0) atomicMax(p.row_top + row, top);
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
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = it0 + u * nthreads;
            if (it >= items) break;
            const int c = cols_lo + (it >> kShift), g = it & (kGroups - 1);
            const int n = n0 + g * 4;
            if (n >= p.N) continue;
            const float sa = sa_s[c];
            float z[kHalves][4];
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                int a[4] = {0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < MAXS; ++r) {
                    if (r < S) {
                        a[0] += (int)v[u][h][r].x; a[1] += (int)v[u][h][r].y; a[2] += (int)v[u][h][r].z; a[3] += (int)v[u][h][r].w;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    z[h][j] = scaled((uint32_t)a[j], sa, sb_s[h * 64 + g * 4 + j], bias_s[h * 64 + g * 4 + j]);
            }
            float y[4];
            with_act(p.act, [&](auto act) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] = act_value<decltype(act)::value>(z[0][j]);
                    if constexpr (GATED) y[j] *= z[kHalves - 1][j];
                }
            });
            if (!GATED && p.resid != nullptr) {
                y[0] = __fadd_rn(y[0], bf16lo_to_f32(res[u].x));
                y[1] = __fadd_rn(y[1], bf16hi_to_f32(res[u].x));
                y[2] = __fadd_rn(y[2], bf16lo_to_f32(res[u].y));
                y[3] = __fadd_rn(y[3], bf16hi_to_f32(res[u].y));
            }
            store4(p, c, n, y, vec_store);
        }
    }
}

}  // namespace
}  // namespace w8a8

#endif  // W8A8_GEMM_I8_EPILOGUES_CUH
