// Layer norm of bf16 rows: forward (optionally with the residual add in front and the int8 quantiser behind) and
// backward with the gradients of weight and bias.
//
//   a    = x, or bf16(res + x), which is also what the residual is overwritten with
//   mean = sum(a) / K        rstd = 1 / sqrt(sum((a - mean)^2) / K + eps)        xhat = (a - mean) * rstd
//   y    = xhat * w + b                      -> bf16, or int8 codes and one scale per row (the quantiser of
//                                               per_token_quant_int8 on the unrounded fp32 y)
//   dx   = rstd * (t - mean(t) - xhat * mean(t * xhat)) [+ dres]   with t = dy * w
//   dw   = sum over rows of dy * xhat        db = sum over rows of dy              (fp32)
//
// The sum that is normalised is the ROUNDED one, the residual as it is stored: the backward pass has only that row,
// and differentiates exactly the function that ran (add_rmsnorm_quant, which has no backward pass, normalises the
// unrounded sum).  The variance comes from the deviations, not from sum(a^2) - mean^2, which loses every digit of a row
// with a large mean.  All statistics and sums are fp32.
//
// Everything here is bound by HBM.  A row belongs to a group of T threads (T a multiple of 32, chosen so that the row
// fits the group's registers, packed as it came), is read once and stays on chip between its reductions.  Rows move in
// accesses of eight elements where width and addresses allow, else of two, else of one; rows wider than the registers
// hold are read again for each reduction (the *_wide kernels).  Arithmetic is on pairs (packed f32x2), without which the
// backward pass was bound by its instructions (52 % of the issue slots, 38 % of HBM).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "launch_common.h"
#include "sm100_ptx.cuh"
#include "w8a8_arith.cuh"

namespace w8a8 {
namespace {

constexpr int kMaxGroupThreads = 1024;
constexpr uint32_t kFullWarp = 0xffffffffu;

// W consecutive bf16 (8, 2 or 1) in one access, and the same as fp32: pairs, or a single value for W = 1
template <int W>
struct Pack {
    uint32_t w[W == 8 ? 4 : 1];
};
template <int W>
__device__ __forceinline__ Pack<W> load_pack(const __nv_bfloat16* p) {
    Pack<W> v;
    if constexpr (W == 8) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        v.w[0] = q.x; v.w[1] = q.y; v.w[2] = q.z; v.w[3] = q.w;
    } else if constexpr (W == 2) {
        v.w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
        v.w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
    return v;
}
template <int W>
__device__ __forceinline__ void store_pack(__nv_bfloat16* p, const Pack<W>& v) {
    if constexpr (W == 8) *reinterpret_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    else if constexpr (W == 2) *reinterpret_cast<uint32_t*>(p) = v.w[0];
    else *reinterpret_cast<uint16_t*>(p) = (uint16_t)v.w[0];
}
template <int W>
struct Vals {
    using T = float2;
    static constexpr int kN = W / 2;
};
template <>
struct Vals<1> {
    using T = float;
    static constexpr int kN = 1;
};
__device__ __forceinline__ float mul(float a, float b) { return __fmul_rn(a, b); }
__device__ __forceinline__ float2 mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float add(float a, float b) { return __fadd_rn(a, b); }
__device__ __forceinline__ float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float fma(float a, float b, float c) { return __fmaf_rn(a, b, c); }
__device__ __forceinline__ float2 fma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float total(float a) { return a; }
__device__ __forceinline__ float total(float2 a) { return __fadd_rn(a.x, a.y); }
__device__ __forceinline__ float top_of(float t, float a) { return fmaxf(t, fabsf(a)); }
__device__ __forceinline__ float top_of(float t, float2 a) { return max3_abs(t, a.x, a.y); }
template <typename T>
__device__ __forceinline__ T all(float v) {
    if constexpr (sizeof(T) == 8) return splat2(v);
    else return v;
}
template <int W>
__device__ __forceinline__ typename Vals<W>::T value(const Pack<W>& v, int i) {
    if constexpr (W == 1) return bf16lo_to_f32(v.w[0]);
    else return bf16x2_to_f32x2(v.w[i]);
}
__device__ __forceinline__ uint32_t rounded(float a) { return pack_bf16x2_rn(a, 0.0f) & 0xffffu; }
__device__ __forceinline__ uint32_t rounded(float2 a) { return pack_bf16x2_rn(a.x, a.y); }

// Sums over the threads of one group: shuffles inside a warp, one exchange through shared memory between the warps.
// Two slots of `red` take turns, so a group needs one barrier per reduction: a slot is written again only after the
// barrier of the reduction in between.
struct Group {
    float2* red;       // [2][32] of this group
    int threads;       // multiple of 32
    int id;            // hardware barrier of the group: 1 + index in the CTA
    int turn = 0;
    __device__ __forceinline__ void barrier() const { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
    template <typename Op>
    __device__ __forceinline__ float2 reduce(float2 v, Op op) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            v = op(v, make_float2(__shfl_xor_sync(kFullWarp, v.x, o), __shfl_xor_sync(kFullWarp, v.y, o)));
        if (threads == 32) return v;
        const int lane = threadIdx.x & 31, warp = (threadIdx.x % threads) >> 5, warps = threads >> 5;
        float2* slot = red + 32 * turn;
        turn ^= 1;
        if (lane == 0) slot[warp] = v;
        barrier();
        v = slot[lane < warps ? lane : 0];
        if (lane >= warps) v = make_float2(0.0f, 0.0f);   // neutral for sums, and for maxima of magnitudes
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            v = op(v, make_float2(__shfl_xor_sync(kFullWarp, v.x, o), __shfl_xor_sync(kFullWarp, v.y, o)));
        return v;
    }
    __device__ __forceinline__ float2 sum2(float2 v) {
        return reduce(v, [](float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); });
    }
    __device__ __forceinline__ float sum(float v) {
        return reduce(make_float2(v, 0.0f), [](float2 a, float2 b) { return make_float2(a.x + b.x, 0.0f); }).x;
    }
    __device__ __forceinline__ float max(float v) {
        return reduce(make_float2(v, 0.0f), [](float2 a, float2 b) { return make_float2(fmaxf(a.x, b.x), 0.0f); }).x;
    }
};

__device__ __forceinline__ float rstd_of(float sumsq, int K, float eps) {
    return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sumsq, (float)K), eps)));
}

struct NormArgs {
    const __nv_bfloat16* x;
    __nv_bfloat16* res;        // null: no residual
    const __nv_bfloat16* w;
    const __nv_bfloat16* b;
    __nv_bfloat16* y;          // bf16 output, or null when the codes are wanted
    int8_t* q;
    float* s;
    float* mean;
    float* rstd;
    int M, K, T;
    float eps;
};

// ---- forward: blockDim = R groups of T threads, one row per group, V accesses of W elements per thread -------------
// The row stays packed (four registers per eight elements) and is widened again for each pass: with 62 registers a
// thread for a widened row, 28 warps an SM did not cover the loads' latency (53 % of HBM).
template <int W, int V, int THREADS, int CTAS, bool ADD, bool QUANT>
__global__ void __launch_bounds__(THREADS, CTAS) layernorm_kernel(const NormArgs p) {
    using T = typename Vals<W>::T;
    constexpr int N = Vals<W>::kN;
    __shared__ float2 red_all[8 * 64];   // a CTA holds at most eight groups
    ptx::grid_launch_dependents();  // a GEMM launched to overlap this kernel may start its set-up and weight loads
    const int G = p.T, g = threadIdx.x / G, t = threadIdx.x - g * G;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / G) + g;
    if (row >= p.M) return;  // whole groups: nobody is left waiting at the group's barrier
    Group grp{red_all + 64 * g, G, 1 + g};
    const int K = p.K;
    const __nv_bfloat16* x = p.x + row * K;
    Pack<W> a[V];
    Pack<W> w1, b1;                      // a thread with one access has its weight and bias requested with the row
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (t + j * G) * W;
        if (c < K) {
            a[j] = load_pack<W>(x + c);
            if constexpr (V == 1) {
                w1 = load_pack<W>(p.w + c);
                b1 = load_pack<W>(p.b + c);
            }
        }
    }
    T acc = all<T>(0.0f);
    if constexpr (ADD) {
        Pack<W> r[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (t + j * G) * W;
            if (c < K) r[j] = load_pack<W>(p.res + row * K + c);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (t + j * G) * W;
            if (c < K) {
#pragma unroll
                for (int i = 0; i < N; ++i) a[j].w[i] = rounded(add(value<W>(r[j], i), value<W>(a[j], i)));
                store_pack<W>(p.res + row * K + c, a[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if ((t + j * G) * W < K) {
#pragma unroll
            for (int i = 0; i < N; ++i) acc = add(acc, value<W>(a[j], i));
        }
    }
    const float mean = __fdiv_rn(grp.sum(total(acc)), (float)K);
    acc = all<T>(0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if ((t + j * G) * W < K) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const T d = add(value<W>(a[j], i), all<T>(-mean));
                acc = fma(d, d, acc);
            }
        }
    }
    const float rstd = rstd_of(grp.sum(total(acc)), K, p.eps);
    if (t == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
    // y of access j; the quantiser evaluates it twice (largest magnitude, codes) rather than hold it
    auto y_of = [&](int j, int c, T (&y)[N]) {
        const Pack<W> w = V == 1 ? w1 : load_pack<W>(p.w + c), b = V == 1 ? b1 : load_pack<W>(p.b + c);
#pragma unroll
        for (int i = 0; i < N; ++i)
            y[i] = fma(mul(add(value<W>(a[j], i), all<T>(-mean)), all<T>(rstd)), value<W>(w, i), value<W>(b, i));
    };
    if constexpr (!QUANT) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (t + j * G) * W;
            if (c < K) {
                T y[N];
                y_of(j, c, y);
                Pack<W> o;
#pragma unroll
                for (int i = 0; i < N; ++i) o.w[i] = rounded(y[i]);
                store_pack<W>(p.y + row * K + c, o);
            }
        }
    } else {
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (t + j * G) * W;
            if (c < K) {
                T y[N];
                y_of(j, c, y);
#pragma unroll
                for (int i = 0; i < N; ++i) top = top_of(top, y[i]);
            }
        }
        float scale, inv;
        scale_from_amax(grp.max(top), scale, inv);
        if (t == 0) p.s[row] = scale;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (t + j * G) * W;
            if (c < K) {
                T y[N];
                y_of(j, c, y);
                int8_t* q = p.q + row * K + c;
                if constexpr (W == 8) {
                    uint32_t o[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[2 * i] = quant_rn_lowbyte(y[i].x, inv);
                        o[2 * i + 1] = quant_rn_lowbyte(y[i].y, inv);
                    }
                    *reinterpret_cast<uint2*>(q) = make_uint2(pack_lowbytes(o[0], o[1], o[2], o[3]), pack_lowbytes(o[4], o[5], o[6], o[7]));
                } else if constexpr (W == 2) {
                    const uint32_t lo = quant_rn_lowbyte(y[0].x, inv) & 0xffu, hi = quant_rn_lowbyte(y[0].y, inv) & 0xffu;
                    *reinterpret_cast<uint16_t*>(q) = (uint16_t)(lo | (hi << 8));
                } else {
                    *q = (int8_t)(quant_rn_lowbyte(y[0], inv) & 0xffu);
                }
            }
        }
    }
}

// rows wider than the registers hold: one CTA per row, every reduction reads the row again (it stays in L1 / L2)
template <bool ADD, bool QUANT>
__global__ void __launch_bounds__(kMaxGroupThreads) layernorm_wide_kernel(const NormArgs p) {
    __shared__ float2 red_all[64];
    ptx::grid_launch_dependents();
    const int64_t row = blockIdx.x;
    Group grp{red_all, (int)blockDim.x, 1};
    const int K = p.K, T = blockDim.x;
    // with a residual the rounded sum is stored first and read back by the thread that stored it
    const __nv_bfloat16* a = ADD ? p.res + row * K : p.x + row * K;
    float sum = 0.0f;
    for (int c = threadIdx.x; c < K; c += T) {
        if constexpr (ADD)
            p.res[row * K + c] = __float2bfloat16_rn(__fadd_rn(__bfloat162float(p.res[row * K + c]), __bfloat162float(p.x[row * K + c])));
        sum += __bfloat162float(a[c]);
    }
    const float mean = __fdiv_rn(grp.sum(sum), (float)K);
    float dev = 0.0f;
    for (int c = threadIdx.x; c < K; c += T) {
        const float d = __bfloat162float(a[c]) - mean;
        dev = fmaf(d, d, dev);
    }
    const float rstd = rstd_of(grp.sum(dev), K, p.eps);
    if (threadIdx.x == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
    auto norm = [&](int c) {
        return fmaf((__bfloat162float(a[c]) - mean) * rstd, __bfloat162float(p.w[c]), __bfloat162float(p.b[c]));
    };
    if constexpr (!QUANT) {
        for (int c = threadIdx.x; c < K; c += T) p.y[row * K + c] = __float2bfloat16_rn(norm(c));
    } else {
        float top = 0.0f, scale, inv;
        for (int c = threadIdx.x; c < K; c += T) top = fmaxf(top, fabsf(norm(c)));
        scale_from_amax(grp.max(top), scale, inv);
        if (threadIdx.x == 0) p.s[row] = scale;
        for (int c = threadIdx.x; c < K; c += T) p.q[row * K + c] = (int8_t)quant_rn(norm(c), inv);
    }
}

struct NormBwdArgs {
    const __nv_bfloat16* dy;
    const __nv_bfloat16* x;
    const float* mean;
    const float* rstd;
    const __nv_bfloat16* w;
    const __nv_bfloat16* dres;   // null: none
    __nv_bfloat16* dx;
    float* partial;              // [gridDim.x][2][K]: this CTA's share of dw and db
    int M, K, T;
};

// ---- backward: one CTA per SM, its groups walk rows; every thread keeps the sums of its own columns in registers ----
// AHEAD: the next row's loads are issued before the current row's reduction, so HBM stays busy across the group's
// barrier; only where both rows fit the registers that THREADS threads leave each (72 for 896, 64 for 1024).
template <int W, int V, int THREADS, bool RES, bool AHEAD>
__global__ void __launch_bounds__(THREADS, 1) layernorm_backward_kernel(const NormBwdArgs p) {
    using T = typename Vals<W>::T;
    constexpr int N = Vals<W>::kN;
    __shared__ float2 red_all[32 * 64];
    extern __shared__ float cols[];   // [R][2][K]: the groups' column sums, when there is more than one group
    const int G = p.T, R = blockDim.x / G, g = threadIdx.x / G, t = threadIdx.x - g * G;
    Group grp{red_all + 64 * g, G, 1 + g};
    const int K = p.K;
    const float inv_k = __fdiv_rn(1.0f, (float)K);
    T dw[V][N], db[V][N];
    Pack<W> w[V], nx[V], ny[V], nr[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int i = 0; i < N; ++i) dw[j][i] = db[j][i] = all<T>(0.0f);
        if ((t + j * G) * W < K) w[j] = load_pack<W>(p.w + (t + j * G) * W);
    }
    float nmean = 0.0f, nrstd = 0.0f;
    const int64_t step = (int64_t)gridDim.x * R;
    auto fetch = [&](int64_t row) {
        if (row < p.M) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = (t + j * G) * W;
                if (c < K) {
                    nx[j] = load_pack<W>(p.x + row * K + c);
                    ny[j] = load_pack<W>(p.dy + row * K + c);
                    if constexpr (RES) nr[j] = load_pack<W>(p.dres + row * K + c);
                }
            }
            nmean = __ldg(p.mean + row);
            nrstd = __ldg(p.rstd + row);
        }
    };
    int64_t row = (int64_t)blockIdx.x * R + g;
    fetch(row);
    for (; row < p.M; row += step) {
        T xh[V][N], tv[V][N];
        Pack<W> r[V];
        const float rstd = nrstd;
        const T rs = all<T>(nrstd), shift = all<T>(-nmean);
        T c0 = all<T>(0.0f), c1 = all<T>(0.0f);   // sums of t = dy * w and of t * xhat
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if ((t + j * G) * W < K) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const T y = value<W>(ny[j], i);
                    xh[j][i] = mul(add(value<W>(nx[j], i), shift), rs);
                    tv[j][i] = mul(y, value<W>(w[j], i));
                    dw[j][i] = fma(y, xh[j][i], dw[j][i]);
                    db[j][i] = add(db[j][i], y);
                    c0 = add(c0, tv[j][i]);
                    c1 = fma(tv[j][i], xh[j][i], c1);
                }
                if constexpr (RES) r[j] = nr[j];
            }
        }
        if constexpr (AHEAD) fetch(row + step);
        const float2 c = grp.sum2(make_float2(total(c0), total(c1)));
        const T m0 = all<T>(-c.x * inv_k), m1 = all<T>(-c.y * inv_k), out_scale = all<T>(rstd);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int col = (t + j * G) * W;
            if (col < K) {
                Pack<W> o;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const T d = fma(xh[j][i], m1, add(tv[j][i], m0));
                    if constexpr (RES) o.w[i] = rounded(fma(d, out_scale, value<W>(r[j], i)));
                    else o.w[i] = rounded(mul(d, out_scale));
                }
                store_pack<W>(p.dx + row * K + col, o);
            }
        }
        if constexpr (!AHEAD) fetch(row + step);
    }
    // column sums of the CTA's groups, added in the groups' order
    float* out = p.partial + (int64_t)blockIdx.x * 2 * K;
    float* to = R == 1 ? out : cols + (size_t)g * 2 * K;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (t + j * G) * W;
        if (c < K) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (W == 1) {
                    to[c] = dw[j][i];
                    to[K + c] = db[j][i];
                } else {   // c and K are even: 8-byte aligned
                    *reinterpret_cast<float2*>(to + c + 2 * i) = dw[j][i];
                    *reinterpret_cast<float2*>(to + K + c + 2 * i) = db[j][i];
                }
            }
        }
    }
    if (R > 1) {
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * K; i += blockDim.x) {
            float v = 0.0f;
            for (int k = 0; k < R; ++k) v += cols[(size_t)k * 2 * K + i];
            out[i] = v;
        }
    }
}

// rows wider than the registers hold: dx by one CTA per row, then the column sums by a second read
template <bool RES>
__global__ void __launch_bounds__(kMaxGroupThreads) layernorm_backward_wide_kernel(const NormBwdArgs p) {
    __shared__ float2 red_all[64];
    const int64_t row = blockIdx.x;
    Group grp{red_all, (int)blockDim.x, 1};
    const int K = p.K, T = blockDim.x;
    const __nv_bfloat16 *x = p.x + row * K, *dy = p.dy + row * K;
    const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
    float2 c = make_float2(0.0f, 0.0f);
    for (int i = threadIdx.x; i < K; i += T) {
        const float tv = __bfloat162float(dy[i]) * __bfloat162float(p.w[i]);
        c.x += tv;
        c.y = fmaf(tv, (__bfloat162float(x[i]) - mean) * rstd, c.y);
    }
    c = grp.sum2(c);
    c.x = __fdiv_rn(c.x, (float)K);
    c.y = __fdiv_rn(c.y, (float)K);
    for (int i = threadIdx.x; i < K; i += T) {
        const float xh = (__bfloat162float(x[i]) - mean) * rstd;
        const float d = fmaf(-xh, c.y, fmaf(__bfloat162float(dy[i]), __bfloat162float(p.w[i]), -c.x));
        p.dx[row * K + i] = __float2bfloat16_rn(RES ? fmaf(d, rstd, __bfloat162float(p.dres[row * K + i])) : d * rstd);
    }
}
__global__ void __launch_bounds__(256) layernorm_wide_columns_kernel(const NormBwdArgs p) {
    const int c = blockIdx.y * 256 + threadIdx.x;
    if (c >= p.K) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
        const float y = __bfloat162float(p.dy[row * p.K + c]);
        dw = fmaf(y, (__bfloat162float(p.x[row * p.K + c]) - __ldg(p.mean + row)) * __ldg(p.rstd + row), dw);
        db += y;
    }
    float* out = p.partial + (int64_t)blockIdx.x * 2 * p.K;
    out[c] = dw;
    out[p.K + c] = db;
}

// sums of the CTAs' shares, in the CTAs' order inside each of eight slices: 32 columns per CTA
__global__ void __launch_bounds__(256) layernorm_column_sum_kernel(const float* __restrict__ partial, int parts, int K,
                                                                   float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float sh[8][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
    float v = 0.0f;
    if (col < 2 * K) {
#pragma unroll 8
        for (int i = slice; i < parts; i += 8) v += partial[(int64_t)i * 2 * K + col];
    }
    sh[slice][threadIdx.x & 31] = v;
    __syncthreads();
    if (slice == 0 && col < 2 * K) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += sh[k][threadIdx.x & 31];
        if (col < K) dw[col] = s;
        else db[col - K] = s;
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------
int sm_count() {
    static thread_local int cached_dev = -1, cached = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev != cached_dev) {
        cudaDeviceGetAttribute(&cached, cudaDevAttrMultiProcessorCount, dev);
        cached_dev = dev;
    }
    return cached;
}

// threads per row (multiple of 32) when each thread makes at most `v` accesses
int group_threads(int accesses, int v) { return ((accesses + v - 1) / v + 31) / 32 * 32; }

// Widest access that the row length and every address allow
template <typename... P>
int access_width(int K, const P*... ptrs) {
    const uintptr_t bits = (... | reinterpret_cast<uintptr_t>(ptrs));
    return K % 8 == 0 && bits % 16 == 0 ? 8 : K % 2 == 0 && bits % 4 == 0 ? 2 : 1;
}

template <int W, int V, int THREADS, int CTAS, bool ADD, bool QUANT>
int launch_norm(NormArgs p, cudaStream_t st) {
    p.T = group_threads((p.K + W - 1) / W, V);
    // narrow rows share a CTA of up to 256 threads: one row each, at most 8 rows
    const int R = p.T >= 256 ? 1 : 256 / p.T;
    layernorm_kernel<W, V, THREADS, CTAS, ADD, QUANT><<<(p.M + R - 1) / R, R * p.T, 0, st>>>(p);
    return check_launch("layernorm");
}

// Accesses per thread: few rows (fewer than fill the device twice) take one wide access per thread, for latency (8 x 7168:
// 7.3 us with four, FEW_US with one); many rows two to eight, for fewer barriers and reductions per byte.
template <bool ADD, bool QUANT>
int dispatch_norm(const NormArgs& p, cudaStream_t st) {
    int w = access_width(p.K, p.x, p.w, p.b, (const __nv_bfloat16*)p.res, (const __nv_bfloat16*)p.y);
    if (QUANT && w == 8 && (reinterpret_cast<uintptr_t>(p.q) & 7)) w = 2;
    if (QUANT && w == 2 && (reinterpret_cast<uintptr_t>(p.q) & 1)) w = 1;
    if (w == 8) {
        if (p.K <= 8192 && p.M <= 2 * sm_count()) return launch_norm<8, 1, 1024, 1, ADD, QUANT>(p, st);
        if (p.K <= 4096) return launch_norm<8, 2, 256, 6, ADD, QUANT>(p, st);
        if (p.K <= 8192) return launch_norm<8, 4, 256, 5, ADD, QUANT>(p, st);
        if (p.K <= 16384) return launch_norm<8, 8, 256, 3, ADD, QUANT>(p, st);
    } else if (w == 2) {
        if (p.K <= 4096) return launch_norm<2, 4, 512, 2, ADD, QUANT>(p, st);
        if (p.K <= 16384) return launch_norm<2, 8, 1024, 1, ADD, QUANT>(p, st);
    } else {
        if (p.K <= 4096) return launch_norm<1, 4, 1024, 1, ADD, QUANT>(p, st);
        if (p.K <= 16384) return launch_norm<1, 16, 1024, 1, ADD, QUANT>(p, st);
    }
    layernorm_wide_kernel<ADD, QUANT><<<p.M, kMaxGroupThreads, 0, st>>>(p);
    return check_launch("layernorm");
}

constexpr int kWideParts = 64;
// Most CTAs whose column sums the workspace has room for; a launch uses one per SM (148 on a B200).
constexpr int kMaxParts = 160;

template <int W, int V, int THREADS, bool RES, bool AHEAD>
int launch_norm_backward(NormBwdArgs p, float* dw, float* db, int parts, cudaStream_t st) {
    p.T = group_threads((p.K + W - 1) / W, V);
    int R = THREADS / p.T;
    if (p.T != 32 && R > 15) R = 15;   // hardware barriers 1..15; a one-warp group needs none
    const int smem = R > 1 ? R * 2 * p.K * 4 : 0;
    static bool opted_in[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (smem > 32 * 1024 && !(dev >= 0 && dev < 64 && opted_in[dev])) {
        if (cudaFuncSetAttribute(layernorm_backward_kernel<W, V, THREADS, RES, AHEAD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 THREADS * W * V * 8) != cudaSuccess)
            return fail(DSV4_ERR_LAUNCH, "layernorm_backward: cannot raise the dynamic shared memory limit");
        if (dev >= 0 && dev < 64) opted_in[dev] = true;
    }
    const int grid = (int)min((int64_t)parts, ((int64_t)p.M + R - 1) / R);
    layernorm_backward_kernel<W, V, THREADS, RES, AHEAD><<<grid, R * p.T, smem, st>>>(p);
    if (int rc = check_launch("layernorm_backward")) return rc;
    layernorm_column_sum_kernel<<<(2 * p.K + 31) / 32, 256, 0, st>>>(p.partial, grid, p.K, dw, db);
    return check_launch("layernorm_backward");
}

template <bool RES>
int dispatch_norm_backward(const NormBwdArgs& p, float* dw, float* db, int parts, cudaStream_t st) {
    const int w = access_width(p.K, p.x, p.dy, p.w, (const __nv_bfloat16*)p.dx, p.dres);
    if (w == 8) {
        if (p.K <= 7168) return launch_norm_backward<8, 1, 896, RES, true>(p, dw, db, parts, st);
        if (p.K <= 8192) return launch_norm_backward<8, 1, 1024, RES, true>(p, dw, db, parts, st);
        if (p.K <= 16384) return launch_norm_backward<8, 4, 512, RES, true>(p, dw, db, parts, st);
    } else if (w == 2) {
        if (p.K <= 7168) return launch_norm_backward<2, 4, 896, RES, true>(p, dw, db, parts, st);
        if (p.K <= 16384) return launch_norm_backward<2, 16, 512, RES, false>(p, dw, db, parts, st);
    } else {
        if (p.K <= 3584) return launch_norm_backward<1, 4, 896, RES, true>(p, dw, db, parts, st);
        if (p.K <= 8192) return launch_norm_backward<1, 16, 512, RES, true>(p, dw, db, parts, st);
        if (p.K <= 16384) return launch_norm_backward<1, 32, 512, RES, false>(p, dw, db, parts, st);
    }
    layernorm_backward_wide_kernel<RES><<<p.M, kMaxGroupThreads, 0, st>>>(p);
    if (int rc = check_launch("layernorm_backward")) return rc;
    const int rows = min(min(kWideParts, parts), p.M);
    layernorm_wide_columns_kernel<<<dim3(rows, (p.K + 255) / 256), 256, 0, st>>>(p);
    if (int rc = check_launch("layernorm_backward")) return rc;
    layernorm_column_sum_kernel<<<(2 * p.K + 31) / 32, 256, 0, st>>>(p.partial, rows, p.K, dw, db);
    return check_launch("layernorm_backward");
}

}  // namespace

int layernorm(void* res, const void* x, const void* w, const void* b, void* y, void* q, void* s, void* mean, void* rstd,
              int M, int K, float eps, cudaStream_t st) {
    NormArgs p;
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.res = static_cast<__nv_bfloat16*>(res);
    p.w = static_cast<const __nv_bfloat16*>(w);
    p.b = static_cast<const __nv_bfloat16*>(b);
    p.y = static_cast<__nv_bfloat16*>(y);
    p.q = static_cast<int8_t*>(q);
    p.s = static_cast<float*>(s);
    p.mean = static_cast<float*>(mean);
    p.rstd = static_cast<float*>(rstd);
    p.M = M; p.K = K; p.T = 0; p.eps = eps;
    if (q != nullptr) return res != nullptr ? dispatch_norm<true, true>(p, st) : dispatch_norm<false, true>(p, st);
    return res != nullptr ? dispatch_norm<true, false>(p, st) : dispatch_norm<false, false>(p, st);
}

int64_t layernorm_backward_workspace(int M, int K) { return (int64_t)min(M, kMaxParts) * 2 * K * 4; }

int layernorm_backward(const void* dy, const void* x, const void* mean, const void* rstd, const void* w, const void* dres,
                       void* dx, void* dw, void* db, void* workspace, int M, int K, cudaStream_t st) {
    const int parts = min(sm_count(), kMaxParts);
    if (parts <= 0) return fail(DSV4_ERR_LAUNCH, "layernorm_backward: no CUDA device");
    NormBwdArgs p;
    p.dy = static_cast<const __nv_bfloat16*>(dy);
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.mean = static_cast<const float*>(mean);
    p.rstd = static_cast<const float*>(rstd);
    p.w = static_cast<const __nv_bfloat16*>(w);
    p.dres = static_cast<const __nv_bfloat16*>(dres);
    p.dx = static_cast<__nv_bfloat16*>(dx);
    p.partial = static_cast<float*>(workspace);
    p.M = M; p.K = K; p.T = 0;
    float *dwf = static_cast<float*>(dw), *dbf = static_cast<float*>(db);
    return dres != nullptr ? dispatch_norm_backward<true>(p, dwf, dbf, parts, st)
                           : dispatch_norm_backward<false>(p, dwf, dbf, parts, st);
}

}  // namespace w8a8
