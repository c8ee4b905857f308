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
// with a large mean.  All statistics and sums are fp32, in an order that sizes, device and the arrays' alignment decide: the
// width of the accesses decides which columns a thread adds up.
//
// Everything here is bound by HBM.  A row belongs to a group of G threads and is read once.
//   * Forward: a row per group, straight from HBM, several CTAs per SM.
//   * Backward: one CTA per SM, so that every thread can keep the column sums of its columns in registers; its groups
//     walk the rows, and the next rows are on their way into shared memory (cp.async) while two are worked on.  Rows whose
//     width or address does not allow 16-byte accesses come in as the 16-byte granules that cover them and are taken apart
//     in shared memory (2-byte accesses to HBM took 1270 us for 8192 x 7165, the granules 191 us).
//   * Rows wider than 16384 are read again for each reduction (the *_wide kernels).
// Arithmetic is on pairs (packed f32x2): the backward pass was otherwise bound by its instructions.
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
// larger magnitude; a NaN stays one and becomes the row's scale (codes alone would turn it into a number)
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float top_of(float t, float a) { return max_nan(t, fabsf(a)); }
__device__ __forceinline__ float top_of(float t, float2 a) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(t), "f"(fabsf(a.x)), "f"(fabsf(a.y)));
    return d;
}
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
    float2* red;       // [2][64] of this group, 16-byte aligned (not used by a group of one warp)
    int threads;       // multiple of 32
    int id;            // hardware barrier of the group: 1 + index in the CTA
    int turn = 0;
    __device__ __forceinline__ void barrier() const { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
    template <typename T, typename Op>
    __device__ __forceinline__ T reduce(T v, Op op) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = op(v, shuffle(v, o));
        if (threads == 32) return v;
        const int lane = threadIdx.x & 31, warp = (threadIdx.x % threads) >> 5, warps = threads >> 5;
        T* slot = reinterpret_cast<T*>(red + 64 * turn);
        turn ^= 1;
        if (lane == 0) slot[warp] = v;
        barrier();
        v = slot[lane < warps ? lane : 0];
        if (lane >= warps) v = T{};   // neutral for sums, and for maxima of magnitudes
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = op(v, shuffle(v, o));
        return v;
    }
    static __device__ __forceinline__ float shuffle(float v, int o) { return __shfl_xor_sync(kFullWarp, v, o); }
    static __device__ __forceinline__ float2 shuffle(float2 v, int o) { return make_float2(shuffle(v.x, o), shuffle(v.y, o)); }
    __device__ __forceinline__ float2 sum2(float2 v) {
        return reduce(v, [](float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); });
    }
    __device__ __forceinline__ float sum(float v) {
        return reduce(v, [](float a, float b) { return a + b; });
    }
    __device__ __forceinline__ float max(float v) {
        return reduce(v, [](float a, float b) { return max_nan(a, b); });
    }
    // Four sums at once: halves of the warp keep two of the values each, quarters one, so that thirteen shuffles do what
    // forty would.  Entries of warps that the group does not have must be zero (clear4).
    __device__ __forceinline__ void clear4() {
        const int i = threadIdx.x % threads;
        if (threads > 32) {
            for (int k = i; k < 256; k += threads) reinterpret_cast<float*>(red)[k] = 0.0f;
            barrier();
        }
    }
    __device__ __forceinline__ float4 sum4(float4 v) {
        const int lane = threadIdx.x & 31;
        const bool up16 = lane & 16, up8 = lane & 8;
        float a = up16 ? v.z : v.x, b = up16 ? v.w : v.y;
        a += shuffle(up16 ? v.x : v.z, 16);
        b += shuffle(up16 ? v.y : v.w, 16);
        float k = up8 ? b : a;
        k += shuffle(up8 ? a : b, 8);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) k += shuffle(k, o);
        if (threads > 32) {
            // value (lane / 8) of warp w at [lane / 8][w]; the two turns use 128 floats each
            float* slot = reinterpret_cast<float*>(red) + 128 * turn;
            turn ^= 1;
            if ((lane & 7) == 0) slot[(lane >> 3) * 32 + ((threadIdx.x % threads) >> 5)] = k;
            barrier();
            const float4 q = *reinterpret_cast<const float4*>(slot + (lane >> 3) * 32 + (lane & 7) * 4);
            k = (q.x + q.y) + (q.z + q.w);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) k += shuffle(k, o);
        }
        return make_float4(__shfl_sync(kFullWarp, k, 0), __shfl_sync(kFullWarp, k, 8), __shfl_sync(kFullWarp, k, 16),
                           __shfl_sync(kFullWarp, k, 24));
    }
    // everything that the group's threads wrote to shared memory is visible to all of them
    __device__ __forceinline__ void sync() const {
        if (threads == 32) __syncwarp();
        else barrier();
    }
};

// ---- rows on their way through shared memory -------------------------------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// One array's rows, `depth` of them in shared memory.  W = 8: thread t owns accesses t, t + G, ... of a row and copies
// exactly those, so what it waits for is its own.  W < 8: the group copies the 16-byte granules that cover the row
// (element by element where a granule leaves the array) to the same offset modulo 16, and meets before it reads them.  Results go straight to HBM, an access of W per lane.
template <int W, int V>
struct RowStage {
    char* base;          // this array's slots in the group's shared memory
    const char* array;   // [M, K] bf16
    int64_t bytes;       // of the array
    int slot_bytes;
    int K, G, t;
    __device__ __forceinline__ const char* row_ptr(int64_t row) const { return array + row * K * 2; }
    __device__ __forceinline__ void issue(int slot, int64_t row) const {
        char* s = base + slot * slot_bytes;
        const char* src = row_ptr(row);
        if constexpr (W == 8) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int a = t + j * G;
                if (a * 8 < K) cp_async16(ptx::smem_u32(s + a * 16), src + a * 16);
            }
        } else {
            const int skew = (int)(reinterpret_cast<uintptr_t>(src) & 15);
            const char* first = src - skew;
            const int granules = (skew + 2 * K + 15) >> 4;
#pragma unroll 1
            for (int i = t; i < granules; i += G) {
                const char* g = first + 16 * i;
                if (g >= array && g + 16 <= array + bytes) {
                    cp_async16(ptx::smem_u32(s + 16 * i), g);
                } else {
#pragma unroll 1
                    for (int b = 0; b < 16; b += 2)
                        if (g + b >= src && g + b < src + 2 * K)
                            *reinterpret_cast<uint16_t*>(s + 16 * i + b) = *reinterpret_cast<const uint16_t*>(g + b);
                }
            }
        }
    }
    // where this thread's accesses of a row that has arrived begin, and access j of them
    __device__ __forceinline__ const char* row(int slot, int64_t r) const {
        const char* s = base + slot * slot_bytes + t * W * 2;
        if constexpr (W != 8) s += reinterpret_cast<uintptr_t>(row_ptr(r)) & 15;
        return s;
    }
    __device__ __forceinline__ Pack<W> at(const char* row, int j) const {
        return load_pack<W>(reinterpret_cast<const __nv_bfloat16*>(row + j * G * W * 2));
    }
};

// int8 codes of W values
template <int W, int N, typename T>
__device__ __forceinline__ void store_codes(int8_t* q, const T (&y)[N], float inv) {
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

__device__ __forceinline__ void scale_of(float top, float& scale, float& inv) {
    scale_from_amax(top, scale, inv);
    if (isnan(top)) scale = top;
}

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
    int M, K, T;               // T: threads of a group
    float eps;
};

// Eight consecutive elements of an array whose base is 16-byte aligned, from any column c on: the two 16-byte words that hold
// them, shifted; by elements where the second would reach past the array's K elements.
__device__ __forceinline__ Pack<8> load_shifted(const __nv_bfloat16* w, int c, int K) {
    Pack<8> o;
    const int s = c & 7;
    if (c - s + 16 <= K) {
        const Pack<8> lo = load_pack<8>(w + c - s), hi = load_pack<8>(w + c - s + 8);
        uint32_t v[8] = {lo.w[0], lo.w[1], lo.w[2], lo.w[3], hi.w[0], hi.w[1], hi.w[2], hi.w[3]};
#pragma unroll
        for (int j = 0; j < 6; ++j) v[j] = s & 4 ? v[j + 2] : v[j];
#pragma unroll
        for (int j = 0; j < 5; ++j) v[j] = s & 2 ? v[j + 1] : v[j];
#pragma unroll
        for (int j = 0; j < 4; ++j) o.w[j] = __funnelshift_r(v[j], v[j + 1], (s & 1) * 16);
    } else {
        const uint16_t* e = reinterpret_cast<const uint16_t*>(w + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) o.w[j] = e[2 * j] | ((uint32_t)e[2 * j + 1] << 16);
    }
    return o;
}

// ---- forward: blockDim = R groups of G threads, one row per group, V accesses of W elements per thread ---------------
// The row stays packed (four registers per eight elements) and is widened again for each pass; the row's pointers are
// formed once (inside the access loops every access had a 64-bit product of its own, and spilled).  8192 x 7168 with the
// residual: 98 us with spills, 76-82 us without, 72 us at the measured copy rate.
//
// SHIFT (W = 8): rows at any offset of the 16 bytes, the same in every array.  The 16-byte words that lie inside the row go
// the ordinary way, from the row's first aligned column on, weight and bias shifted to them; the up to seven elements on
// either side are the business of one thread each.  8192 x 7165 with the residual: 267 us by elements,
// 102 us this way; 8192 x 15157 917 and 283 us.
template <int W, int V, int THREADS, int CTAS, bool ADD, bool QUANT, bool SHIFT = false>
__global__ void __launch_bounds__(THREADS, CTAS) layernorm_kernel(const NormArgs p) {
    static_assert(!SHIFT || W == 8, "16-byte words");
    using T = typename Vals<W>::T;
    constexpr int N = Vals<W>::kN;
    __shared__ __align__(16) float2 red_all[8 * 128];   // a CTA holds at most eight groups
    ptx::grid_launch_dependents();  // a GEMM launched to overlap this kernel may start its set-up and weight loads
    const int G = p.T, g = threadIdx.x / G, t = threadIdx.x - g * G;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / G) + g;
    if (row >= p.M) return;  // whole groups: nobody is left waiting at the group's barrier
    Group grp{red_all + 128 * g, G, 1 + g};
    // columns [c0, c0 + K) in accesses of W
    const int c0 = SHIFT ? min(p.K, (int)(-(reinterpret_cast<intptr_t>(p.x + row * p.K) >> 1) & 7)) : 0;
    const int K = SHIFT ? (p.K - c0) & ~7 : p.K;
    const __nv_bfloat16* x = p.x + row * p.K + c0;
    __nv_bfloat16* res_row = p.res + row * p.K + c0;
    __nv_bfloat16* y_row = p.y + row * p.K + c0;
    int8_t* q_row = p.q + row * p.K + c0;
    // SHIFT: this thread's single element, as an offset from c0: the head's for threads 0..7, the tail's for 8..15
    const int single = t < 8 ? t - c0 : K + t - 8;
    const bool has_single = SHIFT && (t < 8 ? t < c0 : t < 16 && c0 + single < p.K);
    float one = 0.0f;
    Pack<W> a[V];
    Pack<W> w1, b1;                      // a thread with one access has its weight and bias requested with the row
    auto weights_of = [&](const __nv_bfloat16* w, int c) -> Pack<W> {
        if constexpr (SHIFT) return load_shifted(w, c0 + c, p.K);
        else return load_pack<W>(w + c);
    };
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (t + j * G) * W;
        if (c < K) {
            a[j] = load_pack<W>(x + c);
            if constexpr (V == 1) {
                w1 = weights_of(p.w, c);
                b1 = weights_of(p.b, c);
            }
        }
    }
    if (has_single) one = __bfloat162float(x[single]);
    T acc = all<T>(0.0f);
    if constexpr (ADD) {
        Pack<W> r[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (t + j * G) * W;
            if (c < K) r[j] = load_pack<W>(res_row + c);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (t + j * G) * W;
            if (c < K) {
#pragma unroll
                for (int i = 0; i < N; ++i) a[j].w[i] = rounded(add(value<W>(r[j], i), value<W>(a[j], i)));
                store_pack<W>(res_row + c, a[j]);
            }
        }
        if (has_single) {
            const __nv_bfloat16 sum = __float2bfloat16_rn(add(__bfloat162float(res_row[single]), one));
            res_row[single] = sum;
            one = __bfloat162float(sum);
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if ((t + j * G) * W < K) {
#pragma unroll
            for (int i = 0; i < N; ++i) acc = add(acc, value<W>(a[j], i));
        }
    }
    float part = total(acc);
    if (SHIFT) part = add(part, one);
    const float mean = __fdiv_rn(grp.sum(part), (float)p.K);
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
    part = total(acc);
    if (has_single) part = fma(add(one, -mean), add(one, -mean), part);
    const float rstd = rstd_of(grp.sum(part), p.K, p.eps);
    if (t == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
    if (has_single) {
        const int c = c0 + single;
        one = fma(mul(add(one, -mean), rstd), __bfloat162float(p.w[c]), __bfloat162float(p.b[c]));   // y from here on
    }
    // y of access j; the quantiser evaluates it twice (largest magnitude, codes) rather than hold it
    auto y_of = [&](int j, int c, T (&y)[N]) {
        const Pack<W> w = V == 1 ? w1 : weights_of(p.w, c), b = V == 1 ? b1 : weights_of(p.b, c);
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
                store_pack<W>(y_row + c, o);
            }
        }
        if (has_single) y_row[single] = __float2bfloat16_rn(one);
    } else {
        float top = has_single ? fabsf(one) : 0.0f;
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
        scale_of(grp.max(top), scale, inv);
        if (t == 0) p.s[row] = scale;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (t + j * G) * W;
            if (c < K) {
                T y[N];
                y_of(j, c, y);
                store_codes<W>(q_row + c, y, inv);
            }
        }
        if (has_single) q_row[single] = (int8_t)quant_rn(one, inv);
    }
}

// rows wider than the registers hold: one CTA per row, every reduction reads the row again (it stays in L1 / L2)
template <bool ADD, bool QUANT>
__global__ void __launch_bounds__(kMaxGroupThreads) layernorm_wide_kernel(const NormArgs p) {
    __shared__ __align__(16) float2 red_all[128];
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
        for (int c = threadIdx.x; c < K; c += T) top = top_of(top, norm(c));
        scale_of(grp.max(top), scale, inv);
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
    float* partial;              // [gridDim.x][2][K]: this CTA's share of dw and db; 16-byte aligned
    int M, K, T;
    int slot_bytes;
};

// ---- backward: every thread keeps the sums of its own columns in registers over all the rows that its group walks ----
// B rows (1 or 2) at a time: one barrier for both, and two rows' work to hide each other's latencies.  One row at a time
// stood at its barriers (8192 x 7168: 172 us with eight columns per thread and one group of 896 threads, 138 us with 16 and
// two groups, which spilled).  Two rows, 16 columns per thread and 448 threads with 128 registers each: 79 us, of which 4.5
// are the sum of the CTAs' shares; 72 us at the measured copy rate.  Eight columns and 896 threads take 85 to 111 us, with
// the compiler's luck; rows in pieces of two or one elements are better off with them (7165: 191 against 219 us).
template <int W, int V, int B, int DEPTH, int THREADS, bool RES>
__global__ void __launch_bounds__(THREADS, 1) layernorm_backward_kernel(const NormBwdArgs p) {
    using T = typename Vals<W>::T;
    constexpr int N = Vals<W>::kN, kArrays = RES ? 3 : 2;
    __shared__ __align__(16) float2 red_all[15 * 128];
    extern __shared__ __align__(16) char rows_smem[];   // the groups' row slots; at the end their column sums
    ptx::grid_launch_dependents();   // the column sums' kernel
    const int G = p.T, R = blockDim.x / G, g = threadIdx.x / G, t = threadIdx.x - g * G, K = p.K;
    Group grp{red_all + (G == 32 ? 0 : 128 * g), G, 1 + g};
    char* mine = rows_smem + (size_t)g * DEPTH * B * kArrays * p.slot_bytes;
    const int64_t bytes = (int64_t)p.M * K * 2;
    const RowStage<W, V> xs{mine, reinterpret_cast<const char*>(p.x), bytes, p.slot_bytes, K, G, t};
    const RowStage<W, V> ys{mine + DEPTH * B * p.slot_bytes, reinterpret_cast<const char*>(p.dy), bytes, p.slot_bytes, K, G, t};
    const RowStage<W, V> rs{mine + 2 * DEPTH * B * p.slot_bytes, reinterpret_cast<const char*>(p.dres), bytes, p.slot_bytes, K, G, t};
    const float inv_k = __fdiv_rn(1.0f, (float)K);
    if constexpr (B == 2) grp.clear4();
    T dw[V][N], db[V][N];
    Pack<W> w[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int i = 0; i < N; ++i) dw[j][i] = db[j][i] = all<T>(0.0f);
        if ((t + j * G) * W < K) w[j] = load_pack<W>(p.w + (t + j * G) * W);
    }
    const int64_t step = (int64_t)gridDim.x * R * B;
    auto issue = [&](int stage, int64_t first) {
#pragma unroll
        for (int b = 0; b < B; ++b) {
            if (first + b < p.M) {
                xs.issue(stage * B + b, first + b);
                ys.issue(stage * B + b, first + b);
                if constexpr (RES) rs.issue(stage * B + b, first + b);
            }
        }
        cp_async_commit();   // empty past the last row: the count of groups stays in step
    };
    float mean[B], rstd[B], next_mean[B], next_rstd[B];
    auto statistics = [&](int64_t first) {
#pragma unroll
        for (int b = 0; b < B; ++b) {
            next_mean[b] = first + b < p.M ? __ldg(p.mean + first + b) : 0.0f;
            next_rstd[b] = first + b < p.M ? __ldg(p.rstd + first + b) : 0.0f;
        }
    };
    int64_t row = ((int64_t)blockIdx.x * R + g) * B;
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) issue(d, row + d * step);
    statistics(row);
    int stage = 0;
    for (; row < p.M; row += step) {
        cp_async_wait<DEPTH - 2>();
        if constexpr (W != 8) grp.sync();
        // the stage of the rows before: its last readers are behind the barrier above, or are this thread (W = 8)
        issue(stage == 0 ? DEPTH - 1 : stage - 1, row + (DEPTH - 1) * step);
#pragma unroll
        for (int b = 0; b < B; ++b) {
            mean[b] = next_mean[b];
            rstd[b] = next_rstd[b];
        }
        statistics(row + step);
        float c[B][2];   // sums of t = dy * w and of t * xhat
#pragma unroll
        for (int b = 0; b < B; ++b) {
            T c0 = all<T>(0.0f), c1 = all<T>(0.0f);
            if (row + b < p.M) {
                const char* xp = xs.row(stage * B + b, row + b);
                const char* yp = ys.row(stage * B + b, row + b);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if ((t + j * G) * W < K) {
                        const Pack<W> px = xs.at(xp, j), py = ys.at(yp, j);
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            const T y = value<W>(py, i), u = mul(y, value<W>(w[j], i));
                            const T h = mul(add(value<W>(px, i), all<T>(-mean[b])), all<T>(rstd[b]));
                            dw[j][i] = fma(y, h, dw[j][i]);
                            db[j][i] = add(db[j][i], y);
                            c0 = add(c0, u);
                            c1 = fma(u, h, c1);
                        }
                    }
                }
            }
            c[b][0] = total(c0);
            c[b][1] = total(c1);
        }
        if constexpr (B == 2) {
            const float4 q = grp.sum4(make_float4(c[0][0], c[0][1], c[B - 1][0], c[B - 1][1]));
            c[0][0] = q.x; c[0][1] = q.y; c[B - 1][0] = q.z; c[B - 1][1] = q.w;
        } else {
            const float2 q = grp.sum2(make_float2(c[0][0], c[0][1]));
            c[0][0] = q.x; c[0][1] = q.y;
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            if (row + b >= p.M) break;
            const float m0 = -c[b][0] * inv_k, m1 = -c[b][1] * inv_k;
            __nv_bfloat16* dst = p.dx + (row + b) * K;   // outside the access loop, as the pointers below: no spills
            const char* xp = xs.row(stage * B + b, row + b);
            const char* yp = ys.row(stage * B + b, row + b);
            const char* rp = RES ? rs.row(stage * B + b, row + b) : nullptr;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int col = (t + j * G) * W;
                if (col < K) {
                    // read again: cheaper than xhat and t in registers
                    const Pack<W> px = xs.at(xp, j), py = ys.at(yp, j);
                    Pack<W> o, r;
                    if constexpr (RES) r = rs.at(rp, j);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const T h = mul(add(value<W>(px, i), all<T>(-mean[b])), all<T>(rstd[b]));
                        const T d = fma(h, all<T>(m1), fma(value<W>(py, i), value<W>(w[j], i), all<T>(m0)));
                        if constexpr (RES) o.w[i] = rounded(fma(d, all<T>(rstd[b]), value<W>(r, i)));
                        else o.w[i] = rounded(mul(d, all<T>(rstd[b])));
                    }
                    store_pack<W>(dst + col, o);
                }
            }
        }
        if (++stage == DEPTH) stage = 0;
    }
    cp_async_wait<0>();
    // column sums of the CTA's groups, added in the groups' order
    float* out = p.partial + (int64_t)blockIdx.x * 2 * K;
    float* cols = reinterpret_cast<float*>(rows_smem);   // [R][2][K]
    if (R > 1) __syncthreads();
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
                } else {   // c, K and the partial's alignment allow 8 bytes
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
    __shared__ __align__(16) float2 red_all[128];
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
    ptx::grid_dependency_wait();   // may have started while the CTAs still write their shares
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
    float v = 0.0f;
    if (col < 2 * K) {
#pragma unroll 8
        for (int i = slice; i < parts; i += 8) v += __ldcg(partial + (int64_t)i * 2 * K + col);
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
// threads per row (multiple of 32) when each thread makes at most `v` accesses
int group_threads(int accesses, int v) { return ((accesses + v - 1) / v + 31) / 32 * 32; }

// Widest access that the row length and every address allow
template <typename... P>
int access_width(int K, const P*... ptrs) {
    const uintptr_t bits = (... | reinterpret_cast<uintptr_t>(ptrs));
    return K % 8 == 0 && bits % 16 == 0 ? 8 : K % 2 == 0 && bits % 4 == 0 ? 2 : 1;
}

template <int W, int V, int THREADS, int CTAS, bool ADD, bool QUANT, bool SHIFT = false>
int launch_norm(NormArgs p, cudaStream_t st) {
    p.T = group_threads((p.K + W - 1) / W, V);
    // narrow rows share a CTA of up to 256 threads: one row each, at most 8 rows
    const int R = p.T >= 256 ? 1 : 256 / p.T;
    layernorm_kernel<W, V, THREADS, CTAS, ADD, QUANT, SHIFT><<<(unsigned)(((int64_t)p.M + R - 1) / R), R * p.T, 0, st>>>(p);
    return check_launch("layernorm");
}

// Groups per CTA and shared memory of the kernel that walks rows
struct RowsShape {
    int G, R, slot_bytes, smem;
};
constexpr int kRowsSmem = 200 * 1024;
template <int W, int V, int DEPTH>
RowsShape rows_shape(int K, int arrays, int threads, int column_floats) {
    RowsShape s;
    s.G = group_threads((K + W - 1) / W, V);
    // W = 8: whole accesses; otherwise the granules that cover a row at any offset
    s.slot_bytes = W == 8 ? K * 2 : (2 * K + 30 + 15) / 16 * 16;
    s.R = s.G == 32 ? threads / 32 : min(15, threads / s.G);   // hardware barriers 1..15; a one-warp group needs none
    const int per_group = max(DEPTH * arrays * s.slot_bytes, column_floats * 4);
    s.R = max(1, min(s.R, kRowsSmem / per_group));
    s.smem = s.R * per_group;
    return s;
}
// Whether a row begins at the same offset of the 16 bytes in all arrays (the codes': of 8 bytes), and weight and bias at 0
template <bool ADD, bool QUANT>
bool same_offset(const NormArgs& p) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p.x), wb = reinterpret_cast<uintptr_t>(p.w) | reinterpret_cast<uintptr_t>(p.b);
    auto differs = [&](const void* q) { return ((x ^ reinterpret_cast<uintptr_t>(q)) & 15) != 0; };
    if ((wb & 15) || (ADD && differs(p.res))) return false;
    return QUANT ? (((x >> 1) ^ reinterpret_cast<uintptr_t>(p.q)) & 7) == 0 : !differs(p.y);
}

// Few rows (no more than two per SM, or 6144 elements per SM) take one wide access per thread, for latency (8 x 7168 with
// the quantiser: 7.3 us with four accesses, 4 us with one; 600 x 1000: 4.2 and 3.6 us); more rows take four (8192 x 7168 with
// the residual: 121 us with one, 83-99 with two, 76-82 with four; 2000 x 1000: 5.9 us with one, 4.9 with four).
template <bool ADD, bool QUANT>
int dispatch_norm(const NormArgs& p, cudaStream_t st) {
    int w = access_width(p.K, p.x, p.w, p.b, (const __nv_bfloat16*)p.res, (const __nv_bfloat16*)p.y);
    if (QUANT && w == 8 && (reinterpret_cast<uintptr_t>(p.q) & 7)) w = 2;
    if (QUANT && w == 2 && (reinterpret_cast<uintptr_t>(p.q) & 1)) w = 1;
    const int sms = sm_count();
    const bool few = p.M <= 2 * sms || (int64_t)p.M * p.K <= (int64_t)6144 * sms;
    if (w == 8) {
        if (p.K <= 8192 && few) return launch_norm<8, 1, 1024, 1, ADD, QUANT>(p, st);
        if (p.K <= 16384) return launch_norm<8, 4, 512, 2, ADD, QUANT>(p, st);
    } else if (p.K >= 64 && p.K <= 16384 && same_offset<ADD, QUANT>(p)) {
        if (p.K <= 8192 && few) return launch_norm<8, 1, 1024, 1, ADD, QUANT, true>(p, st);
        return launch_norm<8, 4, 512, 1, ADD, QUANT, true>(p, st);
    } else if (w == 2) {
        if (p.K <= 8192) return launch_norm<2, 4, 1024, 1, ADD, QUANT>(p, st);
        if (p.K <= 16384) return launch_norm<2, 8, 1024, 1, ADD, QUANT>(p, st);
    } else {
        if (p.K <= 4096) return launch_norm<1, 4, 1024, 1, ADD, QUANT>(p, st);
        if (p.K <= 8192) return launch_norm<1, 8, 1024, 1, ADD, QUANT>(p, st);
        if (p.K <= 16384) return launch_norm<1, 16, 1024, 1, ADD, QUANT>(p, st);
    }
    layernorm_wide_kernel<ADD, QUANT><<<p.M, kMaxGroupThreads, 0, st>>>(p);
    return check_launch("layernorm");
}

constexpr int kWideParts = 64;
// Most CTAs whose column sums the workspace has room for; a launch uses one per SM (148 on a B200).
constexpr int kMaxParts = 160;

template <int W, int V, int B, int DEPTH, int THREADS, bool RES>
int launch_norm_backward(NormBwdArgs p, float* dw, float* db, int parts, cudaStream_t st) {
    static bool opted_in[64] = {};
    if (!opt_in_shared_memory(layernorm_backward_kernel<W, V, B, DEPTH, THREADS, RES>, kRowsSmem, opted_in))
        return fail(DSV4_ERR_LAUNCH, "layernorm_backward: cannot raise the dynamic shared memory limit");
    RowsShape s = rows_shape<W, V, DEPTH * B>(p.K, RES ? 3 : 2, THREADS, 2 * p.K);
    p.T = s.G;
    p.slot_bytes = s.slot_bytes;
    // few rows: rather one group on every SM than several on some
    const int want = (int)max((int64_t)1, ((int64_t)p.M + (int64_t)parts * B - 1) / ((int64_t)parts * B));
    if (s.R > want) {
        s.smem = s.smem / s.R * want;
        s.R = want;
    }
    const int grid = (int)min((int64_t)parts, ((int64_t)p.M + s.R * B - 1) / (s.R * B));
    layernorm_backward_kernel<W, V, B, DEPTH, THREADS, RES><<<grid, s.R * s.G, s.smem, st>>>(p);
    if (int rc = check_launch("layernorm_backward")) return rc;
    return launch_after(layernorm_column_sum_kernel, dim3((2 * p.K + 31) / 32), dim3(256), 0, st, "layernorm_backward", p.partial, grid,
                        p.K, dw, db);
}

template <bool RES>
int dispatch_norm_backward(const NormBwdArgs& p, float* dw, float* db, int parts, cudaStream_t st) {
    const int w = access_width(p.K, p.x, p.dy, p.w, (const __nv_bfloat16*)p.dx, p.dres);
    if (w == 8) {
        if (p.K <= 8192) return launch_norm_backward<8, 2, 2, 2, 512, RES>(p, dw, db, parts, st);
        if (p.K <= 16384) return launch_norm_backward<8, 4, 1, 2, 512, RES>(p, dw, db, parts, st);
    } else if (w == 2) {
        if (p.K <= 7168) return launch_norm_backward<2, 4, 2, 2, 896, RES>(p, dw, db, parts, st);
        if (p.K <= 8192) return launch_norm_backward<2, 4, 2, 2, 1024, RES>(p, dw, db, parts, st);
        if (p.K <= 16384) return launch_norm_backward<2, 16, 1, 2, 512, RES>(p, dw, db, parts, st);
    } else {
        if (p.K <= 7168) return launch_norm_backward<1, 8, 2, 2, 896, RES>(p, dw, db, parts, st);
        if (p.K <= 8192) return launch_norm_backward<1, 8, 2, 2, 1024, RES>(p, dw, db, parts, st);
        if (p.K <= 16384) return launch_norm_backward<1, 32, 1, 2, 512, RES>(p, dw, db, parts, st);
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
    p.M = M; p.K = K; p.T = 0; p.slot_bytes = 0;
    float *dwf = static_cast<float*>(dw), *dbf = static_cast<float*>(db);
    return dres != nullptr ? dispatch_norm_backward<true>(p, dwf, dbf, parts, st)
                           : dispatch_norm_backward<false>(p, dwf, dbf, parts, st);
}

}  // namespace w8a8
