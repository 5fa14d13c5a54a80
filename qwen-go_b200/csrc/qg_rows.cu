// Tokens in expert order, as operators of their own: the pairs (token, rank)
// that a router selected sorted by expert, the token rows gathered in that
// order, the expert rows weighted and summed back per token, and the
// gradients of both; and the per-token int8 quantiser, which can gather while
// it quantises.  The sum over a token's ranks is the expert loop's
// `out[j] += w * d[j]` of model/moe.go:82-85, in rank order.
//
// With pairs p = t*k + j, e_p = sel_idx[p] and p valid iff 0 <= e_p < E:
//   offsets[e]  = #{p valid : e_p < e}
//   pair_row[p] = offsets[e_p] + #{q < p : e_q = e_p}, -1 for an invalid p
//   gather      rows[pair_row[p]] = x[t]
//     backward  dx[t] = sum_j drows[pair_row[t, j]]
//   combine     out[t] = sum_j w[t, j] rows[pair_row[t, j]]
//     backward  drows[pair_row[p]] = w[p] dout[t];  dw[p] = <rows[pair_row[p]], dout[t]>
// Every kernel is organised by token, so that a token's row is read once for
// its k expert rows, and rows that no pair owns are never touched.  A
// pair_row outside [0, T*k) counts as a pair without a row.
#include <cuda_bf16.h>
#include <float.h>
#include <math_constants.h>

#include "qg_common.cuh"

namespace qg {

// ---- row elements ---------------------------------------------------------
// Rows are read with plain (coherent) loads: with programmatic dependent
// launch the previous kernel may still be writing them when this one starts,
// which the read-only path does not allow.
__device__ __forceinline__ uint4 ld16(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p)
                 : "memory");
    return v;
}
__device__ __forceinline__ int ld_i32(const int32_t *p) {
    int v;
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float ld_f32(const float *p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}

template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ float load(const float *p) { return ld_f32(p); }
    static __device__ __forceinline__ void store(float *p, float v) { *p = v; }
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ float load(const __half *p) {
        unsigned short u;
        asm volatile("ld.global.u16 %0, [%1];" : "=h"(u) : "l"(p) : "memory");
        return __half2float(__ushort_as_half(u));
    }
    static __device__ __forceinline__ void store(__half *p, float v) { *p = __float2half_rn(v); }
};
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float load(const __nv_bfloat16 *p) {
        unsigned short u;
        asm volatile("ld.global.u16 %0, [%1];" : "=h"(u) : "l"(p) : "memory");
        return __uint_as_float((uint32_t)u << 16);
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, float v) {
        *p = __float2bfloat16_rn(v);
    }
};

// Eight consecutive elements, 16-byte aligned; raw as loaded, so that several
// can be in flight before the first is widened.
template <typename T> struct Vec8 {  // 16-bit types: one 16-byte load
    uint4 r;
    __device__ __forceinline__ void load(const T *p) { r = ld16(p); }
    __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float2 f;
            if constexpr (sizeof(T) == 2 && __is_same(T, __half))
                f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            else
                f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void put(T *p, const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (__is_same(T, __half)) {
                __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<uint32_t *>(&h);
            } else {
                __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<uint32_t *>(&h);
            }
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Vec8<float> {  // two 16-byte loads
    uint4 a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = ld16(p);
        b = ld16(p + 4);
    }
    __device__ __forceinline__ void zero() { a = b = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y);
        v[2] = __uint_as_float(a.z), v[3] = __uint_as_float(a.w);
        v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y);
        v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
    }
    static __device__ __forceinline__ void put(float *p, const float (&v)[8]) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
};

// ---- sort -------------------------------------------------------------------
// One CTA per expert e: it reads every pair's expert once to count the pairs
// before its range (e_p < e) and its own, and once more to give its own their
// rows.  No workspace, no atomics, one launch; the order within an expert is
// the pairs' own.  Each warp owns a contiguous range of pairs, so that its
// rows follow those of the warps below it.
constexpr int SORT_MAX_WARPS = 32;

struct Ids4 {
    int v[4];
};
__device__ __forceinline__ Ids4 load_ids(const int32_t *ids, int64_t i, int64_t hi, bool vec) {
    Ids4 r;
    if (vec && i + 4 <= hi) {
        uint4 u;
        asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                     : "l"(ids + i)
                     : "memory");
        r.v[0] = (int)u.x, r.v[1] = (int)u.y, r.v[2] = (int)u.z, r.v[3] = (int)u.w;
    } else {
#pragma unroll
        for (int s = 0; s < 4; s++) r.v[s] = i + s < hi ? ld_i32(ids + i + s) : -1;
    }
    return r;
}

__global__ void k_sort_tokens(const int32_t *ids, int N, int E, int32_t *offsets,
                              int32_t *pair_row, int32_t *row_pair) {
    __shared__ int s_less[SORT_MAX_WARPS], s_eq[SORT_MAX_WARPS], s_valid[SORT_MAX_WARPS];
    pdl_enter();
    const int e = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nw = blockDim.x >> 5;
    const bool vec = (reinterpret_cast<uintptr_t>(ids) & 15) == 0;
    int64_t per = ((int64_t)N + nw - 1) / nw;
    per = (per + 127) & ~int64_t(127);
    const int64_t lo = per * warp, hi = min((int64_t)N, lo + per);
    int less = 0, eq = 0, valid = 0;
    for (int64_t i = lo + lane * 4; i < hi; i += 128) {
        const Ids4 d = load_ids(ids, i, hi, vec);
#pragma unroll
        for (int s = 0; s < 4; s++) {
            less += (unsigned)d.v[s] < (unsigned)e;
            eq += d.v[s] == e;
            valid += (unsigned)d.v[s] < (unsigned)E;
        }
    }
    less = __reduce_add_sync(~0u, less);
    eq = __reduce_add_sync(~0u, eq);
    valid = __reduce_add_sync(~0u, valid);
    if (lane == 0) {
        s_less[warp] = less;
        s_eq[warp] = eq;
        s_valid[warp] = valid;
    }
    __syncthreads();
    const int l = lane < nw ? s_less[lane] : 0;
    const int q = lane < nw ? s_eq[lane] : 0;
    const int start = __reduce_add_sync(~0u, l);
    const int mine = __reduce_add_sync(~0u, q);
    int row = start + __reduce_add_sync(~0u, lane < warp ? q : 0);
    if (threadIdx.x == 0) {
        offsets[e] = start;
        if (e == E - 1) offsets[E] = start + mine;
    }
    const unsigned below = (1u << lane) - 1;
    for (int64_t i0 = lo; i0 < hi; i0 += 128) {
        const int64_t i = i0 + lane * 4;
        Ids4 d;
        if (i < hi) {
            d = load_ids(ids, i, hi, vec);
        } else {
            d.v[0] = d.v[1] = d.v[2] = d.v[3] = -1;
        }
        if (e == 0) {  // pairs without an expert
#pragma unroll
            for (int s = 0; s < 4; s++)
                if (i + s < hi && (unsigned)d.v[s] >= (unsigned)E) pair_row[i + s] = -1;
        }
        unsigned m[4];
        int before = 0, all = 0;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            m[s] = __ballot_sync(~0u, d.v[s] == e);
            before += __popc(m[s] & below);
            all += __popc(m[s]);
        }
        int r = row + before;
#pragma unroll
        for (int s = 0; s < 4; s++)
            if (d.v[s] == e) {
                pair_row[i + s] = r;
                if (row_pair) row_pair[r] = (int)(i + s);
                r++;
            }
        row += all;
    }
    if (e == 0 && row_pair) {  // rows without a pair
        int total = 0;
        for (int w = 0; w < nw; w++) total += s_valid[w];
        for (int64_t i = total + (int64_t)threadIdx.x; i < N; i += blockDim.x) row_pair[i] = -1;
    }
}

// ---- gather -------------------------------------------------------------------
template <typename TI, typename TO, bool VEC>
__global__ void k_gather_rows(const TI *x, int k, int H, int N, const int32_t *pair_row,
                              TO *rows) {
    pdl_enter();
    const int64_t t = blockIdx.x;
    const int i = blockIdx.y * blockDim.x + threadIdx.x;
    const int c = VEC ? i * 8 : i;
    if (c >= H) return;
    if constexpr (VEC) {
        Vec8<TI> in;
        in.load(x + t * H + c);
        float v[8];
        in.get(v);
        for (int j = 0; j < k; j++) {
            const int r = ld_i32(pair_row + t * k + j);
            if ((unsigned)r < (unsigned)N) Vec8<TO>::put(rows + (int64_t)r * H + c, v);
        }
    } else {
        const float v = Elem<TI>::load(x + t * H + c);
        for (int j = 0; j < k; j++) {
            const int r = ld_i32(pair_row + t * k + j);
            if ((unsigned)r < (unsigned)N) Elem<TO>::store(rows + (int64_t)r * H + c, v);
        }
    }
}

// ---- combine --------------------------------------------------------------------
// Four of the token's rows are in flight per thread.  w == null: weights of
// one (the gradient of gather).
template <typename TI, typename TO, bool VEC>
__global__ void k_combine_rows(const TI *rows, const float *w, int k, int H, int N,
                               const int32_t *pair_row, TO *out) {
    pdl_enter();
    const int64_t t = blockIdx.x;
    const int i = blockIdx.y * blockDim.x + threadIdx.x;
    const int c = VEC ? i * 8 : i;
    if (c >= H) return;
    constexpr int U = 4;
    if constexpr (VEC) {
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int j0 = 0; j0 < k; j0 += U) {
            int r[U];
            float wj[U];
            Vec8<TI> in[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                r[u] = j0 + u < k ? ld_i32(pair_row + t * k + j0 + u) : -1;
                wj[u] = w && j0 + u < k ? ld_f32(w + t * k + j0 + u) : 1.f;
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if ((unsigned)r[u] < (unsigned)N) in[u].load(rows + (int64_t)r[u] * H + c);
#pragma unroll
            for (int u = 0; u < U; u++)
                if ((unsigned)r[u] < (unsigned)N) {
                    float v[8];
                    in[u].get(v);
#pragma unroll
                    for (int q = 0; q < 8; q++) acc[q] = fmaf(wj[u], v[q], acc[q]);
                }
        }
        Vec8<TO>::put(out + t * H + c, acc);
    } else {
        float acc = 0.f;
        for (int j0 = 0; j0 < k; j0 += U) {
            float v[U], wj[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int r = j0 + u < k ? ld_i32(pair_row + t * k + j0 + u) : -1;
                const bool on = (unsigned)r < (unsigned)N;
                wj[u] = !on ? 0.f : w ? ld_f32(w + t * k + j0 + u) : 1.f;
                v[u] = on ? Elem<TI>::load(rows + (int64_t)r * H + c) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < U; u++) acc = fmaf(wj[u], v[u], acc);
        }
        Elem<TO>::store(out + t * H + c, acc);
    }
}

// ---- combine, backward ------------------------------------------------------------
// One warp per pair: it reads the pair's expert row and the token's output
// gradient once, for the dot product (dw) and the scaled copy (drows).  The k
// warps of a token share its gradient row through L1.
constexpr int CB_WARPS = 8;
template <typename TG, typename TR, bool VEC>
__global__ void __launch_bounds__(CB_WARPS * 32)
k_combine_rows_backward(const TG *grad_out, const TR *rows, const float *w, int k, int H, int N,
                        const int32_t *pair_row, TR *grad_rows, float *grad_w) {
    pdl_enter();
    const int lane = threadIdx.x & 31;
    const int64_t p = (int64_t)blockIdx.x * CB_WARPS + (threadIdx.x >> 5);
    if (p >= N) return;
    const int r = ld_i32(pair_row + p);
    if ((unsigned)r >= (unsigned)N) {
        if (grad_w && lane == 0) grad_w[p] = 0.f;
        return;
    }
    const float wp = grad_rows ? ld_f32(w + p) : 0.f;
    const TG *g = grad_out + p / k * H;
    const TR *x = rows + (int64_t)r * H;
    TR *gx = grad_rows + (int64_t)r * H;
    float dot = 0.f;
    if constexpr (VEC) {
        constexpr int U = 2;
        for (int c0 = lane * 8; c0 < H; c0 += U * 256) {
            Vec8<TG> gv[U];
            Vec8<TR> xv[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int c = c0 + u * 256;
                gv[u].zero();
                xv[u].zero();
                if (c < H) {
                    gv[u].load(g + c);
                    if (grad_w) xv[u].load(x + c);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int c = c0 + u * 256;
                float a[8], b[8];
                gv[u].get(a);
                xv[u].get(b);
#pragma unroll
                for (int q = 0; q < 8; q++) dot = fmaf(a[q], b[q], dot);
                if (grad_rows && c < H) {
#pragma unroll
                    for (int q = 0; q < 8; q++) a[q] *= wp;
                    Vec8<TR>::put(gx + c, a);
                }
            }
        }
    } else {
        for (int c = lane; c < H; c += 32) {
            const float a = Elem<TG>::load(g + c);
            if (grad_w) dot = fmaf(a, Elem<TR>::load(x + c), dot);
            if (grad_rows) Elem<TR>::store(gx + c, a * wp);
        }
    }
    if (grad_w) {
#pragma unroll
        for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(~0u, dot, o);
        if (lane == 0) grad_w[p] = dot;
    }
}

// ---- per-token int8 ------------------------------------------------------------------
// scale = max(amax / 127, 1e-8), code = clamp(round_half_away(x / scale)),
// the rule of quantizeInt8 (model/moe.go:165-188) with the whole row as the
// group and an IEEE float32 quotient.  A row that holds an infinity or NaN has
// scale NaN and codes 0, so that what is computed from it is NaN.  One CTA per
// row; the row stays in registers between the maximum and the codes up to
// CH * 8 values a thread, longer rows are read twice.  With pair_row, row t
// goes to the k rows of its pairs.
constexpr int QR_THREADS = 256;

__device__ __forceinline__ float amax_or_inf(float m, float v) {
    const float a = fabsf(v);
    return a <= FLT_MAX ? fmaxf(m, a) : CUDART_INF_F;
}
__device__ __forceinline__ uint32_t code_of(float v, float s) {
    const float q = fminf(fmaxf(roundf(__fdiv_rn(v, s)), -127.f), 127.f);
    return (uint32_t)(int)q & 0xFFu;
}

template <typename TI, bool VEC, int CH>
__global__ void __launch_bounds__(QR_THREADS)
k_quantize_rows(const TI *x, int k, int K, int N, const int32_t *pair_row, int8_t *codes,
                int64_t ld, float *scale) {
    __shared__ float s_max[QR_THREADS / 32];
    pdl_enter();
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x, nt = blockDim.x;
    const TI *src = x + t * K;
    float m = 0.f;
    Vec8<TI> keep[CH > 0 ? CH : 1];
    if constexpr (VEC && CH > 0) {
#pragma unroll
        for (int h = 0; h < CH; h++) {
            const int c = (h * nt + tid) * 8;
            keep[h].zero();
            if (c < K) keep[h].load(src + c);
        }
#pragma unroll
        for (int h = 0; h < CH; h++) {
            float v[8];
            keep[h].get(v);
#pragma unroll
            for (int q = 0; q < 8; q++) m = amax_or_inf(m, v[q]);
        }
    } else if constexpr (VEC) {
        for (int c = tid * 8; c < K; c += nt * 8) {
            Vec8<TI> in;
            float v[8];
            in.load(src + c);
            in.get(v);
#pragma unroll
            for (int q = 0; q < 8; q++) m = amax_or_inf(m, v[q]);
        }
    } else {
        for (int c = tid; c < K; c += nt) m = amax_or_inf(m, Elem<TI>::load(src + c));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if ((tid & 31) == 0) s_max[tid >> 5] = m;
    __syncthreads();
    m = s_max[0];
    for (int w = 1; w < nt >> 5; w++) m = fmaxf(m, s_max[w]);
    const bool bad = m > FLT_MAX;
    const float s = bad ? 1.f : fmaxf(__fdiv_rn(m, 127.f), 1e-8f);

    const int n_dst = pair_row ? k : 1;
    auto dst_row = [&](int j) -> int {
        if (!pair_row) return (int)t;
        return ld_i32(pair_row + t * k + j);
    };
    if (tid < n_dst) {
        for (int j = tid; j < n_dst; j += nt) {
            const int r = dst_row(j);
            if ((unsigned)r < (unsigned)N) scale[r] = bad ? CUDART_NAN_F : s;
        }
    }
    auto emit8 = [&](int c, const float (&v)[8]) {
        uint32_t lo = 0, hi = 0;
        if (!bad) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                lo |= code_of(v[q], s) << (8 * q);
                hi |= code_of(v[4 + q], s) << (8 * q);
            }
        }
        for (int j = 0; j < n_dst; j++) {
            const int r = dst_row(j);
            if ((unsigned)r < (unsigned)N)
                *reinterpret_cast<uint2 *>(codes + (int64_t)r * ld + c) = make_uint2(lo, hi);
        }
    };
    if constexpr (VEC && CH > 0) {
#pragma unroll
        for (int h = 0; h < CH; h++) {
            const int c = (h * nt + tid) * 8;
            if (c < K) {
                float v[8];
                keep[h].get(v);
                emit8(c, v);
            }
        }
    } else if constexpr (VEC) {
        for (int c = tid * 8; c < K; c += nt * 8) {
            Vec8<TI> in;
            float v[8];
            in.load(src + c);
            in.get(v);
            emit8(c, v);
        }
    } else {
        // four codes a store; ld is a multiple of 16, so the store that ends
        // past K stays in the row
        for (int c = tid * 4; c < K; c += nt * 4) {
            uint32_t u = 0;
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (!bad && c + q < K) u |= code_of(Elem<TI>::load(src + c + q), s) << (8 * q);
            for (int j = 0; j < n_dst; j++) {
                const int r = dst_row(j);
                if ((unsigned)r < (unsigned)N)
                    *reinterpret_cast<uint32_t *>(codes + (int64_t)r * ld + c) = u;
            }
        }
    }
}

// ---- host side ---------------------------------------------------------------------
static bool is_row_dtype(int dt) {
    return dt == QGMOE_DT_F32 || dt == QGMOE_DT_F16 || dt == QGMOE_DT_BF16;
}
static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Calls f with a null pointer of the dtype's C++ type.
template <typename F> static int with_dtype(int dt, F f) {
    if (dt == QGMOE_DT_F32) return f(static_cast<float *>(nullptr));
    if (dt == QGMOE_DT_F16) return f(static_cast<__half *>(nullptr));
    return f(static_cast<__nv_bfloat16 *>(nullptr));
}

// Threads of a CTA and CTAs along a row for one element group per thread.
static void row_grid(int64_t T, int H, bool vec, dim3 *grid, int *threads) {
    const int n = vec ? H / 8 : H;
    int th = (n + 31) / 32 * 32;
    if (th > 256) th = 256;
    *threads = th;
    *grid = dim3((unsigned)T, (unsigned)((n + th - 1) / th));
}

int check_pairs(int32_t T, int32_t k, const char *what) {
    if (T < 0 || k <= 0 || (int64_t)T * k > QGMOE_MAX_PAIRS)
        return set_error(QGMOE_ERR_INVALID_ARG, "%s: bad T=%d k=%d (k >= 1, T * k <= %d)", what, T,
                         k, QGMOE_MAX_PAIRS);
    return QGMOE_OK;
}

static int check_rows(int32_t T, int32_t k, int32_t H, int dt_a, int dt_b, const char *what) {
    int rc = check_pairs(T, k, what);
    if (rc) return rc;
    if (H <= 0 || H > QGMOE_MAX_ROW)
        return set_error(QGMOE_ERR_INVALID_ARG, "%s: bad row length %d (1..%d)", what, H,
                         QGMOE_MAX_ROW);
    if (!is_row_dtype(dt_a) || !is_row_dtype(dt_b))
        return set_error(QGMOE_ERR_INVALID_ARG, "%s: rows are F32, F16 or BF16 (got %d, %d)", what,
                         dt_a, dt_b);
    return QGMOE_OK;
}

static int launch_combine_rows(const void *rows, int rdt, const float *w, int T, int k, int H,
                               const int32_t *pair_row, void *out, int odt, cudaStream_t s) {
    const bool vec = H % 8 == 0 && aligned16(rows) && aligned16(out);
    dim3 grid;
    int th;
    row_grid(T, H, vec, &grid, &th);
    return with_dtype(rdt, [&](auto *ip) {
        return with_dtype(odt, [&](auto *op) {
            using TI = std::remove_pointer_t<decltype(ip)>;
            using TO = std::remove_pointer_t<decltype(op)>;
            auto kern = vec ? k_combine_rows<TI, TO, true> : k_combine_rows<TI, TO, false>;
            QG_CUDA(launch_pdl(kern, grid, dim3(th), 0, s, 1, static_cast<const TI *>(rows), w, k,
                               H, T * k, pair_row, static_cast<TO *>(out)));
            return (int)QGMOE_OK;
        });
    });
}

int launch_quantize_rows(const void *x, int dt, int T, int k, int K, const int32_t *pair_row,
                         int8_t *codes, int64_t ld, float *scale, cudaStream_t s) {
    const bool vec = K % 8 == 0 && aligned16(x);
    int th = (((vec ? K / 8 : (K + 3) / 4) + 31) / 32) * 32;
    if (th > QR_THREADS) th = QR_THREADS;
    const int per = th * 8;
    const int N = pair_row ? T * k : T;
    return with_dtype(dt, [&](auto *ip) {
        using TI = std::remove_pointer_t<decltype(ip)>;
        auto kern = !vec           ? k_quantize_rows<TI, false, 0>
                    : K <= per     ? k_quantize_rows<TI, true, 1>
                    : K <= 2 * per ? k_quantize_rows<TI, true, 2>
                    : K <= 4 * per ? k_quantize_rows<TI, true, 4>
                                   : k_quantize_rows<TI, true, 0>;
        QG_CUDA(launch_pdl(kern, dim3((unsigned)T), dim3(th), 0, s, 1, static_cast<const TI *>(x),
                           k, K, N, pair_row, codes, ld, scale));
        return (int)QGMOE_OK;
    });
}

int check_quantize_rows(const void *x, int dt, int T, int k, int K, const int32_t *pair_row,
                        const void *codes, int64_t ld, const void *scale) {
    int rc = check_rows(T, k, K, dt, dt, "quantize_rows");
    if (rc) return rc;
    if (!pair_row && k != 1)
        return set_error(QGMOE_ERR_INVALID_ARG, "quantize_rows: k=%d without pair_row", k);
    if (ld < K || ld % 16 || ld > (int64_t)QGMOE_MAX_ROW + 15)
        return set_error(QGMOE_ERR_INVALID_ARG,
                         "quantize_rows: pitch %lld of %d codes (a multiple of 16, >= them)",
                         (long long)ld, K);
    if (T == 0) return QGMOE_OK;
    if (!x || !codes || !scale)
        return set_error(QGMOE_ERR_INVALID_ARG, "quantize_rows: null pointer argument");
    if (!aligned16(codes))
        return set_error(QGMOE_ERR_INVALID_ARG, "quantize_rows: codes must be 16-byte aligned");
    return QGMOE_OK;
}

}  // namespace qg

using namespace qg;

extern "C" {

int qgmoe_sort_tokens(const int32_t *sel_idx, int32_t T, int32_t k, int32_t E, int32_t *offsets,
                      int32_t *pair_row, int32_t *row_pair, void *stream) {
    int rc = check_pairs(T, k, "sort_tokens");
    if (rc) return rc;
    if (E <= 0 || E > QG_MAX_EXPERTS)
        return set_error(QGMOE_ERR_INVALID_ARG, "sort_tokens: E=%d (1..%d)", E, QG_MAX_EXPERTS);
    if (!offsets || (T > 0 && (!sel_idx || !pair_row)))
        return set_error(QGMOE_ERR_INVALID_ARG, "sort_tokens: null pointer argument");
    const int N = T * k;
    // a warp per 512 pairs: fewer leave the reads of a CTA exposed, more only
    // add warps that have nothing to count
    int warps = (N + 511) / 512;
    warps = warps < 1 ? 1 : warps > SORT_MAX_WARPS ? SORT_MAX_WARPS : warps;
    QG_CUDA(launch_pdl(k_sort_tokens, dim3((unsigned)E), dim3(warps * 32), 0,
                       static_cast<cudaStream_t>(stream), 1, sel_idx, N, E, offsets, pair_row,
                       row_pair));
    return QGMOE_OK;
}

int qgmoe_gather_rows(const void *x, int32_t x_dtype, int32_t T, int32_t k, int32_t H,
                      const int32_t *pair_row, void *rows, int32_t rows_dtype, void *stream) {
    int rc = check_rows(T, k, H, x_dtype, rows_dtype, "gather_rows");
    if (rc) return rc;
    if (T == 0) return QGMOE_OK;
    if (!x || !pair_row || !rows)
        return set_error(QGMOE_ERR_INVALID_ARG, "gather_rows: null pointer argument");
    const bool vec = H % 8 == 0 && aligned16(x) && aligned16(rows);
    dim3 grid;
    int th;
    row_grid(T, H, vec, &grid, &th);
    return with_dtype(x_dtype, [&](auto *ip) {
        return with_dtype(rows_dtype, [&](auto *op) {
            using TI = std::remove_pointer_t<decltype(ip)>;
            using TO = std::remove_pointer_t<decltype(op)>;
            auto kern = vec ? k_gather_rows<TI, TO, true> : k_gather_rows<TI, TO, false>;
            QG_CUDA(launch_pdl(kern, grid, dim3(th), 0, static_cast<cudaStream_t>(stream), 1,
                               static_cast<const TI *>(x), k, H, T * k, pair_row,
                               static_cast<TO *>(rows)));
            return (int)QGMOE_OK;
        });
    });
}

int qgmoe_gather_rows_backward(const void *grad_rows, int32_t rows_dtype, int32_t T, int32_t k,
                               int32_t H, const int32_t *pair_row, void *grad_x, int32_t x_dtype,
                               void *stream) {
    int rc = check_rows(T, k, H, x_dtype, rows_dtype, "gather_rows_backward");
    if (rc) return rc;
    if (T == 0) return QGMOE_OK;
    if (!grad_rows || !pair_row || !grad_x)
        return set_error(QGMOE_ERR_INVALID_ARG, "gather_rows_backward: null pointer argument");
    return launch_combine_rows(grad_rows, rows_dtype, nullptr, T, k, H, pair_row, grad_x, x_dtype,
                               static_cast<cudaStream_t>(stream));
}

int qgmoe_combine_rows(const void *rows, int32_t rows_dtype, const float *w, int32_t T, int32_t k,
                       int32_t H, const int32_t *pair_row, void *out, int32_t out_dtype,
                       void *stream) {
    int rc = check_rows(T, k, H, rows_dtype, out_dtype, "combine_rows");
    if (rc) return rc;
    if (T == 0) return QGMOE_OK;
    if (!rows || !w || !pair_row || !out)
        return set_error(QGMOE_ERR_INVALID_ARG, "combine_rows: null pointer argument");
    return launch_combine_rows(rows, rows_dtype, w, T, k, H, pair_row, out, out_dtype,
                               static_cast<cudaStream_t>(stream));
}

int qgmoe_combine_rows_backward(const void *grad_out, int32_t out_dtype, const void *rows,
                                int32_t rows_dtype, const float *w, int32_t T, int32_t k,
                                int32_t H, const int32_t *pair_row, void *grad_rows,
                                float *grad_w, void *stream) {
    int rc = check_rows(T, k, H, rows_dtype, out_dtype, "combine_rows_backward");
    if (rc) return rc;
    if (T == 0 || (!grad_rows && !grad_w)) return QGMOE_OK;
    if (!grad_out || !pair_row || (grad_w && !rows) || (grad_rows && !w))
        return set_error(QGMOE_ERR_INVALID_ARG, "combine_rows_backward: null pointer argument");
    const bool vec = H % 8 == 0 && aligned16(grad_out) && (!rows || aligned16(rows)) &&
                     (!grad_rows || aligned16(grad_rows));
    const int N = T * k;
    return with_dtype(out_dtype, [&](auto *gp) {
        return with_dtype(rows_dtype, [&](auto *rp) {
            using TG = std::remove_pointer_t<decltype(gp)>;
            using TR = std::remove_pointer_t<decltype(rp)>;
            auto kern = vec ? k_combine_rows_backward<TG, TR, true>
                            : k_combine_rows_backward<TG, TR, false>;
            QG_CUDA(launch_pdl(kern, dim3((unsigned)((N + CB_WARPS - 1) / CB_WARPS)),
                               dim3(CB_WARPS * 32), 0, static_cast<cudaStream_t>(stream), 1,
                               static_cast<const TG *>(grad_out), static_cast<const TR *>(rows), w,
                               k, H, N, pair_row, static_cast<TR *>(grad_rows), grad_w));
            return (int)QGMOE_OK;
        });
    });
}

int qgq8_quantize_rows(const void *x, int32_t x_dtype, int32_t T, int32_t k, int32_t K,
                       const int32_t *pair_row, int8_t *codes, int64_t ld, float *scale,
                       void *stream) {
    int rc = check_quantize_rows(x, x_dtype, T, k, K, pair_row, codes, ld, scale);
    if (rc || T == 0) return rc;
    return launch_quantize_rows(x, x_dtype, T, k, K, pair_row, codes, ld, scale,
                                static_cast<cudaStream_t>(stream));
}

}  // extern "C"
