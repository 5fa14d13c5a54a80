// Product in 8-bit integers with a scale for each token and each output
// channel, dense or grouped by expert:
//   y[r, o] = float(sum_i c[r, i] * q[g(r), o, i]) * ws[g(r), o] * s[r]
// c [R, I] int8 codes of the rows with scales s (qgq8_quantize_rows), q
// [G, O, I] int8 weights with scales ws, rows offsets[g] .. offsets[g+1] for
// group g (one group without offsets).  The sum is exact in 32 bits
// (I <= 131071), the product with the scales is float32, rounded once more
// where y has 16 bits.  With SwiGLU the weight rows are gate [0, O/2) and up
// [O/2, O) (model/moe.go:70-76) and y has O/2 columns, silu(gate) * up.
//
// Swap-AB on the tensor cores, as the group-32 GEMMs (qg_umma.cu) do it:
//   D[channels, rows] = Q[channels, I] * C[rows, I]^T   (tcgen05.mma kind::i8)
// so that one tile is 128 channels x up to 256 rows, a batch of few rows costs
// a narrow N instead of an empty M, and 32 lanes of a warp hold 32 neighbouring
// channels of one row, which go out as one coalesced run without a detour
// through shared memory.  Both operands are tiled TMA loads of 128-byte rows
// (128B swizzle), accumulators are int32 in TMEM, double-buffered: eight
// epilogue warps drain one buffer while the next tile accumulates.
//
// Persistent, one CTA per SM, units (group, row tile, channel tile) with the
// channel tile fastest, so that concurrent CTAs share a row tile and, over the
// following units, the group's weights in L2.  Every wait is bounded; a wait
// that runs out raises QG_FLAG_TIMEOUT, the CTA lets its own loads and MMAs
// finish, frees its TMEM and leaves.
#include <cuda_bf16.h>
#include <cudaTypedefs.h>

#include <new>

#include "qg_common.cuh"
#include "qg_sm100.cuh"

namespace qg {
using namespace sm100;

constexpr int I8_M = 128;          // weight rows per tile (= TMEM lanes)
constexpr int I8_BK = 128;         // codes per stage: one swizzled 128-byte row
constexpr int I8_EPI_WARPS = 8;    // warps 0-7: TMEM lane quarter = warp & 3
constexpr int I8_LOAD_WARP = 8;
constexpr int I8_MMA_WARP = 9;
constexpr int I8_THREADS = 10 * 32;
constexpr int I8_MAX_GROUPS = QG_MAX_EXPERTS;
constexpr int I8_MAX_IN = 131071;  // 131071 * 128 * 128 < 2^31: exact int32 sums
constexpr long long I8_WAIT_CYCLES = 4000000000LL;  // ~2 s

// NT: most rows of a tile.  Stages fill the shared memory that one CTA per SM
// may use, so that as many loads as possible are in flight.
template <int NT>
struct I8Cfg {
    static constexpr int A_BYTES = I8_M * I8_BK;
    static constexpr int B_BYTES = NT * I8_BK;
    static constexpr int BOX = NT < 64 ? NT : 64;  // rows of one TMA box of the row codes
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int BUF = NT < 32 ? 32 : NT;  // TMEM columns per accumulator buffer
    static constexpr int TMEM_COLS = 2 * BUF;
    static constexpr int S = 208 * 1024 / STAGE_BYTES < 12 ? 208 * 1024 / STAGE_BYTES : 12;
    static constexpr int BAR_BYTES = 8 * (2 * S + 5) + 16;
    static constexpr int TAB_BYTES = (I8_MAX_GROUPS + 1) * 4;
    static constexpr int SMEM = S * STAGE_BYTES + TAB_BYTES + 16 + BAR_BYTES + 1024;
    static_assert(SMEM <= 232448, "shared memory budget");
    static_assert(STAGE_BYTES % 1024 == 0 && (BOX * I8_BK) % 1024 == 0, "1024-byte aligned tiles");
    static_assert(TMEM_COLS <= 512 && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "TMEM budget");
};

struct I8Args {
    const float *xs;         // [R] row scales
    const float *ws;         // [G * RT * 128] channel scales in tile order
    const int32_t *offsets;  // [G + 1] device, or null: one group of R rows
    int G, R, RT, KB, cols;  // RT channel tiles per group, KB 128-code blocks, y columns
    int nt;                  // rows of a tile (<= NT, a multiple of 16)
    void *y;                 // [R, cols]
    int *err;
};

// kind::i8 instruction descriptor: int8 A/B, int32 D, both K-major.
__device__ __forceinline__ uint32_t idesc_i8(int N) {
    return (2u << 4)                     // D format S32
           | (1u << 7) | (1u << 10)      // A, B signed 8 bits
           | ((uint32_t)(N >> 3) << 17)  // N / 8
           | ((uint32_t)(I8_M >> 4) << 24);
}

// One 128-code block as four K=32 MMAs; descriptors advance by 32 bytes.
__device__ __forceinline__ void umma_i8_k128(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                             uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.eq.b32 t, %3, %3;\n\t"
        "add.u64 a1, %1, 2;\n\tadd.u64 a2, %1, 4;\n\tadd.u64 a3, %1, 6;\n\t"
        "add.u64 b1, %2, 2;\n\tadd.u64 b2, %2, 4;\n\tadd.u64 b3, %2, 6;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], a1, b1, %3, t;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], a2, b2, %3, t;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], a3, b3, %3, t;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

struct I8Unit {
    int g, rt, row0, n;
};

// Unit u from the groups' tile prefix (shared memory).  Row tiles of a group
// all have a.nt rows but the last.
__device__ __forceinline__ I8Unit i8_unit(const I8Args &a, const int *prefix, int u) {
    I8Unit w;
    const int ti = u / a.RT;
    w.rt = u - ti * a.RT;
    int lo = 0, hi = a.G - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= ti) lo = mid; else hi = mid - 1;
    }
    w.g = lo;
    const int tt = ti - prefix[lo];
    int begin = 0, end = a.R;
    if (a.offsets) {
        begin = *(const volatile int32_t *)(a.offsets + lo);
        end = *(const volatile int32_t *)(a.offsets + lo + 1);
    }
    w.row0 = begin + tt * a.nt;
    w.n = min(a.nt, end - w.row0);
    return w;
}

__device__ __forceinline__ void i8_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void i8_store(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void i8_store(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// silu(g) * u = g / (1 + e^-g) * u in float32.  e^-g may overflow to infinity,
// where the quotient is the right limit, -0.
__device__ __forceinline__ float swiglu(float g, float u) {
    return __fdividef(g, 1.f + expf(-g)) * u;
}

template <int NT, typename TO, bool SWIGLU>
__global__ void __launch_bounds__(I8_THREADS, 1)
k_i8(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
     const I8Args a) {
    pdl_launch_dependents();
    using Cfg = I8Cfg<NT>;
    constexpr int S = Cfg::S;
    extern __shared__ uint8_t smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    uint8_t *base = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(base + S * Cfg::STAGE_BYTES);
    uint64_t *empty = full + S;
    uint64_t *accFull = empty + S;     // [2]
    uint64_t *accEmpty = accFull + 2;  // [2]
    uint64_t *drain = accEmpty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    const uint32_t abort_addr = smem_u32(tmem_slot + 1);
    int *prefix = reinterpret_cast<int *>(tmem_slot + 4);

    if (tid == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&accFull[b], 1);
            mbar_init(&accEmpty[b], I8_EPI_WARPS);
        }
        mbar_init(drain, 1);
        st_volatile_shared(abort_addr, 0);
        fence_mbar_init();
        prefetch_tmap(&tmap_w);
        prefetch_tmap(&tmap_x);
    }
    if (warp == I8_MMA_WARP) {
        tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
        tmem_relinquish();
    }
    pdl_wait();
    if (warp == 0) {  // row tiles before each group; a group whose range is not one has none
        int total = 0;
        for (int g0 = 0; g0 < a.G; g0 += 32) {
            const int g = g0 + lane;
            int n = 0;
            if (g < a.G) {
                if (a.offsets) {
                    const int b = *(const volatile int32_t *)(a.offsets + g);
                    const int e = *(const volatile int32_t *)(a.offsets + g + 1);
                    if (b < 0 || e < b || e > a.R)
                        atomicOr(a.err, QG_FLAG_BAD_GROUP);
                    else
                        n = e - b;
                } else {
                    n = a.R;
                }
            }
            int t = (n + a.nt - 1) / a.nt, sum = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(~0u, sum, o);
                if (lane >= o) sum += v;
            }
            if (g < a.G) prefix[g] = total + sum - t;
            total += __shfl_sync(~0u, sum, 31);
        }
        if (lane == 0) prefix[a.G] = total;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int n_units = prefix[a.G] * a.RT;

    auto fail = [&]() {
        if (!ld_volatile_shared(abort_addr)) {
            st_volatile_shared(abort_addr, 1);
            atomicOr(a.err, QG_FLAG_TIMEOUT);
        }
    };

    if (warp < I8_EPI_WARPS) {
        // ============ epilogue: TMEM -> scaled rows ===============================
        // Warp w reads lane quarter w & 3; the two warps of a quarter take
        // alternate runs of 32 row columns.
        const int q = warp & 3, half = warp >> 2;
        int lt = 0;
        for (int u = blockIdx.x; u < n_units; u += gridDim.x, lt++) {
            const int buf = lt & 1;
            const I8Unit w = i8_unit(a, prefix, u);
            const float sw = a.ws[((size_t)w.g * a.RT + w.rt) * I8_M + q * 32 + lane];
            // the lanes wait one by one and must leave the loop together
            if (!__all_sync(~0u, mbar_wait(&accFull[buf], (lt >> 1) & 1, abort_addr,
                                           I8_WAIT_CYCLES))) {
                fail();
                break;
            }
            tc_fence_after();
            for (int c0 = half * 32; c0 < w.n; c0 += 64) {
                const int nc = min(32, w.n - c0);
                const int64_t r0 = (int64_t)w.row0 + c0;
                const float sx = lane < nc ? *(const volatile float *)(a.xs + r0 + lane) : 0.f;
                float v[32];
                tmem_ld32(tmem + buf * Cfg::BUF + c0 + ((uint32_t)(q * 32) << 16), v);
#pragma unroll
                for (int c = 0; c < 32; c++)
                    // the row's scale last: it is as large as the activations
                    // are, and the sum times it may overflow where y does not
                    v[c] = (float)__float_as_int(v[c]) * sw * __shfl_sync(~0u, sx, c);
                if constexpr (SWIGLU) {
                    // lanes 0-15 hold gate rows, 16-31 the up rows of the same
                    // columns: per two rows one exchange gives each half-warp
                    // gate and up of one of them
                    const int o = w.rt * 64 + q * 16 + (lane & 15);
                    const bool up = lane >= 16;
                    TO *yp = static_cast<TO *>(a.y) + r0 * a.cols + o;
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        const float other = __shfl_xor_sync(~0u, up ? v[c] : v[c + 1], 16);
                        const float h = up ? swiglu(other, v[c + 1]) : swiglu(v[c], other);
                        const int cc = c + up;
                        if (cc < nc && o < a.cols) i8_store(yp + (int64_t)cc * a.cols, h);
                    }
                } else {
                    const int o = w.rt * I8_M + q * 32 + lane;
                    TO *yp = static_cast<TO *>(a.y) + r0 * a.cols + o;
                    if (o < a.cols) {
#pragma unroll
                        for (int c = 0; c < 32; c++)
                            if (c < nc) i8_store(yp + (int64_t)c * a.cols, v[c]);
                    }
                }
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&accEmpty[buf]);
        }
    } else if (warp == I8_LOAD_WARP) {
        // ============ loads: weight tile and row tile of each 128-code block ======
        if (lane == 0) {
            int g = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < n_units && ok; u += gridDim.x) {
                const I8Unit w = i8_unit(a, prefix, u);
                const int wrow = (w.g * a.RT + w.rt) * I8_M;
                const int boxes = (w.n + Cfg::BOX - 1) / Cfg::BOX;
                for (int kb = 0; kb < a.KB; kb++, g++) {
                    const int s = g % S;
                    if (!mbar_wait(&empty[s], ((g / S) & 1) ^ 1, abort_addr, I8_WAIT_CYCLES)) {
                        fail();
                        ok = false;
                        break;
                    }
                    uint8_t *dst = base + s * Cfg::STAGE_BYTES;
                    mbar_arrive_expect_tx(&full[s], Cfg::A_BYTES + boxes * Cfg::BOX * I8_BK);
                    tma_load_2d(dst, &tmap_w, kb * I8_BK, wrow, &full[s]);
                    for (int b = 0; b < boxes; b++)
                        tma_load_2d(dst + Cfg::A_BYTES + b * Cfg::BOX * I8_BK, &tmap_x, kb * I8_BK,
                                    w.row0 + b * Cfg::BOX, &full[s]);
                }
            }
            // our own copies land before the shared memory goes, also when
            // another role gave up
            for (int i = g > S ? g - S : 0; i < g; i++)
                mbar_wait(&full[i % S], (i / S) & 1, 0, I8_WAIT_CYCLES);
        }
        __syncwarp();
    } else {
        // ============ MMA issuer ===================================================
        if (lane == 0) {
            int g = 0, lt = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < n_units && ok; u += gridDim.x, lt++) {
                const I8Unit w = i8_unit(a, prefix, u);
                const uint32_t idesc = idesc_i8((w.n + 15) & ~15);
                const int buf = lt & 1;
                if (!mbar_wait(&accEmpty[buf], ((lt >> 1) & 1) ^ 1, abort_addr, I8_WAIT_CYCLES)) {
                    fail();
                    ok = false;
                    break;
                }
                tc_fence_after();
                for (int kb = 0; kb < a.KB; kb++, g++) {
                    const int s = g % S;
                    if (!mbar_wait(&full[s], (g / S) & 1, abort_addr, I8_WAIT_CYCLES)) {
                        fail();
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t st = smem_u32(base + s * Cfg::STAGE_BYTES);
                    umma_i8_k128(tmem + buf * Cfg::BUF, desc_k_sw128(st),
                                 desc_k_sw128(st + Cfg::A_BYTES), idesc, kb != 0);
                    umma_commit(&empty[s]);
                }
                if (ok) umma_commit(&accFull[buf]);
            }
            if (!ok) {
                umma_commit(drain);
                mbar_wait(drain, 0, 0, I8_WAIT_CYCLES);
            }
        }
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == I8_MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::TMEM_COLS);
    }
}

// ---- weight layout -------------------------------------------------------------
// Rows of `groups` groups in tile order, pitch ldw, zeros past the group's
// rows and past I; scales alike.  With SwiGLU, tile rt holds output columns
// [rt*64, rt*64 + 64): of each 32 tile rows the first 16 are gate rows of 16
// columns, the others the up rows of the same columns.
__global__ void k_i8_layout(const int8_t *q, const float *scale, int groups, int O, int I,
                            int swiglu, int RT, int64_t ldw, int8_t *dst, float *dscale) {
    const int64_t row = blockIdx.x;  // of groups * RT * 128
    const int g = (int)(row / ((int64_t)RT * I8_M));
    const int l = (int)(row - (int64_t)g * RT * I8_M);
    int o = l;
    bool live = l < O;
    if (swiglu) {
        const int rt = l / I8_M, r = l % I8_M, cols = O / 2;
        const int c = rt * 64 + (r / 32) * 16 + (r & 15);
        live = c < cols;
        o = (r & 16) ? cols + c : c;
    }
    const int8_t *src = q + ((int64_t)g * O + o) * I;
    for (int64_t i = threadIdx.x; i < ldw; i += blockDim.x)
        dst[row * ldw + i] = live && i < I ? src[i] : (int8_t)0;
    if (threadIdx.x == 0) dscale[row] = live ? scale[(int64_t)g * O + o] : 0.f;
}

// ---- host side -------------------------------------------------------------------
int check_pairs(int32_t T, int32_t k, const char *what);
int check_quantize_rows(const void *x, int dt, int T, int k, int K, const int32_t *pair_row,
                        const void *codes, int64_t ld, const void *scale);
int launch_quantize_rows(const void *x, int dt, int T, int k, int K, const int32_t *pair_row,
                         int8_t *codes, int64_t ld, float *scale, cudaStream_t s);

static PFN_cuTensorMapEncodeTiled_v12000 i8_encode_fn() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000,
                                             cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// 2-D int8 [rows, cols] with row pitch ld bytes, boxes of 128 codes x box_rows
// rows, 128B swizzle, zeros beyond the edges.
static int i8_encode_map(CUtensorMap *map, const int8_t *ptr, int64_t rows, int cols, int64_t ld,
                         int box_rows) {
    auto fn = i8_encode_fn();
    if (!fn) return set_error(QGMOE_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {I8_BK, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(ptr), dims, strides,
                    box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(QGMOE_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return QGMOE_OK;
}

// Makes `device` current for a call and puts the caller's device back.
struct DeviceScope {
    int prev = -1;
    cudaError_t err;
    explicit DeviceScope(int device) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != device)
            err = cudaSetDevice(device);
        else
            prev = -1;
    }
    ~DeviceScope() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};
#define QG_ON_DEVICE(dev)            \
    ::qg::DeviceScope scope_((dev)); \
    QG_CUDA(scope_.err)

}  // namespace qg

using namespace qg;

struct qgq8 {
    int device = 0;
    int G = 0, O = 0, I = 0, cols = 0, RT = 0, KB = 0;
    bool swiglu = false;
    cudaStream_t stream = nullptr;
    int8_t *w = nullptr;   // [G * RT * 128, ldw]
    float *ws = nullptr;   // [G * RT * 128]
    int *err_dev = nullptr;
    CUtensorMap tmap_w{};
    // qgq8_forward's own buffers (it blocks, so no work outlives the call)
    int cap_T = 0;
    float *x_dev = nullptr, *y_dev = nullptr, *s_dev = nullptr;
    int8_t *c_dev = nullptr;
};

namespace qg {

static int64_t i8_pitch(int64_t I) { return (I + 15) & ~int64_t(15); }

// Most rows of a tile.  Short tiles for few rows per group (the stages then
// hold mostly weights), 256 for prompts.
static int i8_tile(int64_t rows_per_group) {
    return rows_per_group <= 16 ? 16 : rows_per_group <= 64 ? 64 : 256;
}

template <int NT, typename TO, bool SWIGLU>
static int launch_i8_t(const qgq8 *h, const CUtensorMap &tx, const I8Args &a, int64_t max_units,
                       cudaStream_t s) {
    auto kern = k_i8<NT, TO, SWIGLU>;
    constexpr int smem = I8Cfg<NT>::SMEM;
    static bool done[64] = {false};
    if (h->device >= 64 || !done[h->device]) {
        QG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        if (h->device < 64) done[h->device] = true;
    }
    int64_t grid = num_sms(h->device);
    if (max_units < grid) grid = max_units;
    QG_CUDA(launch_pdl(kern, dim3((unsigned)grid), dim3(I8_THREADS), smem, s, 1, h->tmap_w, tx, a));
    return QGMOE_OK;
}

template <int NT>
static int launch_i8(const qgq8 *h, const CUtensorMap &tx, const I8Args &a, int ydt, int64_t units,
                     cudaStream_t s) {
    if (h->swiglu)
        return ydt == QGMOE_DT_F32   ? launch_i8_t<NT, float, true>(h, tx, a, units, s)
               : ydt == QGMOE_DT_F16 ? launch_i8_t<NT, __half, true>(h, tx, a, units, s)
                                     : launch_i8_t<NT, __nv_bfloat16, true>(h, tx, a, units, s);
    return ydt == QGMOE_DT_F32   ? launch_i8_t<NT, float, false>(h, tx, a, units, s)
           : ydt == QGMOE_DT_F16 ? launch_i8_t<NT, __half, false>(h, tx, a, units, s)
                                 : launch_i8_t<NT, __nv_bfloat16, false>(h, tx, a, units, s);
}

static int i8_check_product(const qgq8 *h, const int8_t *codes, int64_t ld, const float *scale,
                            int32_t R, const int32_t *offsets, const void *y, int ydt) {
    if (!h) return set_error(QGMOE_ERR_INVALID_ARG, "null handle");
    if (R < 0 || R > QGMOE_MAX_PAIRS)
        return set_error(QGMOE_ERR_INVALID_ARG, "rows=%d (0..%d)", R, QGMOE_MAX_PAIRS);
    if (!offsets && h->G != 1)
        return set_error(QGMOE_ERR_INVALID_ARG, "%d groups need offsets", h->G);
    if (ydt != QGMOE_DT_F32 && ydt != QGMOE_DT_F16 && ydt != QGMOE_DT_BF16)
        return set_error(QGMOE_ERR_INVALID_ARG, "y is F32, F16 or BF16 (got %d)", ydt);
    if (ld < h->I || ld % 16 || ld > (int64_t)QGMOE_MAX_ROW + 15)
        return set_error(QGMOE_ERR_INVALID_ARG,
                         "pitch %lld of %d codes (a multiple of 16, >= them)", (long long)ld, h->I);
    if (R == 0) return QGMOE_OK;
    if (!codes || !scale || !y) return set_error(QGMOE_ERR_INVALID_ARG, "null pointer argument");
    if (reinterpret_cast<uintptr_t>(codes) & 15)
        return set_error(QGMOE_ERR_INVALID_ARG, "codes must be 16-byte aligned");
    return QGMOE_OK;
}

static int i8_product(const qgq8 *h, const int8_t *codes, int64_t ld, const float *scale, int R,
                      const int32_t *offsets, void *y, int ydt, cudaStream_t s) {
    const int64_t per = (R + (int64_t)h->G - 1) / h->G;  // mean rows of a group
    const int nt = i8_tile(per);
    CUtensorMap tx;
    int rc = i8_encode_map(&tx, codes, R, h->I, ld, nt < 64 ? nt : 64);
    if (rc) return rc;
    I8Args a{};
    a.xs = scale;
    a.ws = h->ws;
    a.offsets = offsets;
    a.G = h->G;
    a.R = R;
    a.RT = h->RT;
    a.KB = h->KB;
    a.cols = h->cols;
    a.nt = nt;
    a.y = y;
    a.err = h->err_dev;
    // row tiles: full ones, and at most one partial for each group that has rows
    const int64_t tiles = R / nt + (R < h->G ? R : h->G);
    const int64_t units = tiles * h->RT;
    return nt == 16   ? launch_i8<16>(h, tx, a, ydt, units, s)
           : nt == 64 ? launch_i8<64>(h, tx, a, ydt, units, s)
                      : launch_i8<256>(h, tx, a, ydt, units, s);
}

static void i8_free_work(qgq8 *h) {
    cudaFree(h->x_dev);
    cudaFree(h->y_dev);
    cudaFree(h->s_dev);
    cudaFree(h->c_dev);
    h->x_dev = h->y_dev = h->s_dev = nullptr;
    h->c_dev = nullptr;
    h->cap_T = 0;
}

static int i8_alloc(void **p, size_t bytes) {
    *p = nullptr;
    cudaError_t e = cudaMalloc(p, bytes);
    if (e != cudaSuccess)
        return set_error(QGMOE_ERR_CUDA, "cudaMalloc(%zu): %s", bytes, cudaGetErrorString(e));
    return QGMOE_OK;
}

// Device copies of the weights in tile order.  Host weights travel through a
// staging buffer of whole groups, 64 MB or one group.
static int i8_build(qgq8 *h, const int8_t *q, const float *scale, bool on_device) {
    const int64_t rows = (int64_t)h->G * h->RT * I8_M, ldw = i8_pitch(h->I);
    int rc = i8_alloc(reinterpret_cast<void **>(&h->w), (size_t)rows * ldw);
    if (!rc) rc = i8_alloc(reinterpret_cast<void **>(&h->ws), sizeof(float) * rows);
    if (!rc) rc = i8_alloc(reinterpret_cast<void **>(&h->err_dev), sizeof(int));
    if (!rc) rc = i8_encode_map(&h->tmap_w, h->w, rows, h->I, ldw, I8_M);
    if (rc) return rc;
    QG_CUDA(cudaMemsetAsync(h->err_dev, 0, sizeof(int), h->stream));
    const int64_t gbytes = (int64_t)h->O * h->I;
    if (on_device) {
        // whatever stream the caller wrote the weights on
        QG_CUDA(cudaDeviceSynchronize());
        k_i8_layout<<<(unsigned)rows, 256, 0, h->stream>>>(q, scale, h->G, h->O, h->I, h->swiglu,
                                                           h->RT, ldw, h->w, h->ws);
        QG_CUDA(cudaGetLastError());
        QG_CUDA(cudaStreamSynchronize(h->stream));
        return QGMOE_OK;
    }
    int64_t step = (64ll << 20) / gbytes;
    step = step < 1 ? 1 : step > h->G ? h->G : step;
    int8_t *tq = nullptr;
    float *ts = nullptr;
    rc = i8_alloc(reinterpret_cast<void **>(&tq), (size_t)(step * gbytes));
    if (!rc) rc = i8_alloc(reinterpret_cast<void **>(&ts), sizeof(float) * step * h->O);
    cudaError_t e = cudaSuccess;
    for (int64_t g = 0; g < h->G && !rc && e == cudaSuccess; g += step) {
        const int64_t n = step < h->G - g ? step : h->G - g;
        e = cudaMemcpyAsync(tq, q + g * gbytes, n * gbytes, cudaMemcpyHostToDevice, h->stream);
        if (e == cudaSuccess)
            e = cudaMemcpyAsync(ts, scale + g * h->O, sizeof(float) * n * h->O,
                                cudaMemcpyHostToDevice, h->stream);
        if (e != cudaSuccess) break;
        const int64_t r0 = g * h->RT * I8_M;
        k_i8_layout<<<(unsigned)(n * h->RT * I8_M), 256, 0, h->stream>>>(
            tq, ts, (int)n, h->O, h->I, h->swiglu, h->RT, ldw, h->w + r0 * ldw, h->ws + r0);
        e = cudaGetLastError();
        if (e == cudaSuccess) e = cudaStreamSynchronize(h->stream);  // tq is reused
    }
    cudaFree(tq);
    cudaFree(ts);
    if (!rc && e != cudaSuccess)
        rc = set_error(QGMOE_ERR_CUDA, "weight upload: %s", cudaGetErrorString(e));
    return rc;
}

}  // namespace qg

extern "C" {

int qgq8_create(int32_t groups, int32_t O, int32_t I, const int8_t *q, const float *scale,
                int32_t swiglu, int32_t on_device, int32_t device, qgq8_t **out) {
    if (!out) return set_error(QGMOE_ERR_INVALID_ARG, "null out");
    *out = nullptr;
    if (groups <= 0 || groups > I8_MAX_GROUPS || O <= 0 || I <= 0 || I > I8_MAX_IN)
        return set_error(QGMOE_ERR_INVALID_ARG, "bad shape groups=%d (1..%d) out=%d in=%d (1..%d)",
                         groups, I8_MAX_GROUPS, O, I, I8_MAX_IN);
    if (swiglu && O % 2)
        return set_error(QGMOE_ERR_INVALID_ARG, "SwiGLU needs gate and up rows: out=%d is odd", O);
    const int64_t cols = swiglu ? O / 2 : O, per = swiglu ? 64 : I8_M;
    const int64_t RT = (cols + per - 1) / per;
    if (RT * groups * I8_M > INT32_MAX)
        return set_error(QGMOE_ERR_INVALID_ARG, "groups=%d x out=%d is too many rows", groups, O);
    if (!q || !scale) return set_error(QGMOE_ERR_INVALID_ARG, "null weights");
    if (!qgmoe_device_ok(device))
        return set_error(QGMOE_ERR_NO_DEVICE, "device %d is not a usable sm_100 device", device);
    QG_ON_DEVICE(device);
    qgq8 *h = new (std::nothrow) qgq8();
    if (!h) return set_error(QGMOE_ERR_CUDA, "out of host memory");
    h->device = device;
    h->G = groups;
    h->O = O;
    h->I = I;
    h->cols = (int)cols;
    h->RT = (int)RT;
    h->KB = (I + I8_BK - 1) / I8_BK;
    h->swiglu = swiglu != 0;
    int rc = QGMOE_OK;
    cudaError_t e = cudaStreamCreateWithFlags(&h->stream, cudaStreamNonBlocking);
    if (e != cudaSuccess) rc = set_error(QGMOE_ERR_CUDA, "stream: %s", cudaGetErrorString(e));
    if (!rc) rc = i8_build(h, q, scale, on_device != 0);
    if (rc) {
        qgq8_destroy(h);
        return rc;
    }
    *out = h;
    return QGMOE_OK;
}

int qgq8_destroy(qgq8_t *h) {
    if (!h) return QGMOE_OK;
    {
        DeviceScope scope(h->device);
        cudaDeviceSynchronize();  // products on the caller's streams read the weights
        i8_free_work(h);
        cudaFree(h->w);
        cudaFree(h->ws);
        cudaFree(h->err_dev);
        if (h->stream) cudaStreamDestroy(h->stream);
    }
    delete h;
    return QGMOE_OK;
}

int qgq8_matmul_device(qgq8_t *h, const int8_t *codes, int64_t ld, const float *scale, int32_t R,
                       const int32_t *offsets, void *y, int32_t y_dtype, void *stream) {
    int rc = i8_check_product(h, codes, ld, scale, R, offsets, y, y_dtype);
    if (rc || R == 0) return rc;
    QG_ON_DEVICE(h->device);
    return i8_product(h, codes, ld, scale, R, offsets, y, y_dtype,
                      stream ? static_cast<cudaStream_t>(stream) : h->stream);
}

int qgq8_forward_device(qgq8_t *h, const void *x, int32_t x_dtype, int32_t T, int32_t k,
                        const int32_t *pair_row, const int32_t *offsets, int8_t *codes, int64_t ld,
                        float *scale, void *y, int32_t y_dtype, void *stream) {
    if (!h) return set_error(QGMOE_ERR_INVALID_ARG, "null handle");
    int rc = check_quantize_rows(x, x_dtype, T, k, h->I, pair_row, codes, ld, scale);
    if (rc) return rc;
    const int R = T * k;
    rc = i8_check_product(h, codes, ld, scale, R, offsets, y, y_dtype);
    if (rc || R == 0) return rc;
    QG_ON_DEVICE(h->device);
    cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : h->stream;
    rc = launch_quantize_rows(x, x_dtype, T, k, h->I, pair_row, codes, ld, scale, s);
    if (rc) return rc;
    return i8_product(h, codes, ld, scale, R, offsets, y, y_dtype, s);
}

int qgq8_forward(qgq8_t *h, const float *x, int32_t T, float *y) {
    if (!h) return set_error(QGMOE_ERR_INVALID_ARG, "null handle");
    if (h->G != 1) return set_error(QGMOE_ERR_INVALID_ARG, "%d groups: use the device calls", h->G);
    int rc = check_pairs(T, 1, "qgq8_forward");
    if (rc || T == 0) return rc;
    if (!x || !y) return set_error(QGMOE_ERR_INVALID_ARG, "null x/y");
    QG_ON_DEVICE(h->device);
    const int64_t ld = i8_pitch(h->I);
    if (T > h->cap_T) {
        QG_CUDA(cudaStreamSynchronize(h->stream));
        i8_free_work(h);
        rc = i8_alloc(reinterpret_cast<void **>(&h->x_dev), sizeof(float) * (size_t)T * h->I);
        if (!rc) rc = i8_alloc(reinterpret_cast<void **>(&h->y_dev), sizeof(float) * (size_t)T * h->cols);
        if (!rc) rc = i8_alloc(reinterpret_cast<void **>(&h->s_dev), sizeof(float) * (size_t)T);
        if (!rc) rc = i8_alloc(reinterpret_cast<void **>(&h->c_dev), (size_t)T * ld);
        if (rc) {
            i8_free_work(h);
            return rc;
        }
        h->cap_T = T;
    }
    cudaStream_t s = h->stream;
    QG_CUDA(cudaMemcpyAsync(h->x_dev, x, sizeof(float) * (size_t)T * h->I, cudaMemcpyHostToDevice, s));
    rc = qgq8_forward_device(h, h->x_dev, QGMOE_DT_F32, T, 1, nullptr, nullptr, h->c_dev, ld,
                             h->s_dev, h->y_dev, QGMOE_DT_F32, s);
    if (rc) return rc;
    QG_CUDA(cudaMemcpyAsync(y, h->y_dev, sizeof(float) * (size_t)T * h->cols, cudaMemcpyDeviceToHost, s));
    return qgq8_sync(h, nullptr);
}

int qgq8_sync(qgq8_t *h, void *stream) {
    if (!h) return set_error(QGMOE_ERR_INVALID_ARG, "null handle");
    QG_ON_DEVICE(h->device);
    cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : h->stream;
    int flag = 0;
    QG_CUDA(cudaMemcpyAsync(&flag, h->err_dev, sizeof(int), cudaMemcpyDeviceToHost, s));
    QG_CUDA(cudaStreamSynchronize(s));
    if (!flag) return QGMOE_OK;
    QG_CUDA(cudaMemsetAsync(h->err_dev, 0, sizeof(int), s));
    QG_CUDA(cudaStreamSynchronize(s));
    return set_error((flag & QG_FLAG_TIMEOUT) ? QGMOE_ERR_TIMEOUT : QGMOE_ERR_DEVICE_FLAG,
                     "device error flag 0x%x%s", flag,
                     (flag & QG_FLAG_BAD_GROUP) ? " (group offsets out of order or past the rows)"
                                                : "");
}

}  // extern "C"
