// linear_q8.cu -- the linear layer on 8-bit (e4m3) rows with a scale each, on
// tcgen05 (kind::f8f6f4, FP32 accumulators in TMEM):
//
//   y[m][n] = sx[m] sw[n] sum_k xq[m][k] wq[n][k] + bias[n] + residual[m][n]
//
// The weights are the MMA's M = 128 side and the activation rows its N side, so
// a thread of the epilogue owns one output column n: its scale and bias are
// registers, and a warp writes 32 neighbouring columns of a row whatever the
// rows' alignment.  Operands come by TMA in K blocks of 128 bytes (the 128-byte
// swizzle); rows and columns past the ends read as zeros.
//
// Persistent blocks, one an SM, take tiles of R <= 128 columns by C <= 256 rows
// (any R and C: what an MMA reads beyond them only reaches accumulators that
// nobody stores), all of K, two accumulators, so that a tile's epilogue runs
// beside the next tile's products.  plan_tiles picks R and C.  Large ones are bound
// by the tensor pipe (8192^3 390 us, 2.8 PFLOP/s), few rows by a block's chain of
// MMAs (1 to 64 rows of 8192 x 8192 16 us, 4.2 TB/s).
#include <cuda.h>

#include <atomic>

#include "ptx.cuh"
#include "quant.cuh"
#include "status.h"

namespace rk {
namespace {

struct Q8Args {
    const float *sx, *sw, *bias;
    const void* res;
    void* y;
    long long ldr, ldy;
    int rows, n, k;
};

__device__ uint32_t q8_err;  // set when a bounded wait of a kernel gives up

constexpr int Q8_M = 128;          // the MMA's weight rows
constexpr int Q8_KB = 128;         // bytes of K a block holds: a row of the 128-byte swizzle
constexpr int Q8_MAX_STAGES = 32;
constexpr int Q8_SMEM = 225 * 1024;
constexpr int Q8_EPI = 8;          // warps of the epilogue
constexpr int Q8_THREADS = 32 * (3 + Q8_EPI);  // and weights' loads, products, activations' loads

struct Q8Plan {
    int r, c;                // weight rows (output columns) and activation rows of a tile
    int blocks;              // K blocks of a stage
    int n_tiles, m_tiles;
    int stages;
    uint32_t x_off, stage;   // bytes: the activations' place in a stage, a stage
    uint32_t idesc;
    uint32_t acc_cols, tmem_cols;
    // Panels of 8 column tiles, row tiles one after the other within a panel: the blocks at work at a time share
    // their operands' rows in L2.
    __device__ void decode(int t, int& tn, int& tm) const {
        constexpr int PANEL = 8;
        const int per = PANEL * m_tiles, p = t / per, i = t - p * per;
        const int width = min(PANEL, n_tiles - p * PANEL);
        tm = i / width;
        tn = p * PANEL + i - tm * width;
    }
};

// 32 rows of one output column each lane: scales, bias, residual, the one rounding
template <typename T, bool FULL>
__device__ __forceinline__ void store_rows(const Q8Args& a, long long m, int n, int left, const float (&acc)[32],
                                           const float* sx, float sw, float bias) {
    T* y = static_cast<T*>(a.y) + m * a.ldy + n;
    T rv[32];
    if (a.res) {
        const T* r = static_cast<const T*>(a.res) + m * a.ldr + n;
#pragma unroll
        for (int j = 0; j < 32; j++) {
            if (FULL || j < left) rv[j] = *r;
            r += a.ldr;
        }
    }
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
        const float4 s = *reinterpret_cast<const float4*>(sx + j);
        const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // one scale after the other: their product may leave float's range where the result does not
            float v = fmaf(acc[j + i] * sw, f[i], bias);
            if (a.res && (FULL || j + i < left)) v += to_f32(rv[j + i]);
            if (FULL || j + i < left) *y = from_f32<T>(v);
            y += a.ldy;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(Q8_THREADS, 1)
    linear_q8_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Q8Args a,
                     const Q8Plan p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t full[Q8_MAX_STAGES], empty[Q8_MAX_STAGES], acc_full[2], acc_empty[2], drain;
    __shared__ __align__(16) float sx_sh[Q8_EPI][32];
    __shared__ uint32_t tmem_sh;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // the same for a warp, and known to be
    const int kb = (a.k + Q8_KB - 1) / Q8_KB;  // blocks of K, and stages of them
    const int ks = (kb + p.blocks - 1) / p.blocks;
    const int tiles = p.n_tiles * p.m_tiles;
    const uint32_t stages = p.stages;
    if (warp == 0 && lane == 0) {
        for (uint32_t s = 0; s < stages; s++) { mbar_init(&full[s], 2); mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; s++) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], Q8_EPI); }
        mbar_init(&drain, 1);
        fence_mbar_init();
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_x);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_sh, p.tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_sh;

    if (warp == 0 || warp == 2 + Q8_EPI) {
        // loads: one warp for the weights, one for the activations; issuing copies is what bounds narrow tiles
        const bool w = warp == 0;
        const CUtensorMap* map = w ? &tm_w : &tm_x;
        const uint32_t rows = w ? p.r : p.c, off = w ? 0 : p.x_off;
        uint32_t s = 0, parity = 1, issued = 0;
        bool alive = true;
        for (int t = blockIdx.x; t < tiles && alive; t += gridDim.x) {
            int tn, tm;
            p.decode(t, tn, tm);
            const int row = w ? tn * p.r : tm * p.c;
            for (int b = 0; b < kb; b += p.blocks) {
                if (!mbar_wait_warp(&empty[s], parity, &q8_err, RK_DEV_TIMEOUT_EMPTY)) { alive = false; break; }
                uint8_t* st = ring + s * p.stage + off;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&full[s], rows * Q8_KB * p.blocks);
                    tma_load_2d(st, map, &full[s], b * Q8_KB, row);  // past the end of k: zeros
                    if (p.blocks > 1) tma_load_2d(st + rows * Q8_KB, map, &full[s], (b + 1) * Q8_KB, row);
                }
                if (issued < stages) issued++;
                if (++s == stages) { s = 0; parity ^= 1; }
            }
        }
        // the last copy issued into each stage has landed (instant unless a consumer gave up)
        for (uint32_t q = 0; q < issued; q++) {
            const bool wrapped = s == 0;
            s = wrapped ? stages - 1 : s - 1;
            if (wrapped) parity ^= 1;
            mbar_wait_warp(&full[s], parity ^ 1, &q8_err, RK_DEV_TIMEOUT_DRAIN);
        }
    } else if (warp == 1) {  // products
        uint32_t s = 0, parity = 0, tl = 0;
        // descriptors count 16-byte units; shared memory ends below their 14 bits
        const uint64_t desc = sw128_kmajor_desc(smem_u32(ring), 0);
        const uint32_t desc0 = (uint32_t)desc, desc_hi = (uint32_t)(desc >> 32);
        const uint32_t w_step = p.r * Q8_KB >> 4, x_step = p.c * Q8_KB >> 4;
        bool alive = true;
        for (int t = blockIdx.x; t < tiles && alive; t += gridDim.x, tl++) {
            const uint32_t acc = tl & 1u, ru = tl >> 1;
            if (!mbar_wait_warp(&acc_empty[acc], (ru & 1u) ^ 1u, &q8_err, RK_DEV_TIMEOUT_EMPTY)) break;
            tc_fence_after();
            const uint32_t d = tmem + acc * p.acc_cols;
            uint32_t more = 0;  // the tile's first product overwrites the accumulator
            for (int b = 0; b < ks; b++) {
                if (!mbar_wait_warp(&full[s], parity, &q8_err, RK_DEV_TIMEOUT_FULL)) { alive = false; break; }
                tc_fence_after();
                const uint32_t w = desc0 + s * (p.stage >> 4), x = w + (p.x_off >> 4);
                if (elect_one()) {
                    umma_f8(d, w, x, desc_hi, p.idesc, more);
                    umma_f8(d, w + 2, x + 2, desc_hi, p.idesc, 1);  // 32 bytes on
                    umma_f8(d, w + 4, x + 4, desc_hi, p.idesc, 1);
                    umma_f8(d, w + 6, x + 6, desc_hi, p.idesc, 1);
                    if (p.blocks > 1) {
                        umma_f8(d, w + w_step, x + x_step, desc_hi, p.idesc, 1);
                        umma_f8(d, w + w_step + 2, x + x_step + 2, desc_hi, p.idesc, 1);
                        umma_f8(d, w + w_step + 4, x + x_step + 4, desc_hi, p.idesc, 1);
                        umma_f8(d, w + w_step + 6, x + x_step + 6, desc_hi, p.idesc, 1);
                    }
                    umma_commit(&empty[s]);
                }
                more = 1;
                if (++s == stages) { s = 0; parity ^= 1; }
            }
            if (elect_one()) umma_commit(&acc_full[acc]);
        }
        if (elect_one()) umma_commit(&drain);
        mbar_wait_warp(&drain, 0, &q8_err, RK_DEV_TIMEOUT_DRAIN);
        tc_fence_before();
    } else {  // epilogue: lane quarter warp % 4 = 32 output columns; the warps of a quarter share the tile's rows
        constexpr int SHARE = Q8_EPI / 4, CHUNKS = 8 / SHARE;
        const int quarter = warp & 3, part = (warp - 2) >> 2;
        float* sx_w = sx_sh[warp - 2];
        // a tile's scales and bias are fetched while the tile before it is stored (31000 x 2048 x 256 f32: 78 -> 55 us)
        float sx[CHUNKS], sw = 0.f, bias = 0.f;
        auto fetch = [&](int t) {
            if (t >= tiles) return;
            int tn, tm;
            p.decode(t, tn, tm);
            const int i = quarter * 32 + lane, n = tn * p.r + i;
            const bool n_ok = i < p.r && n < a.n;
            sw = n_ok ? a.sw[n] : 0.f;
            bias = n_ok && a.bias ? a.bias[n] : 0.f;
#pragma unroll
            for (int j = 0; j < CHUNKS; j++) {
                const int c = (part + j * SHARE) * 32 + lane;
                const long long m = (long long)tm * p.c + c;
                sx[j] = c < p.c && m < a.rows ? a.sx[m] : 0.f;
            }
        };
        fetch(blockIdx.x);
        uint32_t tl = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, tl++) {
            int tn, tm;
            p.decode(t, tn, tm);
            const int i = quarter * 32 + lane, n = tn * p.r + i;
            const bool n_ok = i < p.r && n < a.n;
            const uint32_t acc = tl & 1u, ru = tl >> 1;
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[acc], ru & 1u, &q8_err, RK_DEV_TIMEOUT_ACC))) break;
            tc_fence_after();
            const uint32_t col0 = tmem + acc * p.acc_cols + ((uint32_t)(quarter * 32) << 16);
            const long long m0 = (long long)tm * p.c;
            const int cols = quarter * 32 < p.r ? (int)min((long long)p.c, a.rows - m0) : 0;
            const float sw_t = sw, bias_t = bias;
            float sx_t[CHUNKS];
#pragma unroll
            for (int j = 0; j < CHUNKS; j++) sx_t[j] = sx[j];
            fetch(t + gridDim.x);
#pragma unroll
            for (int j = 0; j < CHUNKS; j++) {
                const int c = (part + j * SHARE) * 32, left = cols - c;
                if (left <= 0) break;  // the same for the whole warp
                __syncwarp();
                sx_w[lane] = sx_t[j];
                float v[32];
                tmem_ld32(col0 + c, v);
                __syncwarp();
                if (n_ok) {
                    if (left >= 32) store_rows<T, true>(a, m0 + c, n, 32, v, sx_w, sw_t, bias_t);
                    else store_rows<T, false>(a, m0 + c, n, left, v, sx_w, sw_t, bias_t);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, p.tmem_cols);
    }
}

// ---------------------------------------------------------------- host

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// 8-bit rows as a tensor map of boxes of 128 columns x `box` rows
bool q8_map(CUtensorMap* m, const void* base, long long ld, int rows, int cols, int box) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    if (rows == 1) ld = ((long long)cols + 15) / 16 * 16;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t boxes[2] = {Q8_KB, (cuuint32_t)box};
    cuuint32_t estr[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename K>
cudaError_t set_smem(K kernel, size_t bytes, std::atomic<uint64_t>& ready) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && ready.load(std::memory_order_acquire) >> dev & 1) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    return e;
}

struct Operands {
    const void *x, *w;
    long long ldx, ldw;
};

// Tile sizes: the least estimated time over R in steps of 8 and C in steps of 16.  Measured on B200, in clocks of a
// block of K: its four MMAs take 4 max(C / 2, 66), its bytes come at about 72 a clock and SM from L2 when all SMs
// pull.  An SM's tiles take their blocks of
// K, or their epilogues where those are longer; the last epilogue stands alone.
void plan_tiles(const Q8Args& a, int sms, Q8Plan& p) {
    const int kb = (a.k + Q8_KB - 1) / Q8_KB;
    double best = 1e300;
    for (int r = Q8_M; r >= 8; r -= 8) {
        const long long nt = ((long long)a.n + r - 1) / r;
        if (r > 8 && r - 8 >= a.n) continue;
        for (int c = 256; c >= 16; c -= 16) {
            if (c > 16 && c - 16 >= a.rows) continue;
            const long long mt = ((long long)a.rows + c - 1) / c, tiles = nt * mt;
            const long long waves = (tiles + sms - 1) / sms;
            const double mma = c > 132 ? 2.0 * c : 264.0, bytes = (r + c) * (Q8_KB / 72.0);
            const double main = kb * (mma > bytes ? mma : bytes), epi = 600.0 + 8.0 * c;
            const double t = waves * (main > epi ? main : epi) + (main < epi ? main : epi);
            if (t < best * 0.999) {
                best = t;
                p.r = r;
                p.c = c;
                p.n_tiles = (int)nt;
                p.m_tiles = (int)mt;
            }
        }
    }
    p.blocks = p.r + p.c <= 192 && kb > 1 ? 2 : 1;
    p.idesc = umma_idesc_e4m3(Q8_M, p.c);
    p.acc_cols = (uint32_t)(p.c + 31) / 32 * 32;
    p.tmem_cols = 64;
    while (p.tmem_cols < 2 * p.acc_cols) p.tmem_cols *= 2;
    p.x_off = (uint32_t)(p.blocks * p.r * Q8_KB);    // multiples of 8 rows: 1024-byte aligned
    p.stage = (uint32_t)(p.blocks * (p.r + p.c) * Q8_KB);
}

template <typename T>
cudaError_t launch(const Operands& o, const Q8Args& a, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};  // devices on which the kernel's shared memory is set
    cudaError_t e = set_smem(linear_q8_kernel<T>, Q8_SMEM, ready);
    if (e != cudaSuccess) return e;
    Q8Plan p = {};
    plan_tiles(a, sm_count(), p);
    const long long tiles = (long long)p.n_tiles * p.m_tiles;
    if (tiles > 0x7fff0000LL) return cudaErrorInvalidValue;
    CUtensorMap mw, mx;
    if (!q8_map(&mw, o.w, o.ldw, a.n, a.k, p.r) || !q8_map(&mx, o.x, o.ldx, a.rows, a.k, p.c)) return cudaErrorInvalidValue;
    // an MMA reads 128 weight rows from a block's start, past the end of the last stage where a tile has fewer
    const int last = (int)p.stage - (p.blocks - 1) * p.r * Q8_KB, over = Q8_M * Q8_KB > last ? Q8_M * Q8_KB - last : 0;
    p.stages = (Q8_SMEM - 1024 - over) / (int)p.stage;
    if (p.stages > Q8_MAX_STAGES) p.stages = Q8_MAX_STAGES;
    const int grid = tiles < sm_count() ? (int)tiles : sm_count();
    linear_q8_kernel<T><<<grid, Q8_THREADS, 1024 + over + p.stages * (int)p.stage, st>>>(mw, mx, a, p);
    return cudaSuccess;
}

}  // namespace

void* q8_err_word() {
    void* p = nullptr;
    return cudaGetSymbolAddress(&p, q8_err) == cudaSuccess ? p : nullptr;
}

}  // namespace rk

using namespace rk;

extern "C" rk_status rk_linear_q8(const void* x, long long ldx, const float* x_scale, const void* w, long long ldw,
                                  const float* w_scale, const float* bias, const void* residual, long long ldr,
                                  void* y, long long ldy, int rows, int n, int k, int dtype, void* stream) {
    const char* who = "rk_linear_q8: unsupported arguments";
    if (!dtype_ok(dtype) || !size_ok(rows, 0) || !size_ok(n, 1) || !size_ok(k, 1))
        return fail(RK_ERR_CANNOT_IMPLEMENT, who);
    if (rows == 0) return RK_OK;
    const size_t e = dtype_bytes(dtype);
    if (!x || !x_scale || !w || !w_scale || !y || !pitch_ok(ldx, rows, k) || !pitch_ok(ldw, n, k) ||
        !pitch_ok(ldy, rows, n) || (residual && !pitch_ok(ldr, rows, n)) || !aligned(x_scale, 4) ||
        !aligned(w_scale, 4) || !aligned(bias, 4) || !aligned(residual, e) || !aligned(y, e))
        return fail(RK_ERR_CANNOT_IMPLEMENT, who);
    if (!aligned(x, 16) || !aligned(w, 16) || (rows > 1 && ldx % 16) || (n > 1 && ldw % 16))
        return fail(RK_ERR_CANNOT_IMPLEMENT,
                    "rk_linear_q8: 8-bit rows start on 16-byte boundaries (base and row pitch)");
    const Operands o{x, w, ldx, ldw};
    const Q8Args a{x_scale, w_scale, bias, residual, y, ldr, ldy, rows, n, k};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t ce = dtype == RK_DTYPE_F32 ? launch<float>(o, a, st) : dtype == RK_DTYPE_F16 ? launch<__half>(o, a, st)
                                                                                             : launch<__nv_bfloat16>(o, a, st);
    const cudaError_t le = cudaGetLastError();
    if (ce == cudaSuccess) ce = le;
    return ce == cudaSuccess ? RK_OK : fail_cuda_err(RK_ERR_LAUNCH, "rk_linear_q8", ce);
}
