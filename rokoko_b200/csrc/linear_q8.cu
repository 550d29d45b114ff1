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
// Two forms:
//   tiles   one persistent block an SM, 128 x BN tiles, two accumulators, so
//           that a tile's epilogue runs beside the next tile's products
//   split   few tiles: the blocks of a cluster share a tile's K and add up
//           their accumulators through each other's shared memory, in rank
//           order; many loads in flight, the weights' bytes are the cost
#include <cooperative_groups.h>
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

constexpr int Q8_M = 128;          // weight rows of a tile
constexpr int Q8_KB = 128;         // bytes of K a stage holds
constexpr int Q8_W_BYTES = Q8_M * Q8_KB;
constexpr int Q8_MAX_STAGES = 12;
constexpr size_t Q8_SMEM = 225 * 1024;
constexpr size_t Q8_SPLIT_SMEM = 112 * 1024;  // two blocks an SM

__host__ __device__ constexpr uint32_t stage_bytes(int bn) { return Q8_W_BYTES + bn * Q8_KB; }

// one output: scales, bias, residual, the one rounding
template <typename T>
__device__ __forceinline__ void store_out(const Q8Args& a, long long m, int n, float acc, float sx, float sw, float bias) {
    float v = acc * (sx * sw) + bias;
    if (a.res) v += to_f32(static_cast<const T*>(a.res)[m * a.ldr + n]);
    static_cast<T*>(a.y)[m * a.ldy + n] = from_f32<T>(v);
}

// the MMAs of one stage
template <int BN>
__device__ __forceinline__ void stage_mma(uint32_t d, const uint8_t* st, bool accumulate) {
    constexpr uint32_t idesc = umma_idesc_e4m3(Q8_M, BN);
    const uint32_t w = smem_u32(st), x = w + Q8_W_BYTES;
#pragma unroll
    for (int kk = 0; kk < Q8_KB / 32; kk++)
        umma_f8(d, sw128_kmajor_desc(w + kk * 32, 0), sw128_kmajor_desc(x + kk * 32, 0), idesc,
                accumulate || kk > 0 ? 1u : 0u);
}

// Tiles in panels of 8 column tiles, row tiles fastest within a panel's column
// block: the blocks at work at a time share their operands' rows in L2.
struct Q8Tiles {
    int n_tiles, m_tiles;
    __device__ void decode(int t, int& tn, int& tm) const {
        constexpr int PANEL = 8;
        const int per = PANEL * m_tiles, p = t / per, r = t - p * per;
        const int width = min(PANEL, n_tiles - p * PANEL);
        tm = r / width;
        tn = p * PANEL + r - tm * width;
    }
};

template <typename T, int BN>
__global__ void __launch_bounds__(320, 1)
    q8_tiles_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Q8Args a,
                    int stages) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t full[Q8_MAX_STAGES], empty[Q8_MAX_STAGES], acc_full[2], acc_empty[2], drain;
    __shared__ uint32_t tmem_sh;
    __shared__ int dead;
    constexpr uint32_t STAGE = stage_bytes(BN), COLS = 2 * BN < 32 ? 32 : 2 * BN;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kb = (a.k + Q8_KB - 1) / Q8_KB;
    const Q8Tiles g{(a.n + Q8_M - 1) / Q8_M, (a.rows + BN - 1) / BN};
    const int tiles = g.n_tiles * g.m_tiles;
    if (warp == 0 && lane == 0) {
        for (int s = 0; s < stages; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; s++) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 8); }
        mbar_init(&drain, 1);
        dead = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_x);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_sh, COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_sh;

    if (warp == 0) {
        if (lane == 0) {  // loads
            uint32_t i = 0;
            bool alive = true;
            for (int t = blockIdx.x; t < tiles && alive; t += gridDim.x) {
                int tn, tm;
                g.decode(t, tn, tm);
                for (int b = 0; b < kb; b++, i++) {
                    const uint32_t s = i % stages, r = i / stages;
                    if (!mbar_wait(&empty[s], (r & 1u) ^ 1u, &q8_err, RK_DEV_TIMEOUT_EMPTY)) { alive = false; break; }
                    uint8_t* st = ring + (size_t)s * STAGE;
                    mbar_arrive_expect_tx(&full[s], STAGE);
                    tma_load_2d(st, &tm_w, &full[s], b * Q8_KB, tn * Q8_M);
                    tma_load_2d(st + Q8_W_BYTES, &tm_x, &full[s], b * Q8_KB, tm * BN);
                }
            }
            for (uint32_t q = i > (uint32_t)stages ? i - stages : 0u; q < i; q++)
                mbar_wait(&full[q % stages], (q / stages) & 1u, &q8_err, RK_DEV_TIMEOUT_DRAIN);
        }
    } else if (warp == 1) {
        if (lane == 0) {  // products
            uint32_t i = 0, tl = 0;
            bool alive = true;
            for (int t = blockIdx.x; t < tiles && alive; t += gridDim.x, tl++) {
                const uint32_t acc = tl & 1u, ru = tl >> 1;
                if (!mbar_wait(&acc_empty[acc], (ru & 1u) ^ 1u, &q8_err, RK_DEV_TIMEOUT_EMPTY)) break;
                tc_fence_after();
                for (int b = 0; b < kb; b++, i++) {
                    const uint32_t s = i % stages, r = i / stages;
                    if (!mbar_wait(&full[s], r & 1u, &q8_err, RK_DEV_TIMEOUT_FULL)) { alive = false; break; }
                    tc_fence_after();
                    stage_mma<BN>(tmem + acc * BN, ring + (size_t)s * STAGE, b > 0);
                    umma_commit(&empty[s]);
                }
                umma_commit(&acc_full[acc]);
            }
            umma_commit(&drain);
            mbar_wait(&drain, 0, &q8_err, RK_DEV_TIMEOUT_DRAIN);
            tc_fence_before();
        }
    } else {  // epilogue: lane quarter warp % 4 = 32 output columns; two warps of a quarter share the tile's rows
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint32_t tl = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, tl++) {
            int tn, tm;
            g.decode(t, tn, tm);
            const int n = tn * Q8_M + quarter * 32 + lane;
            const bool n_ok = n < a.n;
            const float sw = n_ok ? a.sw[n] : 0.f, bias = n_ok && a.bias ? a.bias[n] : 0.f;
            const uint32_t acc = tl & 1u, ru = tl >> 1;
            const bool ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[acc], ru & 1u, &q8_err, RK_DEV_TIMEOUT_ACC));
            tc_fence_after();
            if (!ok && lane == 0) dead = 1;
            const uint32_t col0 = tmem + acc * BN + ((uint32_t)(quarter * 32) << 16);
            const int m0 = tm * BN;
            for (int c = half * 32; c < BN && ok; c += 64) {
                const int left = a.rows - m0 - c;
                if (left <= 0) break;
                const float sx = lane < left ? a.sx[m0 + c + lane] : 0.f;
                float v[32];
                tmem_ld32(col0 + c, v);
                if (left >= 32) {
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        const float s = __shfl_sync(0xffffffffu, sx, j);
                        if (n_ok) store_out<T>(a, (long long)m0 + c + j, n, v[j], s, sw, bias);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        const float s = __shfl_sync(0xffffffffu, sx, j);
                        if (n_ok && j < left) store_out<T>(a, (long long)m0 + c + j, n, v[j], s, sw, bias);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);
            asm volatile("bar.sync 1, 256;" ::: "memory");  // all epilogue warps, whatever happened above
            if (dead) break;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, COLS);
    }
}

// One tile per cluster; block `rank` of it sums its share of the K blocks.
template <typename T, int BN>
__global__ void __launch_bounds__(192)
    q8_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Q8Args a,
                    int stages) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t full[Q8_MAX_STAGES], empty[Q8_MAX_STAGES], acc_full;
    __shared__ uint32_t tmem_sh;
    constexpr uint32_t STAGE = stage_bytes(BN), COLS = BN < 32 ? 32 : BN;
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x / ranks, n_tiles = (a.n + Q8_M - 1) / Q8_M;
    const int tn = tile % n_tiles, tm = tile / n_tiles;
    const int kb = (a.k + Q8_KB - 1) / Q8_KB;
    const int b0 = (int)((long long)kb * rank / ranks), b1 = (int)((long long)kb * (rank + 1) / ranks);
    if (warp == 0 && lane == 0) {
        for (int s = 0; s < stages; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(&acc_full, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_sh, COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_sh;
    float* red = reinterpret_cast<float*>(ring);  // [BN][128], once the ring is done with
    if (warp == 0) {
        if (lane == 0) {
            int i = 0;
            for (int b = b0; b < b1; b++, i++) {
                const int s = i % stages, r = i / stages;
                if (!mbar_wait(&empty[s], (r & 1) ^ 1, &q8_err, RK_DEV_TIMEOUT_EMPTY)) break;
                uint8_t* st = ring + (size_t)s * STAGE;
                mbar_arrive_expect_tx(&full[s], STAGE);
                tma_load_2d(st, &tm_w, &full[s], b * Q8_KB, tn * Q8_M);
                tma_load_2d(st + Q8_W_BYTES, &tm_x, &full[s], b * Q8_KB, tm * BN);
            }
            for (int q = i > stages ? i - stages : 0; q < i; q++)
                mbar_wait(&full[q % stages], (q / stages) & 1, &q8_err, RK_DEV_TIMEOUT_DRAIN);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int i = 0;
            for (int b = b0; b < b1; b++, i++) {
                const int s = i % stages, r = i / stages;
                if (!mbar_wait(&full[s], r & 1, &q8_err, RK_DEV_TIMEOUT_FULL)) break;
                tc_fence_after();
                stage_mma<BN>(tmem, ring + (size_t)s * STAGE, i > 0);
                umma_commit(&empty[s]);
            }
            umma_commit(&acc_full);  // lands when every product above is done
        }
    }
    __syncwarp();
    // every warp: the accumulator is complete, and with it all reads of the ring
    const bool ok = __all_sync(0xffffffffu, mbar_wait(&acc_full, 0, &q8_err, RK_DEV_TIMEOUT_ACC));
    tc_fence_after();
    __syncthreads();
    const int cols = min(BN, a.rows - tm * BN);
    if (warp >= 2) {
        const int quarter = warp & 3;
        const uint32_t col0 = tmem + ((uint32_t)(quarter * 32) << 16);
        for (int c = 0; c < cols; c += 16) {
            float v[16];
            tmem_ld16(col0 + c, v);
#pragma unroll
            for (int j = 0; j < 16; j++) red[(c + j) * Q8_M + quarter * 32 + lane] = v[j];
        }
        tc_fence_before();
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    for (int u = threadIdx.x; u < (cols - rank + ranks - 1) / ranks * Q8_M; u += 192) {
        const int c = u / Q8_M * ranks + rank, i = u % Q8_M;
        const int n = tn * Q8_M + i;
        if (n >= a.n || !ok) continue;
        float v = 0.f;
        if (ranks > 1) {
            for (int b = 0; b < ranks; b++) v += cluster.map_shared_rank(red, b)[c * Q8_M + i];
        } else {
            v = red[c * Q8_M + i];
        }
        const long long m = (long long)tm * BN + c;
        store_out<T>(a, m, n, v, a.sx[m], a.sw[n], a.bias ? a.bias[n] : 0.f);
    }
    if (ranks > 1) cluster.sync();  // no block leaves while another reads its sums
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, COLS);
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

template <typename T, int BN>
cudaError_t launch_tiles(const Operands& o, const Q8Args& a, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};  // devices on which the kernel's shared memory is set
    cudaError_t e = set_smem(q8_tiles_kernel<T, BN>, Q8_SMEM, ready);
    if (e != cudaSuccess) return e;
    CUtensorMap mw, mx;
    if (!q8_map(&mw, o.w, o.ldw, a.n, a.k, Q8_M) || !q8_map(&mx, o.x, o.ldx, a.rows, a.k, BN)) return cudaErrorInvalidValue;
    int stages = (int)((Q8_SMEM - 1024) / stage_bytes(BN));
    if (stages > Q8_MAX_STAGES) stages = Q8_MAX_STAGES;
    const long long tiles = ((long long)a.n + Q8_M - 1) / Q8_M * (((long long)a.rows + BN - 1) / BN);
    if (tiles > 0x7fff0000LL) return cudaErrorInvalidValue;
    const int grid = tiles < sm_count() ? (int)tiles : sm_count();
    q8_tiles_kernel<T, BN><<<grid, 320, 1024 + stages * stage_bytes(BN), st>>>(mw, mx, a, stages);
    return cudaSuccess;
}

template <typename T, int BN>
cudaError_t launch_split(const Operands& o, const Q8Args& a, int ranks, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};  // devices on which the kernel's shared memory is set
    cudaError_t e = set_smem(q8_split_kernel<T, BN>, Q8_SPLIT_SMEM, ready);
    if (e != cudaSuccess) return e;
    CUtensorMap mw, mx;
    if (!q8_map(&mw, o.w, o.ldw, a.n, a.k, Q8_M) || !q8_map(&mx, o.x, o.ldx, a.rows, a.k, BN)) return cudaErrorInvalidValue;
    int stages = (int)((Q8_SPLIT_SMEM - 1024) / stage_bytes(BN));
    if (stages > Q8_MAX_STAGES) stages = Q8_MAX_STAGES;
    const int tiles = (a.n + Q8_M - 1) / Q8_M * ((a.rows + BN - 1) / BN);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * ranks);
    cfg.blockDim = dim3(192);
    cfg.dynamicSmemBytes = 1024 + stages * stage_bytes(BN);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, q8_split_kernel<T, BN>, mw, mx, a, stages);
}

template <typename T>
cudaError_t launch(const Operands& o, const Q8Args& a, cudaStream_t st) {
    const int sms = sm_count(), kb = (a.k + Q8_KB - 1) / Q8_KB;
    const long long nt = ((long long)a.n + Q8_M - 1) / Q8_M;
    const int bn = a.rows <= 16 ? 16 : a.rows <= 32 ? 32 : a.rows <= 64 ? 64 : 128;
    const long long tiles = nt * (((long long)a.rows + bn - 1) / bn);
    if (tiles <= sms) {
        int ranks = 1;
        while (ranks < 8 && tiles * ranks * 2 <= 2 * sms && kb >= ranks * 2) ranks *= 2;
        switch (bn) {
            case 16: return launch_split<T, 16>(o, a, ranks, st);
            case 32: return launch_split<T, 32>(o, a, ranks, st);
            case 64: return launch_split<T, 64>(o, a, ranks, st);
            default: return launch_split<T, 128>(o, a, ranks, st);
        }
    }
    if (a.rows <= 64) return launch_tiles<T, 64>(o, a, st);
    if (a.rows <= 128) return launch_tiles<T, 128>(o, a, st);
    return launch_tiles<T, 256>(o, a, st);
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
    if (!dtype_ok(dtype) || rows < 0 || n < 1 || k < 1) return fail(RK_ERR_CANNOT_IMPLEMENT, who);
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
