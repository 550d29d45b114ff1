// linear_q4.cu -- the linear layer with 4-bit weights in groups along the
// reduction, for few rows, and the quantiser that makes such weights:
//
//   y[m][n] = sum_g s[n][g] sum_{k in g} (q[n][k] - z[n][g]) x[m][k] + bias[n] + residual[m][n]
//
// Byte j of a weight row holds columns 2j (low half) and 2j + 1 (high half).
#include <cooperative_groups.h>

#include <atomic>

#include "quant.cuh"
#include "status.h"

#ifndef Q4_TARGET
#define Q4_TARGET 12
#endif
#ifndef Q4_CTAS
#define Q4_CTAS 2
#endif
namespace rk {
namespace {

constexpr int Q4_ZERO = 8;  // the zero point of weights that have none of their own

struct Q4Args {
    const void* x;
    const uint8_t* w;
    const void* s;
    const uint8_t* z;
    const float* bias;
    const void* res;
    void* y;
    long long ldx, ldw, ldr, ldy;
    int rows, n, k, group, groups, s_dtype;
    bool x_vec;  // rows of x start on 16-byte boundaries
};

// ---------------------------------------------------------------- the product
//
// Weight rows are the M = 16 side of mma.m16n8k16 and activation rows the N side, eight columns a tile.  Codes
// become 16-bit values without a conversion: a code or'ed into the mantissa of 128 (bf16) or 1024 (half) reads
// 128 + q, and 128 + z subtracted leaves the exact small integer q - z.  The sum over a group is scaled once, in 32
// bits, so nothing of scale x code is rounded.  32-bit activations are three exact bf16 parts in three columns
// whose sums are added at the end (24 bits); 16-bit ones are one column.
//
// The order of k within a matrix instruction is free, so a thread's fragment is whatever lies next to one another:
// lane (g, t) reads 4 / SUB words of rows g and g + 8, the quad t = 0..3 covering one group (SUB = 1: 128 columns in
// 16-byte loads, 2: 64 in 8-byte ones, 4: 32 in 4-byte ones).  A word's codes 0..7 come out in pairs (0, 4), (1, 5),
// (2, 6), (3, 7), and the activations lie in shared memory in that order.

template <typename T> struct Q4Type;
template <> struct Q4Type<float> { static constexpr int PARTS = 3; static constexpr bool HALF = false; };
template <> struct Q4Type<__half> { static constexpr int PARTS = 1; static constexpr bool HALF = true; };
template <> struct Q4Type<__nv_bfloat16> { static constexpr int PARTS = 1; static constexpr bool HALF = false; };

constexpr int Q4_CHUNK = 128;  // columns a warp takes at a time
constexpr int Q4_WARPS = 8;
// chunks of weights on their way to a warp's registers
__host__ __device__ constexpr int q4_ahead(int nt) { return nt <= 4 ? 4 : 2; }

template <bool HALF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (HALF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// the two codes at bits 4i and 4i + 16 of a word, less the zero point (zz: magic + z in both halves)
template <bool HALF>
__device__ __forceinline__ uint32_t q4_pair(uint32_t w, int i, uint32_t zz) {
    constexpr uint32_t magic = HALF ? 0x64006400u : 0x43004300u;
    const uint32_t v = ((w >> (4 * i)) & 0x000f000fu) | magic;
    uint32_t r;
    if (HALF) asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(zz));
    else asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(zz));
    return r;
}

template <typename T>
__device__ __forceinline__ uint16_t bits16(T v) { return *reinterpret_cast<uint16_t*>(&v); }

// x = hi + mid + lo in bf16, exactly: 8 bits of the mantissa each, cut off, so that nothing overflows
__device__ __forceinline__ void split3(float x, uint16_t (&p)[3]) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7f800000u) == 0x7f800000u) {  // infinities and NaN go whole into the first part
        p[0] = bits16(__float2bfloat16_rn(x));
        p[1] = p[2] = 0;
        return;
    }
    const float r1 = x - __uint_as_float(u & 0xffff0000u);
    const uint32_t u1 = __float_as_uint(r1);
    p[0] = (uint16_t)(u >> 16);
    p[1] = (uint16_t)(u1 >> 16);
    p[2] = bits16(__float2bfloat16_rn(r1 - __uint_as_float(u1 & 0xffff0000u)));
}

// where the 8 columns `b` of a chunk's 16 lie among its 16-byte blocks: a quad's four words side by side
template <int SUB>
__device__ __forceinline__ int q4_block(int b) {
    if (SUB == 1) return (b & 3) * 4 + (b >> 2);
    if (SUB == 2) return ((b >> 3) * 2 + (b & 1)) * 4 + ((b & 7) >> 1);
    return b;
}

// One block: wn tiles of 16 weight rows x (8 / wn) warps that share a tile's chunks; the blocks of a cluster share
// the chunks of their tiles.  Partial sums meet in shared memory, in a fixed order.
template <typename T, int SUB, int NT>
__global__ void __launch_bounds__(32 * Q4_WARPS, NT <= 4 ? 2 : 1)
    linear_q4_kernel(const Q4Args a, int wn, int stage_chunks, int row_block) {
    using Ty = Q4Type<T>;
    constexpr int PARTS = Ty::PARTS, ROWS = NT * 8 / PARTS, COLS = NT * 8;
    constexpr int WORDS = 4 / SUB, AHEAD = q4_ahead(NT);
    constexpr uint32_t MAGIC = Ty::HALF ? 0x64006400u : 0x43004300u;
    extern __shared__ __align__(16) uint8_t smem[];
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wk = Q4_WARPS / wn, kw = warp / wn;
    const int n_block = (int)(blockIdx.x / ranks) * wn * 16;
    const int n0 = n_block + (warp % wn) * 16;
    const long long m0 = ((long long)row_block + blockIdx.y) * ROWS;
    const int rows = (int)(a.rows - m0 < ROWS ? a.rows - m0 : ROWS);
    const int all = (a.k + Q4_CHUNK - 1) / Q4_CHUNK;
    const int begin = (int)((long long)all * rank / ranks), end = (int)((long long)all * (rank + 1) / ranks);
    const int steps = (end - begin + wk - 1) / wk;       // of every warp
    const int stage_steps = stage_chunks / wk;            // a multiple of AHEAD
    const int pitch = stage_chunks * 256 + 64;            // bytes of a column: conflict-free 16-byte reads
    const int row_bytes = (int)(((long long)a.k + 31) / 32 * 16);
    // rows past the last one read the last one; their sums are not stored
    const uint8_t* wp[2];
    size_t sp[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int n = n0 + g + 8 * i < a.n ? n0 + g + 8 * i : a.n - 1;
        wp[i] = a.w + (long long)n * a.ldw + t * (16 / SUB);
        sp[i] = (size_t)n * a.groups;
    }
    const int per = SUB == 1 ? a.group / Q4_CHUNK : 1;    // chunks a group, where a group is larger

    uint32_t w[AHEAD][2][4];
    float sc[AHEAD][2][SUB];
    uint32_t zz[AHEAD][2][SUB];
    auto load = [&](int step, uint32_t (&w)[2][4], float (&sc)[2][SUB], uint32_t (&zz)[2][SUB]) {
        const int c = begin + step * wk + kw;
#pragma unroll
        for (int i = 0; i < 2; i++) {
#pragma unroll
            for (int s = 0; s < SUB; s++) {
                const int off = c * 64 + s * (64 / SUB);
                const bool in = c < end && off + t * (16 / SUB) < row_bytes;
                const uint8_t* p = wp[i] + off;
                if constexpr (SUB == 1) {
                    const uint4 v = in ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
                    w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
                } else if constexpr (SUB == 2) {
                    const uint2 v = in ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0, 0);
                    w[i][2 * s] = v.x; w[i][2 * s + 1] = v.y;
                } else {
                    w[i][s] = in ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
                }
                const int gi = SUB == 1 ? (per == 1 ? c : c / per) : c * SUB + s;
                const bool gin = c < end && gi < a.groups;
                sc[i][s] = gin ? load_as_f32(a.s, sp[i] + gi, a.s_dtype) : 0.f;
                zz[i][s] = MAGIC + (gin && a.z ? a.z[sp[i] + gi] * 0x10001u : Q4_ZERO * 0x10001u);
            }
        }
    };
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
    for (int d = 0; d < AHEAD; d++) load(d, w[d], sc[d], zz[d]);

    for (int step0 = 0; step0 < steps; step0 += AHEAD) {
        if (step0 % stage_steps == 0) {
            // the activations of the next chunks, 8 columns at a time
            if (step0) __syncthreads();
            const int c0 = begin + step0 * wk, nc = min(stage_chunks, end - c0);
            for (int u = threadIdx.x; u < rows * nc * 16; u += 32 * Q4_WARPS) {
                const int m = u / (nc * 16), b = u - m * (nc * 16);
                const long long col = (long long)c0 * Q4_CHUNK + b * 8;
                const T* x = static_cast<const T*>(a.x) + (m0 + m) * a.ldx + col;
                T v[8];
                if (a.x_vec && col + 8 <= a.k) {
                    struct alignas(16) Q { T v[16 / sizeof(T)]; };
#pragma unroll
                    for (int i = 0; i < 8; i += 16 / sizeof(T)) *reinterpret_cast<Q*>(v + i) = *reinterpret_cast<const Q*>(x + i);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = col + i < a.k ? x[i] : from_f32<T>(0.f);
                }
                uint16_t p[8][3];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if constexpr (PARTS == 3) split3(v[i], p[i]);
                    else p[i][0] = bits16(v[i]);
                }
                uint8_t* dst = smem + (size_t)m * PARTS * pitch + ((b >> 4) * 16 + q4_block<SUB>(b & 15)) * 16;
#pragma unroll
                for (int q = 0; q < PARTS; q++)
                    *reinterpret_cast<uint4*>(dst + (size_t)q * pitch) =
                        make_uint4(p[0][q] | (uint32_t)p[4][q] << 16, p[1][q] | (uint32_t)p[5][q] << 16,
                                   p[2][q] | (uint32_t)p[6][q] << 16, p[3][q] | (uint32_t)p[7][q] << 16);
            }
            __syncthreads();
        }
#pragma unroll
        for (int d = 0; d < AHEAD; d++) {
            const int step = step0 + d;
            if (begin + step * wk + kw < end) {  // the same for the whole warp
                const uint8_t* xb = smem + (size_t)g * pitch + ((step % stage_steps) * wk + kw) * 256 + t * 16;
#pragma unroll
                for (int s = 0; s < SUB; s++) {
                    float part[NT][4];
#pragma unroll
                    for (int j = 0; j < NT; j++) part[j][0] = part[j][1] = part[j][2] = part[j][3] = 0.f;
#pragma unroll
                    for (int q = s * WORDS; q < (s + 1) * WORDS; q++) {
                        uint32_t f0[4], f1[4];
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            f0[i] = q4_pair<Ty::HALF>(w[d][i][q], 0, zz[d][i][s]);
                            f0[i + 2] = q4_pair<Ty::HALF>(w[d][i][q], 1, zz[d][i][s]);
                            f1[i] = q4_pair<Ty::HALF>(w[d][i][q], 2, zz[d][i][s]);
                            f1[i + 2] = q4_pair<Ty::HALF>(w[d][i][q], 3, zz[d][i][s]);
                        }
#pragma unroll
                        for (int j = 0; j < NT; j++) {
                            const uint4 b = *reinterpret_cast<const uint4*>(xb + (size_t)j * 8 * pitch + q * 64);
                            mma16816<Ty::HALF>(part[j], f0, b.x, b.y);
                            mma16816<Ty::HALF>(part[j], f1, b.z, b.w);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        acc[j][0] += sc[d][0][s] * part[j][0];
                        acc[j][1] += sc[d][0][s] * part[j][1];
                        acc[j][2] += sc[d][1][s] * part[j][2];
                        acc[j][3] += sc[d][1][s] * part[j][3];
                    }
                }
            }
            load(step + AHEAD, w[d], sc[d], zz[d]);
        }
    }

    // partial sums: red[warp][COLS][16 rows], then over the warps of a tile, then over the cluster's blocks
    float* red = reinterpret_cast<float*>(smem);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NT; j++) {
        float* r = red + ((size_t)warp * COLS + j * 8 + 2 * t) * 17 + g;
        r[0] = acc[j][0];
        r[17] = acc[j][1];
        r[8] = acc[j][2];
        r[25] = acc[j][3];
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    // block `rank` finishes its share of the outputs
    const int outs = rows * wn * 16;
    for (int u = rank * 32 * Q4_WARPS + threadIdx.x; u < outs; u += ranks * 32 * Q4_WARPS) {
        const int m = u / (wn * 16), i = u - m * (wn * 16);
        const int n = n_block + i;
        if (n >= a.n) continue;
        float v = 0.f;
        for (int b = 0; b < ranks; b++) {
            const float* rb = ranks > 1 ? cluster.map_shared_rank(red, b) : red;
#pragma unroll
            for (int q = PARTS - 1; q >= 0; q--)
                for (int k = 0; k < wk; k++)
                    v += rb[((size_t)(k * wn + (i >> 4)) * COLS + m * PARTS + q) * 17 + (i & 15)];
        }
        if (a.bias) v += a.bias[n];
        if (a.res) v += to_f32(static_cast<const T*>(a.res)[(m0 + m) * a.ldr + n]);
        static_cast<T*>(a.y)[(m0 + m) * a.ldy + n] = from_f32<T>(v);
    }
    if (ranks > 1) cluster.sync();  // no block leaves while another reads its sums
}

constexpr int Q4_SMEM = 200 * 1024;

template <typename T, int SUB, int NT>
cudaError_t launch_nt(const Q4Args& a, cudaStream_t st) {
    auto kernel = linear_q4_kernel<T, SUB, NT>;
    static std::atomic<uint64_t> ready{0};  // devices on which the kernel's shared memory is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4_SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    constexpr int PARTS = Q4Type<T>::PARTS, ROWS = NT * 8 / PARTS;
    const int tiles = (a.n + 15) / 16, chunks = (a.k + Q4_CHUNK - 1) / Q4_CHUNK;
    const int target = Q4_TARGET * sm_count();  // warps with work of their own
    int wn = Q4_WARPS;
    constexpr int AHEAD = q4_ahead(NT), COLS = NT * 8;
    auto stage_bytes = [&](int chunks_) { return COLS * (chunks_ * 256 + 64); };
    while (wn > 1 && (long long)tiles * (Q4_WARPS / wn) < target && Q4_WARPS / wn * 2 <= chunks &&
           stage_bytes(Q4_WARPS / wn * 2 * AHEAD) <= Q4_SMEM)
        wn /= 2;
    const int wk = Q4_WARPS / wn, unit = wk * AHEAD;
    const int groups_n = (tiles + wn - 1) / wn;
    int ranks = 1;
    while (ranks < 8 && (long long)groups_n * ranks * 2 <= Q4_CTAS * sm_count() && chunks >= ranks * 2 * unit) ranks *= 2;
    // activations of `stage` chunks at a time; two blocks an SM where their registers allow it
    const int mine = (chunks + ranks - 1) / ranks;
    int stage = (mine + unit - 1) / unit * unit;
    while (stage > unit && stage_bytes(stage) > (NT <= 4 ? Q4_SMEM / 2 : Q4_SMEM)) stage -= unit;
    size_t smem = (size_t)stage_bytes(stage);
    const size_t red = (size_t)Q4_WARPS * NT * 8 * 17 * 4;
    if (smem < red) smem = red;
    if (smem > Q4_SMEM) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(groups_n * ranks);
    cfg.blockDim = dim3(32 * Q4_WARPS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const int blocks = (int)(((long long)a.rows + ROWS - 1) / ROWS);
    for (int b = 0; b < blocks; b += 65535) {  // row blocks are the grid's second dimension
        cfg.gridDim.y = blocks - b < 65535 ? blocks - b : 65535;
        e = cudaLaunchKernelEx(&cfg, kernel, a, wn, stage, b);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

template <typename T, int SUB>
cudaError_t launch_sub(const Q4Args& a, cudaStream_t st) {
    if constexpr (Q4Type<T>::PARTS == 3) {
        if (a.rows <= 2) return launch_nt<T, SUB, 1>(a, st);
        if (a.rows <= 5) return launch_nt<T, SUB, 2>(a, st);
        if (a.rows <= 8) return launch_nt<T, SUB, 3>(a, st);
        if (a.rows <= 16) return launch_nt<T, SUB, 6>(a, st);
        if (a.rows <= 24) return launch_nt<T, SUB, 9>(a, st);
        return launch_nt<T, SUB, 12>(a, st);
    } else {
        if (a.rows <= 8) return launch_nt<T, SUB, 1>(a, st);
        if (a.rows <= 16) return launch_nt<T, SUB, 2>(a, st);
        if (a.rows <= 32) return launch_nt<T, SUB, 4>(a, st);
        return launch_nt<T, SUB, 8>(a, st);
    }
}

template <typename T>
cudaError_t launch(const Q4Args& a, cudaStream_t st) {
    if (a.group == 32) return launch_sub<T, 4>(a, st);
    if (a.group == 64) return launch_sub<T, 2>(a, st);
    return launch_sub<T, 1>(a, st);
}

// largest finite value of a scale's type
__device__ __forceinline__ float store_scale(void* p, size_t i, float s, int dtype) {
    if (dtype == RK_DTYPE_F32) {
        static_cast<float*>(p)[i] = s;
        return s;
    }
    if (dtype == RK_DTYPE_F16) {
        const __half h = __float2half_rn(fminf(s, 65504.f));
        static_cast<__half*>(p)[i] = h;
        return __half2float(h);
    }
    const __nv_bfloat16 b = __float2bfloat16_rn(fminf(s, 3.3895313892515355e38f));
    static_cast<__nv_bfloat16*>(p)[i] = b;
    return __bfloat162float(b);
}

// One warp per (row, group).  With zero points the codes 0..15 span
// [min(w, 0), max(w, 0)]; without, s = max|w| / 7 around code 8.  Codes are
// chosen for the scale as it is stored.  Each lane writes whole bytes; columns
// past k get code 0 in the rest of the row's last 16 bytes.
template <typename T>
__global__ void __launch_bounds__(256)
    quantize_q4_kernel(const T* w, long long ldw, uint8_t* q, long long ldq, void* s_out, uint8_t* z_out, int n,
                       int k, int group, int groups, int s_dtype) {
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const long long row = unit / groups;
    const int g = (int)(unit - row * groups);
    if (row >= n) return;
    const T* src = w + row * ldw;
    const int k0 = g * group, k1 = k0 + group < k ? k0 + group : k;
    float lo = 0.f, hi = 0.f;
    for (int c = k0 + lane; c < k1; c += 32) {
        const float v = to_f32(src[c]);
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
    }
    for (int o = 16; o; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    // both ends halved first: their difference may pass the largest float
    float s = z_out ? (hi * 0.5f - lo * 0.5f) / 7.5f : fmaxf(hi, -lo) / 7.f;
    int z = Q4_ZERO;
    if (lane == 0) s = store_scale(s_out, (size_t)unit, s, s_dtype);
    s = __shfl_sync(0xffffffffu, s, 0);
    if (z_out) {
        z = s > 0.f ? (int)fminf(fmaxf(rintf(-lo / s), 0.f), 15.f) : 0;
        if (lane == 0) z_out[unit] = (uint8_t)z;
    }
    const int end = g == groups - 1 ? (k + 31) / 32 * 32 : k1;  // the last group also fills the row's pad
    for (int c = k0 + 2 * lane; c < end; c += 64) {
        int code[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            code[j] = 0;
            if (c + j < k1) {
                const float v = s > 0.f ? rintf(to_f32(src[c + j]) / s) + (float)z : (float)z;
                code[j] = (int)fminf(fmaxf(v, 0.f), 15.f);
            }
        }
        q[row * ldq + (c >> 1)] = (uint8_t)(code[0] | code[1] << 4);
    }
}

bool group_ok(int group) { return group == 32 || group == 64 || (group >= 128 && group % 128 == 0); }

}  // namespace
}  // namespace rk

using namespace rk;

extern "C" rk_status rk_linear_q4(const void* x, long long ldx, const void* w, long long ldw, const void* scales,
                                  const uint8_t* zeros, const float* bias, const void* residual, long long ldr,
                                  void* y, long long ldy, int rows, int n, int k, int group, int dtype,
                                  int scale_dtype, void* stream) {
    const char* who = "rk_linear_q4: unsupported arguments";
    if (!dtype_ok(dtype) || !dtype_ok(scale_dtype) || rows < 0 || n < 1 || k < 1) return fail(RK_ERR_CANNOT_IMPLEMENT, who);
    if (!group_ok(group))
        return fail(RK_ERR_CANNOT_IMPLEMENT, "rk_linear_q4: groups are of 32, 64 or a multiple of 128 columns");
    if (rows == 0) return RK_OK;
    const size_t e = dtype_bytes(dtype);
    const long long row_bytes = ((long long)k + 31) / 32 * 16;
    if (!x || !w || !scales || !y || !pitch_ok(ldx, rows, k) || !pitch_ok(ldy, rows, n) ||
        (residual && !pitch_ok(ldr, rows, n)) || !aligned(x, e) || !aligned(y, e) || !aligned(residual, e) ||
        !aligned(bias, 4) || !aligned(scales, dtype_bytes(scale_dtype)))
        return fail(RK_ERR_CANNOT_IMPLEMENT, who);
    if (!aligned(w, 16) || (n > 1 && (ldw % 16 || ldw < row_bytes)))
        return fail(RK_ERR_CANNOT_IMPLEMENT,
                    "rk_linear_q4: weight rows hold ceil(k / 32) x 16 bytes and start on 16-byte boundaries");
    Q4Args a{x, static_cast<const uint8_t*>(w), scales, zeros, bias, residual, y, ldx, ldw, ldr, ldy, rows, n, k,
             group, (int)(((long long)k + group - 1) / group), scale_dtype,
             aligned(x, 16) && (rows == 1 || ldx * (long long)e % 16 == 0)};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t ce = dtype == RK_DTYPE_F32 ? launch<float>(a, st) : dtype == RK_DTYPE_F16 ? launch<__half>(a, st)
                                                                                          : launch<__nv_bfloat16>(a, st);
    const cudaError_t le = cudaGetLastError();
    if (ce == cudaSuccess) ce = le;
    return ce == cudaSuccess ? RK_OK : fail_cuda_err(RK_ERR_LAUNCH, "rk_linear_q4", ce);
}

extern "C" rk_status rk_quantize_q4(const void* w, long long ldw, void* q, long long ldq, void* scales,
                                    uint8_t* zeros, int n, int k, int group, int dtype, int scale_dtype,
                                    void* stream) {
    const char* who = "rk_quantize_q4: unsupported arguments";
    if (!dtype_ok(dtype) || !dtype_ok(scale_dtype) || n < 0 || k < 1) return fail(RK_ERR_CANNOT_IMPLEMENT, who);
    if (!group_ok(group))
        return fail(RK_ERR_CANNOT_IMPLEMENT, "rk_quantize_q4: groups are of 32, 64 or a multiple of 128 columns");
    if (n == 0) return RK_OK;
    const long long row_bytes = ((long long)k + 31) / 32 * 16;
    if (!w || !q || !scales || !pitch_ok(ldw, n, k) || !aligned(w, dtype_bytes(dtype)) ||
        !aligned(scales, dtype_bytes(scale_dtype)) || !aligned(q, 16) || (n > 1 && (ldq % 16 || ldq < row_bytes)))
        return fail(RK_ERR_CANNOT_IMPLEMENT, who);
    const int groups = (int)(((long long)k + group - 1) / group);
    const long long blocks = ((long long)n * groups + 7) / 8;
    if (blocks > 0x7fffffffLL) return fail(RK_ERR_CANNOT_IMPLEMENT, "rk_quantize_q4: too many groups for one launch");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int b = (int)blocks;
    uint8_t* qo = static_cast<uint8_t*>(q);
    switch (dtype) {
        case RK_DTYPE_F32:
            quantize_q4_kernel<float><<<b, 256, 0, st>>>(static_cast<const float*>(w), ldw, qo, ldq, scales, zeros, n,
                                                         k, group, groups, scale_dtype);
            break;
        case RK_DTYPE_F16:
            quantize_q4_kernel<__half><<<b, 256, 0, st>>>(static_cast<const __half*>(w), ldw, qo, ldq, scales, zeros,
                                                          n, k, group, groups, scale_dtype);
            break;
        default:
            quantize_q4_kernel<__nv_bfloat16><<<b, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(w), ldw, qo, ldq,
                                                                 scales, zeros, n, k, group, groups, scale_dtype);
            break;
    }
    const cudaError_t ce = cudaGetLastError();
    return ce == cudaSuccess ? RK_OK : fail_cuda_err(RK_ERR_LAUNCH, "rk_quantize_q4", ce);
}
