// linear_q4.cu -- the linear layer with 4-bit weights in groups along the
// reduction, for few rows, and the quantiser that makes such weights:
//
//   y[m][n] = sum_g s[n][g] sum_{k in g} (q[n][k] - z[n][g]) x[m][k] + bias[n] + residual[m][n]
//
// Byte j of a weight row holds columns 2j (low half) and 2j + 1 (high half).
#include <atomic>

#include "quant.cuh"
#include "status.h"

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

// Warps of a block and chunks of weights on their way to a warp's registers: what 64 K registers hold.
__host__ __device__ constexpr int q4_warps(int nt) { return nt <= 4 ? 16 : 8; }
__host__ __device__ constexpr int q4_ahead(int nt) { return nt <= 2 ? 4 : 2; }

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
    const uint32_t mask = 0x000f000fu, magic = HALF ? 0x64006400u : 0x43004300u;
    uint32_t v, r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(w >> (4 * i)), "r"(mask), "r"(magic));  // (w & mask) | magic
    if (HALF) asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(zz));
    else asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(zz));
    return r;
}

template <typename T>
__device__ __forceinline__ uint16_t bits16(T v) { return *reinterpret_cast<uint16_t*>(&v); }

// x = hi + mid + lo in bf16, exactly: 8 bits of the mantissa each, cut off, so that nothing overflows.  Infinities and
// NaN go whole into the first part.
__device__ __forceinline__ void split3(float x, uint32_t (&p)[3]) {
    const uint32_t u = __float_as_uint(x);
    const bool finite = (u & 0x7f800000u) != 0x7f800000u;
    const float r1 = finite ? x - __uint_as_float(u & 0xffff0000u) : 0.f;
    const uint32_t u1 = __float_as_uint(r1);
    p[0] = u >> 16 | (!finite && (u & 0x007fffffu) ? 0x40u : 0u);
    p[1] = u1 >> 16;
    p[2] = bits16(__float2bfloat16_rn(r1 - __uint_as_float(u1 & 0xffff0000u)));
}

// Eight columns of a row as the 16-byte blocks of their parts: the pairs (0, 4), (1, 5), (2, 6), (3, 7).
template <typename T>
__device__ __forceinline__ void q4_blocks(const T* x, long long left, bool vec, uint4 (&out)[Q4Type<T>::PARTS]) {
    if constexpr (sizeof(T) == 4) {
        float v[8];
        if (vec && left >= 8) {
            *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(x);
            *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(x + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = i < left ? x[i] : 0.f;
        }
        uint32_t p[8][3];
#pragma unroll
        for (int i = 0; i < 8; i++) split3(v[i], p[i]);
#pragma unroll
        for (int q = 0; q < 3; q++)
            out[q] = make_uint4(p[0][q] | p[4][q] << 16, p[1][q] | p[5][q] << 16, p[2][q] | p[6][q] << 16,
                                p[3][q] | p[7][q] << 16);
    } else {
        uint4 v;
        if (vec && left >= 8) {
            v = *reinterpret_cast<const uint4*>(x);
        } else {
            uint32_t e[8];
#pragma unroll
            for (int i = 0; i < 8; i++) e[i] = i < left ? bits16(x[i]) : 0u;
            v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
        out[0] = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                            __byte_perm(v.y, v.w, 0x7632));
    }
}

// where the 8 columns `b` of a chunk's 16 lie among its 16-byte blocks: a quad's four words side by side
template <int SUB>
__device__ __forceinline__ int q4_block(int b) {
    if (SUB == 1) return (b & 3) * 4 + (b >> 2);
    if (SUB == 2) return ((b >> 3) * 2 + (b & 1)) * 4 + ((b & 7) >> 1);
    return b;
}

// How a launch is divided, the same for all of its blocks.
struct Q4Plan {
    int wn;          // tiles of 16 weight rows a block works on at a time; the warps of a tile share its chunks
    int rows;        // most weight rows of a block
    int stage;       // chunks whose activations and scales lie in shared memory at a time
    int pitch;       // bytes of a column's activations there, 64 mod 128: reads meet no bank twice
    int s_pitch;     // scales of a weight row there (odd)
    int s_off, z_off, out_off, red_off;  // shared memory: activations, scales, zero points, sums, partial sums
    int row_block;   // first block of activation rows
};

// One block an SM, each with its share of the weight rows (as even as whole rows allow, tiles of 16 at a time, the
// last one short) over the whole of k: every weight is read once, by one warp, and the sums never leave the block.
// The next tiles' weights are on their way while a tile's partial sums meet in shared memory, in a fixed order.
template <typename T, int SUB, int NT>
__global__ void __launch_bounds__(32 * q4_warps(NT), 1) linear_q4_kernel(const Q4Args a, const Q4Plan p) {
    using Ty = Q4Type<T>;
    constexpr int PARTS = Ty::PARTS, ROWS = NT * 8 / PARTS;
    constexpr int WORDS = 4 / SUB, WARPS = q4_warps(NT), THREADS = 32 * WARPS, AHEAD = q4_ahead(NT);
    constexpr uint32_t MAGIC = Ty::HALF ? 0x6400u : 0x4300u;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wn = p.wn, wk = WARPS / wn, kw = warp / wn, tile = warp % wn;
    const int n0 = (int)((long long)a.n * blockIdx.x / gridDim.x);
    const int n1 = (int)((long long)a.n * (blockIdx.x + 1) / gridDim.x);
    const long long m0 = ((long long)p.row_block + blockIdx.y) * ROWS;
    const int rows = (int)(a.rows - m0 < ROWS ? a.rows - m0 : ROWS), cols = rows * PARTS;
    const int all = (a.k + Q4_CHUNK - 1) / Q4_CHUNK;
    const int row_bytes = (int)(((long long)a.k + 31) / 32 * 16);
    const int passes = (n1 - n0 + wn * 16 - 1) / (wn * 16);
    float* out = reinterpret_cast<float*>(smem + p.out_off);
    float* red = reinterpret_cast<float*>(smem + p.red_off);
    const float* s_sh = reinterpret_cast<const float*>(smem + p.s_off) + (tile * 16 + g) * p.s_pitch;
    const uint16_t* z_sh = reinterpret_cast<const uint16_t*>(smem + p.z_off) + (tile * 16 + g) * p.s_pitch;
    // columns that no activation row fills repeat the last one
    int xo[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) xo[j] = min(j * 8 + g, cols - 1) * p.pitch + t * 16;

    uint32_t w[AHEAD][2][4];
    int c0 = 0, nc = min(p.stage, all);  // chunks of the stage
    int per = (nc + wk - 1) / wk;         // of a warp and tile
    // what to load next: chunk l_lc of the rows at l_p[]; chunks below l_full lie whole in all 16 rows
    int l_n = 0, l_lc = 0, l_left = 0, l_full = 0;
    const uint8_t* l_p[2];
    auto aim = [&](int n) {
        l_n = n;
        l_lc = kw;
        l_left = per;
        l_full = n + 16 <= n1 ? min(nc, row_bytes / 64 - c0) : 0;
#pragma unroll
        for (int i = 0; i < 2; i++) l_p[i] = a.w + (long long)(n + g + 8 * i) * a.ldw + (c0 + kw) * 64 + t * (16 / SUB);
    };
    auto load = [&](uint32_t (&w)[2][4]) {
        if (l_lc < l_full) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if constexpr (SUB == 1) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4*>(l_p[i]));
                    w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
                } else if constexpr (SUB == 2) {
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const uint2 v = __ldg(reinterpret_cast<const uint2*>(l_p[i] + s * 32));
                        w[i][2 * s] = v.x; w[i][2 * s + 1] = v.y;
                    }
                } else {
#pragma unroll
                    for (int s = 0; s < 4; s++) w[i][s] = __ldg(reinterpret_cast<const uint32_t*>(l_p[i] + s * 16));
                }
            }
        } else {  // the last rows, the last columns: a word at a time, zeros beyond them
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int left = l_lc < nc && l_n + g + 8 * i < n1 ? row_bytes - (c0 + l_lc) * 64 - t * (16 / SUB) : 0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int off = j / WORDS * (64 / SUB) + j % WORDS * 4;
                    w[i][j] = off < left ? __ldg(reinterpret_cast<const uint32_t*>(l_p[i] + off)) : 0u;
                }
            }
        }
        if (--l_left == 0) {
            aim(l_n + wn * 16);
        } else {
            l_lc += wk;
            l_p[0] += wk * 64;
            l_p[1] += wk * 64;
        }
    };

    for (;;) {
        aim(n0 + tile * 16);
#pragma unroll
        for (int d = 0; d < AHEAD; d++) load(w[d]);
        // this stage's activations and scales
        for (int m = 0; m < rows; m++)
            for (int b = threadIdx.x; b < nc * 16; b += THREADS) {
                const long long col = (long long)c0 * Q4_CHUNK + b * 8;
                uint4 v[PARTS];
                q4_blocks<T>(static_cast<const T*>(a.x) + (m0 + m) * a.ldx + col, a.k - col, a.x_vec, v);
                uint8_t* dst = smem + m * PARTS * p.pitch + ((b >> 4) * 16 + q4_block<SUB>(b & 15)) * 16;
#pragma unroll
                for (int q = 0; q < PARTS; q++) *reinterpret_cast<uint4*>(dst + q * p.pitch) = v[q];
            }
        for (int i = warp; i < n1 - n0; i += WARPS) {
            const size_t row = (size_t)(n0 + i) * a.groups;
            for (int b = lane; b < nc * SUB; b += 32) {
                const int gi = SUB == 1 ? (c0 + b) / (a.group / Q4_CHUNK) : c0 * SUB + b;
                const size_t at = row + min(gi, a.groups - 1);  // past the last group x is zero
                reinterpret_cast<float*>(smem + p.s_off)[i * p.s_pitch + b] = load_as_f32(a.s, at, a.s_dtype);
                if (a.z) reinterpret_cast<uint16_t*>(smem + p.z_off)[i * p.s_pitch + b] = (uint16_t)(MAGIC + a.z[at]);
            }
        }
        __syncthreads();
        float acc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        int pass = 0, at = 0;  // the tile and chunk worked on
        while (pass < passes) {
#pragma unroll
            for (int d = 0; d < AHEAD; d++) {
                if (pass >= passes) break;
                const int lc = kw + at * wk;
                if (lc < nc) {  // the same for the whole warp
                    const uint8_t* xb = smem + lc * 256;
                    const int so = pass * wn * 16 * p.s_pitch + lc * SUB;
#pragma unroll
                    for (int s = 0; s < SUB; s++) {
                        const float s0 = s_sh[so + s], s1 = s_sh[so + 8 * p.s_pitch + s];
                        uint32_t zz[2] = {(MAGIC + Q4_ZERO) * 0x10001u, (MAGIC + Q4_ZERO) * 0x10001u};
                        if (a.z) {
                            zz[0] = z_sh[so + s] * 0x10001u;
                            zz[1] = z_sh[so + 8 * p.s_pitch + s] * 0x10001u;
                        }
                        float part[NT][4];
#pragma unroll
                        for (int j = 0; j < NT; j++) part[j][0] = part[j][1] = part[j][2] = part[j][3] = 0.f;
#pragma unroll
                        for (int q = s * WORDS; q < (s + 1) * WORDS; q++) {
                            uint32_t f0[4], f1[4];
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                f0[i] = q4_pair<Ty::HALF>(w[d][i][q], 0, zz[i]);
                                f0[i + 2] = q4_pair<Ty::HALF>(w[d][i][q], 1, zz[i]);
                                f1[i] = q4_pair<Ty::HALF>(w[d][i][q], 2, zz[i]);
                                f1[i + 2] = q4_pair<Ty::HALF>(w[d][i][q], 3, zz[i]);
                            }
#pragma unroll
                            for (int j = 0; j < NT; j++) {
                                const uint4 b = *reinterpret_cast<const uint4*>(xb + xo[j] + q * 64);
                                mma16816<Ty::HALF>(part[j], f0, b.x, b.y);
                                mma16816<Ty::HALF>(part[j], f1, b.z, b.w);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < NT; j++) {
                            acc[j][0] += s0 * part[j][0];
                            acc[j][1] += s0 * part[j][1];
                            acc[j][2] += s1 * part[j][2];
                            acc[j][3] += s1 * part[j][3];
                        }
                    }
                }
                load(w[d]);
                if (++at == per) {
                    // the warps' sums of this tile: red[pass & 1][warp][16 rows][columns], added up by `rows` threads
                    float* r = red + ((pass & 1) * WARPS + warp) * 16 * (NT * 8 + 1) + g * (NT * 8 + 1) + 2 * t;
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        r[j * 8] = acc[j][0];
                        r[j * 8 + 1] = acc[j][1];
                        r[8 * (NT * 8 + 1) + j * 8] = acc[j][2];
                        r[8 * (NT * 8 + 1) + j * 8 + 1] = acc[j][3];
                        acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
                    }
                    __syncthreads();
                    for (int u = threadIdx.x; u < wn * 16 * rows; u += THREADS) {
                        const int i = u % (wn * 16), m = u / (wn * 16), n = pass * wn * 16 + i;
                        if (n < n1 - n0) {
                            const float* rb = red + ((pass & 1) * WARPS + (i >> 4)) * 16 * (NT * 8 + 1) +
                                              (i & 15) * (NT * 8 + 1) + m * PARTS;
                            float v = c0 ? out[m * p.rows + n] : 0.f;
                            for (int k = 0; k < wk; k++) {
#pragma unroll
                                for (int q = PARTS - 1; q >= 0; q--) v += rb[k * wn * 16 * (NT * 8 + 1) + q];
                            }
                            out[m * p.rows + n] = v;
                        }
                    }
                    at = 0;
                    pass++;
                }
            }
        }
        c0 += nc;
        __syncthreads();
        if (c0 >= all) break;
        nc = min(p.stage, all - c0);
        per = (nc + wk - 1) / wk;
    }
    for (int m = 0; m < rows; m++)
        for (int i = threadIdx.x; i < n1 - n0; i += THREADS) {
            float v = out[m * p.rows + i];
            if (a.bias) v += a.bias[n0 + i];
            if (a.res) v += to_f32(static_cast<const T*>(a.res)[(m0 + m) * a.ldr + n0 + i]);
            static_cast<T*>(a.y)[(m0 + m) * a.ldy + n0 + i] = from_f32<T>(v);
        }
}

constexpr int Q4_SMEM = 220 * 1024;

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
    constexpr int PARTS = Q4Type<T>::PARTS, ROWS = NT * 8 / PARTS, WARPS = q4_warps(NT);
    constexpr int MAX_ROWS = 512;  // weight rows of a block: their sums and scales lie in shared memory
    const int chunks = (a.k + Q4_CHUNK - 1) / Q4_CHUNK, sms = sm_count();
    const int m = a.rows < ROWS ? a.rows : ROWS;
    int blocks_n = a.n < sms ? a.n : sms;
    while ((a.n + blocks_n - 1) / blocks_n > MAX_ROWS) blocks_n += sms;
    Q4Plan p = {};
    p.rows = (a.n + blocks_n - 1) / blocks_n;
    // as many warps on a tile as it has chunks for
    p.wn = 1;
    while (p.wn < WARPS && WARPS / p.wn > chunks) p.wn *= 2;
    const int red = 2 * WARPS * 16 * (NT * 8 + 1) * 4;
    const int tiles_rows = (p.rows + p.wn * 16 - 1) / (p.wn * 16) * p.wn * 16;
    auto smem_of = [&](int stage) {
        p.stage = stage;
        p.pitch = stage * 256 + 64;
        p.s_pitch = stage * SUB | 1;
        p.s_off = m * PARTS * p.pitch;
        p.z_off = p.s_off + tiles_rows * p.s_pitch * 4;
        p.out_off = p.z_off + (a.z ? tiles_rows * p.s_pitch * 2 : 0);
        p.red_off = p.out_off + m * p.rows * 4;
        return p.red_off + red;
    };
    int stage = chunks < 1024 ? chunks : 1024;
    while (stage > 1 && smem_of(stage) > Q4_SMEM) stage -= stage > 16 ? 8 : 1;
    const int smem = smem_of(stage);
    if (smem > Q4_SMEM) return cudaErrorInvalidConfiguration;
    const int blocks_m = (int)(((long long)a.rows + ROWS - 1) / ROWS);
    for (p.row_block = 0; p.row_block < blocks_m; p.row_block += 65535) {
        const dim3 grid(blocks_n, blocks_m - p.row_block < 65535 ? blocks_m - p.row_block : 65535);
        kernel<<<grid, 32 * WARPS, smem, st>>>(a, p);
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
