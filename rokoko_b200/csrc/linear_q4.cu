// linear_q4.cu -- the linear layer with 4-bit weights in groups along the
// reduction, for few rows, and the quantiser that makes such weights:
//
//   y[m][n] = sum_g s[n][g] sum_{k in g} (q[n][k] - z[n][g]) x[m][k] + bias[n] + residual[m][n]
//
// Byte j of a weight row holds columns 2j (low half) and 2j + 1 (high half).
//
// The product runs on tcgen05 (kind::f8f6f4) without rounding anything of the
// weights, or of x in 16 bits.  A whole number up to 16 in a byte, with a sign at
// its top, is an e4m3 number already: it reads 2^-9 times as much, so q - z comes
// out of a word of codes by bytewise arithmetic (signed_codes).  The zero point is
// taken off there and not from the sums: z sum x is rounded, and a large x whose
// weight is zero would leave its rounding behind.  x is scaled by a power of two,
// the same for a row, and split into e5m2 parts, each sixteen times finer than the
// one before: three hold the 8 and 11 bits of bfloat16 and half, six 23 of the 24
// of float (Q4Type says how far below a row's largest).  The parts are columns of
// the MMA's N side; a group's accumulators are read back, put together and scaled
// in 32 bits:
//
//   sum_g s 2^9 sum_p 16^-p D_p
//
// Two launches.  The first (q4_parts_kernel) lays the parts out in the
// workspace as the second wants them in shared memory.  The second gives each SM
// an even share of the weight rows, at most 128, the MMA's M side; a share of at
// most 64 (32) rows fills the 128 with 2 (4) ranges of k one below the other,
// whose parts are N columns of their own: an MMA takes 66 clocks whatever N <=
// 112 is, so its rows are what must not lie idle.  Some warps turn codes into
// operands, one thread issues the MMAs, eight warps add up the accumulators.  The
// weights' bytes are read once.  Bound by the latency of a step in the warps of
// codes, with small groups by that of reading accumulators back: 1 x 8192 x 8192
// bf16 21.8 us, 4 x 16384 x 16384 half with zero points 75 us (1.9 TB/s), 24 x
// 5003 x 4001 float in groups of 32 72 us.
//
// A row with an infinity, a NaN, or magnitudes too far apart does not fit the
// parts; its sums are done one by one in 32 bits instead.
#include <cuda_fp8.h>

#include <atomic>
#include <type_traits>

#include "ptx.cuh"
#include "q4_plan.h"
#include "quant.cuh"
#include "status.h"

namespace rk {
namespace {

constexpr int Q4_ZERO = 8;  // the zero point of weights that have none of their own

// The parts of a type, and how many binades below its row's largest magnitude a value may lie to be left to them.  The
// parts' last place is 2^-24 with three and 2^-36 with six where the largest lies in [2^13, 2^14), which holds bfloat16
// exactly down to 30 binades and half down to 27.  Of float the last place may be lost (1.6 % of values), below 27
// binades up to 8 of it: 16 u of a value (u = 2^-24), half of what the sums' last roundings are allowed.
template <typename T> struct Q4Type { static constexpr int PARTS = 3, SPAN = 30; };
template <> struct Q4Type<__half> { static constexpr int PARTS = 3, SPAN = 27; };
template <> struct Q4Type<float> { static constexpr int PARTS = 6, SPAN = 30; };

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
    bool x_vec;   // rows of x start on 16-byte boundaries
    uint8_t* ws;  // per pass: its steps' stages, then the rows' Q4Row
};

// ---------------------------------------------------------------- the parts of x

// row, column byte -> offset in a tile of 128-byte rows in the 128-byte swizzle
__device__ __forceinline__ uint32_t q4_swizzle(uint32_t row, uint32_t byte) {
    return row * 128 + ((byte >> 4 ^ (row & 7)) << 4) + (byte & 15);
}

// Block (y: activation row, x: a slice of the blocks of K).  Every block looks over its whole row for the largest and
// smallest magnitude, then writes the parts of its slice: eight columns a thread, in the order 0, 2, 4, 6, 1, 3, 5, 7
// that the codes of a word come out in.
template <typename T>
__global__ void __launch_bounds__(256) q4_parts_kernel(const Q4Args a, const Q4Plan p) {
    constexpr int PARTS = Q4Type<T>::PARTS;
    __shared__ int sh_max[8], sh_min[8];
    const int pass = p.pass0 + blockIdx.y / Q4_ROWS, m = blockIdx.y % Q4_ROWS;
    const long long row = (long long)pass * Q4_ROWS + m;
    if (row >= a.rows) return;
    // The product may start when every block of this launch has: it fetches weights until it needs the parts.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    uint8_t* ws = a.ws + (size_t)pass * p.pass_bytes;
    auto load8 = [&](long long c, float (&v)[8]) {
        struct alignas(16) Q { T v[16 / sizeof(T)]; };
        if (a.x_vec && c + 8 <= a.k) {
#pragma unroll
            for (int i = 0; i < 8; i += 16 / sizeof(T)) {
                const Q q = *reinterpret_cast<const Q*>(x + c + i);
#pragma unroll
                for (int j = 0; j < 16 / (int)sizeof(T); j++) v[i + j] = to_f32(q.v[j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = c + i < a.k ? to_f32(x[c + i]) : 0.f;
        }
    };
    // exponents as integers order like magnitudes; zeros do not count
    int top = 0, low = 255;
    for (long long c = threadIdx.x * 8LL; c < a.k; c += 256 * 8) {
        float v[8];
        load8(c, v);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t u = __float_as_uint(v[i]) & 0x7fffffffu;
            const int e = (int)(u >> 23);
            top = max(top, e);
            if (u) low = min(low, e);
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_min_sync(0xffffffffu, low);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) { sh_max[warp] = top; sh_min[warp] = low; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) { top = max(top, sh_max[i]); low = min(low, sh_min[i]); }
    const bool odd = top == 255 || (low < 255 && low < top - Q4Type<T>::SPAN);
    // the largest magnitude comes to lie in [2^13, 2^14): e5m2 ends at 57344
    const int shift = min(126, 13 - (top - 127));
    const float scale = odd ? 0.f : __uint_as_float((uint32_t)(shift + 127) << 23);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        const int back = 9 - shift;  // may pass a float's exponents: two factors
        Q4Row r;
        r.inv = ldexpf(1.f, back / 2);
        r.inv2 = ldexpf(1.f, back - back / 2);
        r.odd = odd;
        r.pad = 0;
        reinterpret_cast<Q4Row*>(ws + (size_t)p.steps * p.x_bytes)[m] = r;
    }
    const int blocks = p.h * p.steps;
    // two blocks of K a warp at a time
    for (int b = blockIdx.x * 2 + warp * 2 * gridDim.x + (lane >> 4); b < blocks; b += 16 * gridDim.x) {
        const int g8 = lane & 15;
        float v[8];
        load8((long long)b * Q4_KB + g8 * 8, v);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = odd ? 0.f : v[i] * scale;
        const int range = b / p.steps, step = b - range * p.steps;
        uint8_t* st = ws + (size_t)step * p.x_bytes;
#pragma unroll
        for (int q = 0; q < PARTS; q++) {
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const __nv_fp8_storage_t f = __nv_cvt_float_to_fp8(v[i], __NV_SATFINITE, __NV_E5M2);
                v[i] = (v[i] - __half2float(__half(__nv_cvt_fp8_to_halfraw(f, __NV_E5M2)))) * 16.f;
                w[i & 1] |= (uint32_t)f << (8 * (i >> 1));
            }
            *reinterpret_cast<uint2*>(st + q4_swizzle(range * p.nc + q * p.mq + m, g8 * 8)) = make_uint2(w[0], w[1]);
        }
    }
}

// ---------------------------------------------------------------- the product

__device__ uint32_t q4_err;  // set when a bounded wait of the kernel gives up

// Four codes 0..15 in a word's bytes, z in each byte of `z`: q - z in e4m3, times 2^-9.  The bytes of u + 0x80 - z never
// carry and keep the top bit where q >= z, which the sign is the inverse of.  (The negative side by complement and the
// increments by mask, without vabsdiff4: two more instructions, 78 us for 75 at 4 x 16384 x 16384.)
__device__ __forceinline__ uint32_t signed_codes(uint32_t u, uint32_t z) {
    uint32_t size;
    asm("vabsdiff4.u32.u32.u32 %0, %1, %2, %3;" : "=r"(size) : "r"(u), "r"(z), "r"(0));
    return size | (~(u + (0x80808080u - z)) & 0x80808080u);
}

// 32 lanes x 4 columns, not waited for
__device__ __forceinline__ void tmem_ld4(uint32_t taddr, float (&v)[4]) {
    uint32_t r[4];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = __uint_as_float(r[i]);
}
template <int N>
__device__ __forceinline__ void tmem_ld_wait(float (&v)[N][4]) {  // the loads above are in v after it
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) asm volatile("" : "+f"(v[i][j]));
}

// MB: activation rows that a thread has sums for; SUB: groups of a block of K
template <typename T, int MB, int SUB>
__global__ void __launch_bounds__(Q4_THREADS, 1) linear_q4_kernel(const Q4Args a, const Q4Plan p) {
    constexpr int PARTS = Q4Type<T>::PARTS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t full[Q4_STAGES], empty[Q4_STAGES], d_full[4], d_empty[4], drain;
    __shared__ uint32_t tmem_sh;
    __shared__ int lost;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // the same for a warp, and known to be
    const int n0 = (int)((long long)a.n * blockIdx.x / gridDim.x), n1 = (int)((long long)a.n * (blockIdx.x + 1) / gridDim.x);
    const int pass = p.pass0 + blockIdx.y;
    const long long m0 = (long long)pass * Q4_ROWS;
    const int rows = (int)(a.rows - m0 < Q4_ROWS ? a.rows - m0 : Q4_ROWS);
    const uint8_t* ws = a.ws + (size_t)pass * p.pass_bytes;
    const uint32_t stage = p.stage;
    if (warp == 0 && lane == 0) {
        // a stage is full when the x copy (its bytes) and both halves' codes are there, empty when the products and the
        // warps of sums that look at it are done with it
        for (int s = 0; s < p.stages; s++) { mbar_init(&full[s], 3); mbar_init(&empty[s], SUB == 1 ? 5 : 9); }
        for (int s = 0; s < p.accs; s++) { mbar_init(&d_full[s], 1); mbar_init(&d_empty[s], 4); }
        mbar_init(&drain, 1);
        lost = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_sh, p.tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_sh;
    float* red = reinterpret_cast<float*>(ring);  // [sets][rows][128], once the ring is done with

    if (warp == 0) {  // x: one copy a step, once the first launch is done
        asm volatile("griddepcontrol.wait;" ::: "memory");
        int i = 0, s = 0;
        uint32_t parity = 1;
        for (; i < p.steps; i++) {
            if (!mbar_wait_warp(&empty[s], parity, &q4_err, RK_DEV_TIMEOUT_EMPTY)) { lost = 1; break; }
            if (elect_one()) {
                mbar_arrive_expect_tx(&full[s], p.x_bytes);
                bulk_load(ring + s * stage + Q4_A_BYTES, ws + (size_t)i * p.x_bytes, p.x_bytes, &full[s]);
            }
            if (++s == p.stages) { s = 0; parity ^= 1; }
        }
        for (int q = i > p.stages ? i - p.stages : 0; q < i; q++)  // no copy outlives the block
            mbar_wait_warp(&full[q % p.stages], q / p.stages & 1, &q4_err, RK_DEV_TIMEOUT_DRAIN);
    } else if (warp == 1) {  // products
        const uint64_t desc = sw128_kmajor_desc(smem_u32(ring), 0);
        const uint32_t desc0 = (uint32_t)desc, desc_hi = (uint32_t)(desc >> 32);
        uint32_t d = 0, d_parity = 1, parity = 0;
        int s = 0;
        bool alive = true;
        for (int i = 0; i < p.steps && alive; i++) {
            if (!mbar_wait_warp(&full[s], parity, &q4_err, RK_DEV_TIMEOUT_FULL)) { alive = false; break; }
            const uint32_t w = desc0 + s * (stage >> 4), x = w + (Q4_A_BYTES >> 4);
#pragma unroll
            for (int b = 0; b < SUB; b++) {
                if (!mbar_wait_warp(&d_empty[d], d_parity, &q4_err, RK_DEV_TIMEOUT_EMPTY)) { alive = false; break; }
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int e = 0; e < 4 / SUB; e++) {
                        const int kk = b * (4 / SUB) + e;
                        umma_f8(tmem + d * p.acc_cols, w + 2 * kk, x + 2 * kk, desc_hi, p.idesc, e > 0 ? 1u : 0u);
                    }
                    umma_commit(&d_full[d]);
                    if (b == SUB - 1) umma_commit(&empty[s]);
                }
                if ((int)++d == p.accs) { d = 0; d_parity ^= 1; }
            }
            if (++s == p.stages) { s = 0; parity ^= 1; }
        }
        if (!alive) lost = 1;
        if (elect_one()) umma_commit(&drain);
        mbar_wait_warp(&drain, 0, &q4_err, RK_DEV_TIMEOUT_DRAIN);
        tc_fence_before();
    } else if (warp < 2 + Q4_CODES) {
        // Codes.  A warp takes one half (64 rows) of a step at a time, eight units of 16 bytes a lane, and the scales of
        // those rows; as soon as a unit is laid out, its successor's load is on its way.
        const int u = lane & 3, half = (warp & 1) * 64;
        const int row_bytes = (int)(((long long)a.k + 31) / 32 * 16);
        const int shift = p.h == 4 ? 5 : p.h == 2 ? 6 : 7;                       // row -> range
        const uint8_t* src[2];                                                   // first rows of the half's two 32s
        uint32_t there = 0;                                                      // units whose rows are there
        int k_off[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int i = half + e * 32 + (lane >> 2), range = i >> shift;
            src[e] = a.w + (long long)(n0 + i - range * p.pad) * a.ldw + (long long)range * p.steps * 64 + u * 16;
            k_off[e] = range * p.steps * 64 + u * 16;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (n0 + i + 8 * j - range * p.pad < n1) there |= 1u << (e * 4 + j);
        }
        // what is not there stays as it is: rows that nobody stores, columns where x is zero
        auto mask_of = [&](int step) {
            uint32_t m = there;
            if (k_off[0] + step * 64 >= row_bytes) m &= 0xf0u;
            if (k_off[1] + step * 64 >= row_bytes) m &= 0x0fu;
            return step < p.steps ? m : 0u;
        };
        // two rows a lane for the scales
        const uint32_t per = a.group > Q4_KB ? a.group / Q4_KB : 1;              // blocks of K a group
        size_t sz[2];
        uint32_t block0[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int i = half + e * 32 + lane, range = i >> shift;
            sz[e] = (size_t)min(n0 + i - range * p.pad, a.n - 1) * a.groups;
            block0[e] = range * p.steps;
        }
        uint32_t s_raw[2][SUB], z_raw[2][SUB];
        const uint32_t pick = (SUB == 4 ? u : SUB == 2 ? u >> 1 : 0) * 0x1111u;  // the group of this lane's columns
        auto fetch = [&](int step) {                                             // converted only when they are used
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int b = 0; b < SUB; b++) {
                    const uint32_t block = block0[e] + step;
                    const uint32_t g = SUB == 1 && per > 1 ? block / per : block * SUB + b;
                    const size_t at = sz[e] + min(g, a.groups - 1u);             // past the last group x is zero
                    z_raw[e][b] = a.z ? a.z[at] : Q4_ZERO;
                    s_raw[e][b] = a.s_dtype == RK_DTYPE_F32 ? static_cast<const uint32_t*>(a.s)[at]
                                                            : static_cast<const uint16_t*>(a.s)[at];
                }
        };
        uint4 w[8] = {};
        auto load = [&](int j, int step, uint32_t m) {
            if (m >> j & 1) w[j] = __ldg(reinterpret_cast<const uint4*>(src[j >> 2] + (j & 3) * 8 * a.ldw + (long long)step * 64));
        };
        constexpr int STRIDE = Q4_CODES / 2;
        const int first = (warp - 2) >> 1;
        {
            const uint32_t m = mask_of(first);
#pragma unroll
            for (int j = 0; j < 8; j++) load(j, first, m);
            fetch(first);
        }
        const uint32_t dst = (half + (lane >> 2)) * 128 + ((2 * u ^ (lane >> 2)) << 4);
        int s = first % p.stages;
        uint32_t parity = (first / p.stages & 1) ^ 1;
        bool alive = true;
#pragma unroll 1
        for (int i = first; i < p.steps; i += STRIDE) {
            const uint32_t m = mask_of(i + STRIDE);
            alive = __all_sync(0xffffffffu, mbar_wait(&empty[s], parity, &q4_err, RK_DEV_TIMEOUT_EMPTY));
            if (!alive) break;
            uint8_t* st = ring + s * stage;
            auto turn = [&](auto own) {  // own: the weights have zero points
                uint32_t zeros[2] = {};  // of this lane's two rows, a byte a group
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int b = 0; b < SUB; b++) zeros[e] |= z_raw[e][b] << (8 * b);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint4 c = w[j];
                    constexpr uint32_t M = 0x0f0f0f0fu;
                    uint8_t* to = st + j * 1024;
                    uint32_t z = Q4_ZERO * 0x01010101u;
                    if constexpr (decltype(own)::value) {
                        z = __shfl_sync(0xffffffffu, zeros[j >> 2], (lane >> 2) + 8 * (j & 3));
                        asm("prmt.b32 %0, %0, %0, %1;" : "+r"(z) : "r"(pick));
                    }
                    // the second 16 bytes' place differs from the first's in the swizzled chunk's lowest bit
                    *reinterpret_cast<uint4*>(to + dst) = make_uint4(signed_codes(c.x & M, z), signed_codes(c.x >> 4 & M, z),
                                                                     signed_codes(c.y & M, z), signed_codes(c.y >> 4 & M, z));
                    *reinterpret_cast<uint4*>(to + (dst ^ 16)) =
                        make_uint4(signed_codes(c.z & M, z), signed_codes(c.z >> 4 & M, z), signed_codes(c.w & M, z),
                                   signed_codes(c.w >> 4 & M, z));
                    load(j, i + STRIDE, m);
                }
            };
            if (a.z) turn(std::true_type{});
            else turn(std::false_type{});
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int b = 0; b < SUB; b++) {
                    const uint32_t r = s_raw[e][b];
                    const float f = a.s_dtype == RK_DTYPE_F32 ? __uint_as_float(r)
                                    : a.s_dtype == RK_DTYPE_F16 ? __half2float(__ushort_as_half((uint16_t)r))
                                                                : __uint_as_float(r << 16);
                    reinterpret_cast<float*>(st + p.s_off)[(half + e * 32 + lane) * SUB + b] = f;
                }
            if (i + STRIDE < p.steps) fetch(i + STRIDE);
            // Orders these plain writes before the MMAs' reads: here, where there is time, and not in the issuing thread.
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[s]);
            s += STRIDE;
            while (s >= p.stages) { s -= p.stages; parity ^= 1; }
        }
        if (!alive && lane == 0) lost = 1;
    } else {
        // Sums: lane i of the MMA's rows = range i / pad, weight row n0 + i % pad.  Two sets of four warps take turns at
        // the accumulators.
        const int quarter = warp & 3, i = quarter * 32 + lane, range = quarter * 32 / p.pad;
        const int set = (warp - 2 - Q4_CODES) >> 2;
        const uint32_t base = tmem + ((uint32_t)(quarter * 32) << 16) + range * p.nc;
        float acc[MB];
#pragma unroll
        for (int m = 0; m < MB; m++) acc[m] = 0.f;
        uint32_t d = set, d_parity = 0;
        bool alive = true;
        constexpr int TURN = SUB == 1 ? 2 : 1;  // steps from one to the next that this set looks at
        int s = SUB == 1 ? set % p.stages : 0;
        uint32_t parity = SUB == 1 ? set / p.stages & 1 : 0;
#pragma unroll 1
        for (int step = SUB == 1 ? set : 0; step < p.steps && alive; step += TURN) {
            alive = __all_sync(0xffffffffu, mbar_wait(&full[s], parity, &q4_err, RK_DEV_TIMEOUT_FULL));
            if (!alive) break;
            const float* scales = reinterpret_cast<const float*>(ring + s * stage + p.s_off) + i * SUB;
#pragma unroll 1
            for (int b = SUB == 1 ? 0 : set; b < SUB; b += 2) {
                alive = __all_sync(0xffffffffu, mbar_wait(&d_full[d], d_parity, &q4_err, RK_DEV_TIMEOUT_ACC));
                if (!alive) break;
                tc_fence_after();
                const float f = scales[b];
#pragma unroll
                for (int m = 0; m < MB; m += 4) {
                    if (m < p.mq) {
                        float v[PARTS][4];
#pragma unroll
                        for (int q = 0; q < PARTS; q++) tmem_ld4(base + d * p.acc_cols + q * p.mq + m, v[q]);
                        tmem_ld_wait(v);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            float t = v[PARTS - 1][j];
#pragma unroll
                            for (int q = PARTS - 2; q >= 0; q--) t = fmaf(t, 0.0625f, v[q][j]);
                            acc[m + j] = fmaf(f, t, acc[m + j]);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&d_empty[d]);
                d += 2;
                if ((int)d >= p.accs) { d = set; d_parity ^= 1; }
            }
            if (alive && lane == 0) mbar_arrive(&empty[s]);
            s += TURN;
            while (s >= p.stages) { s -= p.stages; parity ^= 1; }
        }
        if (!alive && lane == 0) lost = 1;
        // every warp of sums has read its last accumulator: all products are done, and nothing of the ring is in use
        asm volatile("bar.sync 1, %0;" ::"n"(32 * Q4_SUMS) : "memory");
#pragma unroll
        for (int m = 0; m < MB; m++)
            if (alive && m < rows) red[(set * Q4_ROWS + m) * Q4_M + i] = acc[m];
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, p.tmem_cols);
    }
    if (lost) return;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the first launch's rows, here read plainly
    const Q4Row* info = reinterpret_cast<const Q4Row*>(ws + (size_t)p.steps * p.x_bytes);
    for (int m = 0; m < rows; m++) {
        const Q4Row r = info[m];
        if (!r.odd) {
            for (int i = threadIdx.x; i < n1 - n0; i += Q4_THREADS) {
                const int n = n0 + i;
                float v = 0.f;
                for (int h = 0; h < p.h; h++) v += red[m * Q4_M + h * p.pad + i] + red[(Q4_ROWS + m) * Q4_M + h * p.pad + i];
                v = v * r.inv * r.inv2;
                if (a.bias) v += a.bias[n];
                if (a.res) v += to_f32(static_cast<const T*>(a.res)[(m0 + m) * a.ldr + n]);
                static_cast<T*>(a.y)[(m0 + m) * a.ldy + n] = from_f32<T>(v);
            }
        } else {  // a warp a weight row, one by one
            const T* x = static_cast<const T*>(a.x) + (m0 + m) * a.ldx;
            for (int n = n0 + warp; n < n1; n += Q4_THREADS / 32) {
                const uint8_t* w = a.w + (long long)n * a.ldw;
                float v = 0.f;
                for (int k = lane; k < a.k; k += 32) {
                    const size_t g = (size_t)n * a.groups + k / a.group;
                    const int q = (w[k >> 1] >> (k & 1) * 4 & 15) - (a.z ? a.z[g] : Q4_ZERO);
                    v += (load_as_f32(a.s, g, a.s_dtype) * (float)q) * to_f32(x[k]);  // q x may pass the largest float
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                if (lane == 0) {
                    if (a.bias) v += a.bias[n];
                    if (a.res) v += to_f32(static_cast<const T*>(a.res)[(m0 + m) * a.ldr + n]);
                    static_cast<T*>(a.y)[(m0 + m) * a.ldy + n] = from_f32<T>(v);
                }
            }
        }
    }
}

// ---------------------------------------------------------------- host

template <typename T, int MB, int SUB>
cudaError_t launch_mb(const Q4Args& a, cudaStream_t st) {
    auto kernel = linear_q4_kernel<T, MB, SUB>;
    Q4Plan p;
    static std::atomic<uint64_t> ready{0};  // devices on which the kernel's shared memory is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4_SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    if (!q4_plan(a.rows, a.n, a.k, a.group, sizeof(T), sm_count(), p)) return cudaErrorInvalidConfiguration;
    p.idesc = umma_idesc_e4m3(Q4_M, p.mma_n) | 1u << 10;  // B in e5m2
    const int passes = (int)(((long long)a.rows + Q4_ROWS - 1) / Q4_ROWS);
    for (p.pass0 = 0; p.pass0 < passes; p.pass0 += 2047) {  // rows and passes are the grids' second dimension
        const int n = passes - p.pass0 < 2047 ? passes - p.pass0 : 2047;
        const int rows = n > 1 ? n * Q4_ROWS : (a.rows - p.pass0 * Q4_ROWS < Q4_ROWS ? a.rows - p.pass0 * Q4_ROWS : Q4_ROWS);
        const int slices = (p.h * p.steps + 15) / 16;  // 16 blocks of K a block: two a warp
        q4_parts_kernel<T><<<dim3(slices, rows), 256, 0, st>>>(a, p);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)p.grid, n);
        cfg.blockDim = dim3(Q4_THREADS);
        cfg.dynamicSmemBytes = p.smem;
        cfg.stream = st;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, kernel, a, p);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

template <typename T, int SUB>
cudaError_t launch_sub(const Q4Args& a, cudaStream_t st) {
    if (a.rows <= 4) return launch_mb<T, 4, SUB>(a, st);
    if (a.rows <= 8) return launch_mb<T, 8, SUB>(a, st);
    if (a.rows <= 16) return launch_mb<T, 16, SUB>(a, st);
    return launch_mb<T, 32, SUB>(a, st);
}

template <typename T>
cudaError_t launch(const Q4Args& a, cudaStream_t st) {
    if (a.group == 32) return launch_sub<T, 4>(a, st);
    if (a.group == 64) return launch_sub<T, 2>(a, st);
    return launch_sub<T, 1>(a, st);
}

// A scale rounded to its type, at most the largest finite value there, as it is stored.
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
    const int k0 = g * group, k1 = k - k0 > group ? k0 + group : k;
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

void* q4_err_word() {
    void* p = nullptr;
    return cudaGetSymbolAddress(&p, q4_err) == cudaSuccess ? p : nullptr;
}

}  // namespace rk

using namespace rk;

extern "C" size_t rk_linear_q4_workspace_size(int rows, int n, int k, int group, int dtype) {
    if (!size_ok(rows, 0) || !size_ok(n, 1) || !size_ok(k, 1) || !group_ok(group) || !dtype_ok(dtype)) return 0;
    return rows ? q4_workspace(rows, k, dtype_bytes(dtype)) : 0;
}

extern "C" rk_status rk_linear_q4(const void* x, long long ldx, const void* w, long long ldw, const void* scales,
                                  const uint8_t* zeros, const float* bias, const void* residual, long long ldr,
                                  void* y, long long ldy, void* workspace, size_t workspace_size, int rows, int n,
                                  int k, int group, int dtype, int scale_dtype, void* stream) {
    const char* who = "rk_linear_q4: unsupported arguments";
    if (!dtype_ok(dtype) || !dtype_ok(scale_dtype) || !size_ok(rows, 0) || !size_ok(n, 1) || !size_ok(k, 1))
        return fail(RK_ERR_CANNOT_IMPLEMENT, who);
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
    if (!workspace || workspace_size < q4_workspace(rows, k, e) || !aligned(workspace, 256))
        return fail(RK_ERR_WORKSPACE, "rk_linear_q4: workspace too small or not 256-byte aligned");
    Q4Args a{x, static_cast<const uint8_t*>(w), scales, zeros, bias, residual, y, ldx, ldw, ldr, ldy, rows, n, k,
             group, (int)(((long long)k + group - 1) / group), scale_dtype,
             aligned(x, 16) && (rows == 1 || ldx * (long long)e % 16 == 0), static_cast<uint8_t*>(workspace)};
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
    if (!dtype_ok(dtype) || !dtype_ok(scale_dtype) || !size_ok(n, 0) || !size_ok(k, 1))
        return fail(RK_ERR_CANNOT_IMPLEMENT, who);
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
