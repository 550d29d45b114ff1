// rms_norm.cu -- root-mean-square norm with the residual's addition, its output
// in the input's type or in 8 bits with a scale for each row, and the same
// 8-bit rows without the norm.
//
//   h = x + residual            (32 bit)
//   y = h / sqrt(mean(h^2) + eps) * w
//   q = e4m3(y / s),  s = max(max|y|, 1e-30) / 448
#include <cuda_fp8.h>

#include <atomic>

#include "ptx.cuh"
#include "quant.cuh"
#include "status.h"

namespace rk {
namespace {

struct NormArgs {
    const void *x, *res, *w;
    void *sum, *y;
    uint8_t* q;
    float* scale;
    long long ldx, ldr, lds, ldy, ldq;
    int rows, cols;
    float eps;
    float inv_cols;
    uint32_t xoff, roff;  // x and res modulo 16 bytes
};

__device__ uint32_t norm_err;  // set when a bounded wait of the streaming kernel gives up

constexpr int RING_BYTES = 208 * 1024;  // shared memory of an SM that the streaming kernel's rings share

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};
template <int VEC>
struct alignas(VEC) Codes {
    uint8_t v[VEC];
};

template <int VEC>
__device__ __forceinline__ void store_codes(uint8_t* q, const float (&v)[VEC], float inv_scale) {
    Codes<VEC> c;
    if constexpr (VEC == 1) {
        c.v[0] = __nv_cvt_float_to_fp8(v[0] * inv_scale, __NV_SATFINITE, __NV_E4M3);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const __nv_fp8x2_storage_t p =
                __nv_cvt_float2_to_fp8x2(make_float2(v[j] * inv_scale, v[j + 1] * inv_scale), __NV_SATFINITE, __NV_E4M3);
            c.v[j] = (uint8_t)(p & 0xff);
            c.v[j + 1] = (uint8_t)(p >> 8);
        }
    }
    *reinterpret_cast<Codes<VEC>*>(q) = c;
}

// One row's elements of a thread: h = x + residual goes out at once, h w stays
// in registers; sums of squares and the largest |h w| come back.
template <typename T, int VEC>
struct RowPart {
    float ss = 0.f, top = 0.f;
    __device__ __forceinline__ void add(const Pack<T, VEC>& x, const Pack<T, VEC>& r, const Pack<T, VEC>& w, bool res,
                                        bool norm, T* sum, float (&hw)[VEC]) {
        float h[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            h[j] = to_f32(x.v[j]);
            if (res) h[j] += to_f32(r.v[j]);
            ss += h[j] * h[j];
            hw[j] = norm ? h[j] * to_f32(w.v[j]) : h[j];
            top = max_nan(top, fabsf(hw[j]));
        }
        if (sum) {
            Pack<T, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; j++) o.v[j] = from_f32<T>(h[j]);
            *reinterpret_cast<Pack<T, VEC>*>(sum) = o;
        }
    }
    template <int LANES>
    __device__ __forceinline__ void reduce() {  // over aligned groups of LANES lanes
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
    }
    // over the block: one barrier, which the row's slot of shared memory is free after
    __device__ __forceinline__ bool reduce_block(float2 (&red)[32], bool ok) {
        const int lane = threadIdx.x & 31, n = blockDim.x >> 5;
        reduce<32>();
        if (lane == 0) red[threadIdx.x >> 5] = make_float2(ss, top);
        ok = __syncthreads_and(ok);
        const float2 v = lane < n ? red[lane] : make_float2(0.f, 0.f);
        ss = v.x;
        top = v.y;
        if (n > 8) reduce<32>();
        else reduce<8>();
        ss = __shfl_sync(0xffffffffu, ss, 0);
        top = __shfl_sync(0xffffffffu, top, 0);
        return ok;
    }
};

// What a row's elements h w are multiplied by, and its 8-bit scale.  The row's
// factor cancels from y / scale, so a code is h w times 448 / max|h w|: three
// roundings in all, which keeps the codes off the wrong side of a step as well
// as a division by the scale does.  Rows near the scale's floor go through it.
struct RowFactors {
    float y, q, scale;
    __device__ __forceinline__ RowFactors(const NormArgs& a, float ss, float top) {
        y = a.w ? rsqrtf(ss * a.inv_cols + a.eps) : 1.f;
        scale = max_nan(top * y, AMAX_FLOOR) * (1.f / Q8_MAX);
        q = top >= AMAX_FLOOR && top * y >= AMAX_FLOOR ? __fdiv_rn(Q8_MAX, top) : y / scale;
        if (q > 3e38f) q = 3e38f;  // zeros of such a row stay zeros
    }
};

template <typename T, int VEC>
__device__ __forceinline__ void store_part(const NormArgs& a, long long row, int c, const float (&hw)[VEC],
                                           const RowFactors& f) {
    if (a.y) {
        Pack<T, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; j++) o.v[j] = from_f32<T>(hw[j] * f.y);
        *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.y) + row * a.ldy + c) = o;
    }
    if (a.q) store_codes<VEC>(a.q + row * a.ldq + c, hw, f.q);
}

// A row per group of G lanes, or per block (G = 0), held in registers: NV
// vectors of VEC elements a thread.  The sum of squares and the largest |h w|
// are reduced together, so a row is read once and a block has one barrier; the
// largest |y| is the largest |h w| times the row's factor.
template <typename T, int VEC, int NV, int G>
__global__ void __launch_bounds__(G ? 256 : 1024) norm_rows_kernel(const NormArgs a) {
    __shared__ float2 red[32];
    const int n = G ? G : blockDim.x, tid = G ? threadIdx.x % (G ? G : 1) : threadIdx.x;
    const long long row_ = G ? (long long)blockIdx.x * (256 / (G ? G : 1)) + threadIdx.x / (G ? G : 1) : blockIdx.x;
    const bool live = row_ < a.rows;
    const long long row = live ? row_ : a.rows - 1;  // lanes past the last row take part in the shuffles
    using P = Pack<T, VEC>;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* r = static_cast<const T*>(a.res) + row * a.ldr;
    P px[NV], pr[NV], pw[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * n + tid) * VEC;
        if (c < a.cols) {
            px[i] = *reinterpret_cast<const P*>(x + c);
            if (a.res) pr[i] = *reinterpret_cast<const P*>(r + c);
        }
    }
    if (a.w) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * n + tid) * VEC;
            if (c < a.cols) pw[i] = *reinterpret_cast<const P*>(static_cast<const T*>(a.w) + c);
        }
    }
    float hw[NV][VEC];
    RowPart<T, VEC> p;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * n + tid) * VEC;
        if (c < a.cols)
            p.add(px[i], pr[i], pw[i], a.res, a.w,
                  a.sum && live ? static_cast<T*>(a.sum) + row * a.lds + c : nullptr, hw[i]);
    }
    if constexpr (G) p.template reduce<G>();
    else p.reduce_block(red, true);
    if (!live) return;
    const RowFactors f(a, p.ss, p.top);
    if (a.q && tid == 0) a.scale[row] = f.scale;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * n + tid) * VEC;
        if (c < a.cols) store_part<T, VEC>(a, row, c, hw[i], f);
    }
}

// The 16-byte granules that hold a row; every granule holds at least one byte of it.
__device__ __forceinline__ uint32_t granules(const void* row, uint32_t bytes, const char** first) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(row), lo = p & ~uintptr_t(15);
    *first = reinterpret_cast<const char*>(lo);
    return (uint32_t)(((p + bytes + 15) & ~uintptr_t(15)) - lo);
}

constexpr int MAX_STAGES = 4;

// The rows on their way to a block that walks over them: `stages` slots of shared memory, each for a row of x and one of
// the residual behind it, whole granules.  One thread loads.
struct RowRing {
    uint8_t* slots;
    uint64_t* bar;
    int stages;
    uint32_t slot_bytes, stage_bytes, row_bytes;
    template <typename T>
    __device__ __forceinline__ void load(const NormArgs& a, long long row, int s) const {
        const char *px, *pr;
        const uint32_t nx = granules(static_cast<const T*>(a.x) + row * a.ldx, row_bytes, &px);
        uint32_t nr = 0;
        if (a.res) nr = granules(static_cast<const T*>(a.res) + row * a.ldr, row_bytes, &pr);
        mbar_arrive_expect_tx(&bar[s], nx + nr);
        bulk_load(slots + (size_t)s * stage_bytes, px, nx, &bar[s]);
        if (a.res) bulk_load(slots + (size_t)s * stage_bytes + slot_bytes, pr, nr, &bar[s]);
    }
    // A wait for slot s gave up at `row`: no copy may outlive the block.
    __device__ __forceinline__ void drain(const NormArgs& a, long long row, long long step, int s, uint32_t parity) const {
        for (int k = 0; k < stages; k++)
            if (row + k * step < a.rows) {
                const int q = s + k < stages ? s + k : s + k - stages;
                mbar_wait(&bar[q], s + k < stages ? parity : parity ^ 1, &norm_err, RK_DEV_TIMEOUT_DRAIN);
            }
    }
};

// Many rows: resident blocks walk over the rows, the next rows of x and the
// residual on their way into a ring of `stages` slots of shared memory (a bulk
// copy each) while one row is worked on in registers.  The copies move the
// granules around a row, so rows may start anywhere (VEC = 1 then reads single
// elements from shared memory).  Bound by memory: 16384 x 8192 bf16 with a
// residual, 8-bit output, 168 us = 5.6 TB/s, 87 % of a plain copy's rate, against
// 178 to 309 us a row a block.  With VEC = 1 single elements' instructions are the
// cost (8191 columns: 336 us); norm_shifted_kernel takes most such rows.
template <typename T, int VEC, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
    norm_stream_kernel(const NormArgs a, int stages, uint32_t slot_bytes) {
    extern __shared__ __align__(128) uint8_t slots[];
    __shared__ __align__(8) uint64_t bar[MAX_STAGES];
    __shared__ float2 red[2][32];
    using P = Pack<T, VEC>;
    const int n = blockDim.x, tid = threadIdx.x;
    const long long step = gridDim.x;
    const RowRing ring{slots, bar, stages, slot_bytes, slot_bytes * (a.res ? 2 : 1), (uint32_t)a.cols * (uint32_t)sizeof(T)};
    if (tid == 0) {
        for (int s = 0; s < stages; s++) mbar_init(&bar[s], 1);
        fence_mbar_init();
    }
    __syncthreads();
    long long row = blockIdx.x;
    if (tid == 0)
        for (int s = 0; s < stages; s++)
            if (row + s * step < a.rows) ring.load<T>(a, row + s * step, s);
    P pw[NV];
    if (a.w) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * n + tid) * VEC;
            if (c < a.cols) pw[i] = *reinterpret_cast<const P*>(static_cast<const T*>(a.w) + c);
        }
    }
    int s = 0, flip = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (; row < a.rows; row += step) {
        ok = mbar_wait(&bar[s], parity, &norm_err, RK_DEV_TIMEOUT_FULL);
        const uint8_t* slot = slots + (size_t)s * ring.stage_bytes;
        const T* x = reinterpret_cast<const T*>(slot + (VEC == 1 ? (uint32_t)((a.xoff + row * a.ldx * sizeof(T)) & 15) : 0));
        const T* r = reinterpret_cast<const T*>(slot + slot_bytes +
                                                (VEC == 1 ? (uint32_t)((a.roff + row * a.ldr * sizeof(T)) & 15) : 0));
        float hw[NV][VEC];
        RowPart<T, VEC> p;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * n + tid) * VEC;
            if (c < a.cols) {
                P px = *reinterpret_cast<const P*>(x + c), pr;
                if (a.res) pr = *reinterpret_cast<const P*>(r + c);
                p.add(px, pr, pw[i], a.res, a.w, a.sum && ok ? static_cast<T*>(a.sum) + row * a.lds + c : nullptr, hw[i]);
            }
        }
        ok = p.reduce_block(red[flip], ok);
        flip ^= 1;
        if (!ok) break;  // the same for the whole block
        if (tid == 0 && row + stages * step < a.rows) ring.load<T>(a, row + stages * step, s);
        if (++s == stages) { s = 0; parity ^= 1; }
        const RowFactors f(a, p.ss, p.top);
        if (a.q && tid == 0) a.scale[row] = f.scale;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * n + tid) * VEC;
            if (c < a.cols) store_part<T, VEC>(a, row, c, hw[i], f);
        }
    }
    if (!ok && tid == 0) ring.drain(a, row, step, s, parity);
}

// norm_stream_kernel for rows off the 16-byte grid.  Elements are worked on where
// they lie, in vectors that are aligned in x, the residual, the sum and y, all of
// which begin at the same place within 16 bytes.  A block's rows are a multiple of
// 8 rows apart, so each begins `skip` elements into its first vector.  The 8-bit
// rows lie on a grid of their own: a lane puts the rest of its vector's codes and
// the start of its right neighbour's together, and only the seams between warps go
// out by single bytes.  Against single elements, with a residual and 8-bit output:
// 16384 x 8185 bf16 217 us (4.3 TB/s) for 336, 8000 x 8001 f32 136 for 208, 16384 x
// 4001 f16 113 for 178; 16384 x 8191 bf16, one block an SM, 295 for 336.
template <typename T, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
    norm_shifted_kernel(const NormArgs a, int stages, uint32_t slot_bytes) {
    constexpr int VEC = 16 / sizeof(T);
    extern __shared__ __align__(128) uint8_t slots[];
    __shared__ __align__(8) uint64_t bar[MAX_STAGES];
    __shared__ float2 red[2][32];
    using P = Pack<T, VEC>;
    const int tid = threadIdx.x, lane = tid & 31;
    const int first = tid / 32 * (32 * NV) + lane;  // a warp's vectors lie together
    const long long step = gridDim.x;
    const RowRing ring{slots, bar, stages, slot_bytes, slot_bytes * (a.res ? 2 : 1), (uint32_t)a.cols * (uint32_t)sizeof(T)};
    const int skip = (int)((a.xoff + (long long)blockIdx.x * a.ldx * (long long)sizeof(T)) & 15) / (int)sizeof(T);
    if (tid == 0) {
        for (int s = 0; s < stages; s++) mbar_init(&bar[s], 1);
        fence_mbar_init();
    }
    __syncthreads();
    long long row = blockIdx.x;
    if (tid == 0)
        for (int s = 0; s < stages; s++)
            if (row + s * step < a.rows) ring.load<T>(a, row + s * step, s);
    P pw[NV];
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const int c = (first + i * 32) * VEC - skip + j;
            pw[i].v[j] = a.w && c >= 0 && c < a.cols ? static_cast<const T*>(a.w)[c] : from_f32<T>(0.f);
        }
    int s = 0, flip = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (; row < a.rows; row += step) {
        ok = mbar_wait(&bar[s], parity, &norm_err, RK_DEV_TIMEOUT_FULL);
        const uint8_t* slot = slots + (size_t)s * ring.stage_bytes;
        float hw[NV][VEC];
        RowPart<T, VEC> p;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = first + i * 32, c = at * VEC - skip;
#pragma unroll
            for (int j = 0; j < VEC; j++) hw[i][j] = 0.f;
            if (c < a.cols) {
                P px = *reinterpret_cast<const P*>(slot + at * 16), pr;
                if (a.res) pr = *reinterpret_cast<const P*>(slot + slot_bytes + at * 16);
                T* sum = a.sum && ok ? static_cast<T*>(a.sum) + row * a.lds + c : nullptr;
                if (c >= 0 && c + VEC <= a.cols) {
                    p.add(px, pr, pw[i], a.res, a.w, sum, hw[i]);
                } else {  // the row's ends: what does not belong to it counts as zeros
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                        if (c + j < 0 || c + j >= a.cols) { px.v[j] = from_f32<T>(0.f); pr.v[j] = from_f32<T>(0.f); }
                    p.add(px, pr, pw[i], a.res, a.w, nullptr, hw[i]);
                    if (sum) {
#pragma unroll
                        for (int j = 0; j < VEC; j++)
                            if (c + j >= 0 && c + j < a.cols)
                                sum[j] = from_f32<T>(to_f32(px.v[j]) + (a.res ? to_f32(pr.v[j]) : 0.f));
                    }
                }
            }
        }
        ok = p.reduce_block(red[flip], ok);
        flip ^= 1;
        if (!ok) break;  // the same for the whole block
        if (tid == 0 && row + stages * step < a.rows) ring.load<T>(a, row + stages * step, s);
        if (++s == stages) { s = 0; parity ^= 1; }
        const RowFactors f(a, p.ss, p.top);
        if (a.q && tid == 0) a.scale[row] = f.scale;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (first + i * 32) * VEC - skip;
            if (a.y && c < a.cols) {
                P o;
                T* y = static_cast<T*>(a.y) + row * a.ldy + c;
#pragma unroll
                for (int j = 0; j < VEC; j++) o.v[j] = from_f32<T>(hw[i][j] * f.y);
                if (c >= 0 && c + VEC <= a.cols) {
                    *reinterpret_cast<P*>(y) = o;
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                        if (c + j >= 0 && c + j < a.cols) y[j] = o.v[j];
                }
            }
        }
        if (!a.q) continue;
        uint64_t own[NV];  // every lane's: its neighbour may need them
#pragma unroll
        for (int i = 0; i < NV; i++) {
            Codes<8> k = {};
            store_codes<VEC>(k.v, hw[i], f.q);
            own[i] = *reinterpret_cast<const uint64_t*>(&k);
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int to = (first + i * 32) * VEC, left = a.cols - to;
            uint64_t next = __shfl_down_sync(0xffffffffu, own[i], 1);
            if (i + 1 < NV) {
                const uint64_t after = __shfl_sync(0xffffffffu, own[i + 1 < NV ? i + 1 : i], 0);
                if (lane == 31) next = after;
            }
            const bool tail = i == NV - 1 && lane == 31, head = i == 0 && lane == 0 && tid > 0;
            uint8_t* q = a.q + row * a.ldq + to;
            uint64_t all = own[i] >> (8 * skip);
            if (skip) all |= next << (8 * (VEC - skip));
            if (!tail && left >= VEC) {
                if constexpr (VEC == 8) *reinterpret_cast<uint64_t*>(q) = all;
                else *reinterpret_cast<uint32_t*>(q) = (uint32_t)all;
            } else if (!tail && left > 0) {
                for (int j = 0; j < left; j++) q[j] = (uint8_t)(all >> (8 * j));
            }
            if (i == 0 || i == NV - 1) {  // the seam between two warps: each stores its own
                const int count = head ? min(skip, left + skip) : tail ? min(left, VEC - skip) : 0;
                uint8_t* at = head ? q - skip : q;
                const uint64_t codes = head ? own[i] : all;
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if (j < count) at[j] = (uint8_t)(codes >> (8 * j));
            }
        }
    }
    if (!ok && tid == 0) ring.drain(a, row, step, s, parity);
}

// Rows that do not fit one block's registers: read twice, the second time from L2.
template <typename T>
__global__ void __launch_bounds__(1024) norm_long_rows_kernel(const NormArgs a) {
    __shared__ float2 red[32];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* r = a.res ? static_cast<const T*>(a.res) + row * a.ldr : nullptr;
    const T* w = static_cast<const T*>(a.w);
    using P = Pack<T, 1>;
    RowPart<T, 1> p;
    float hw[1];
    for (int c = threadIdx.x; c < a.cols; c += 1024)
        p.add(P{x[c]}, r ? P{r[c]} : P{}, w ? P{w[c]} : P{}, r, w, nullptr, hw);
    p.reduce_block(red, true);
    const RowFactors f(a, p.ss, p.top);
    if (a.q && threadIdx.x == 0) a.scale[row] = f.scale;
    RowPart<T, 1> again;
    for (int c = threadIdx.x; c < a.cols; c += 1024) {
        again.add(P{x[c]}, r ? P{r[c]} : P{}, w ? P{w[c]} : P{}, r, w,
                  a.sum ? static_cast<T*>(a.sum) + row * a.lds + c : nullptr, hw);
        store_part<T, 1>(a, row, c, hw, f);
    }
}

// columns that one block holds: 1024 threads x 32 elements
constexpr int MAX_COLS = 32768;

template <typename T, int VEC, int NV, int G>
void launch_group(const NormArgs& a, cudaStream_t st) {
    constexpr int per = 256 / G;
    norm_rows_kernel<T, VEC, NV, G><<<(int)(((long long)a.rows + per - 1) / per), 256, 0, st>>>(a);
}

template <typename T, int VEC, int NV>
void launch_block(const NormArgs& a, int vectors, cudaStream_t st) {
    const int threads = ((vectors + NV - 1) / NV + 31) / 32 * 32;
    norm_rows_kernel<T, VEC, NV, 0><<<a.rows, threads, 0, st>>>(a);
}

// SHIFTED: rows off the 16-byte grid in vectors (VEC elements), as norm_shifted_kernel takes them
template <typename T, int VEC, int NV, int THREADS, bool SHIFTED = false>
cudaError_t launch_stream(const NormArgs& a, int vectors, cudaStream_t st) {
    void (*kernel)(NormArgs, int, uint32_t);
    if constexpr (SHIFTED) kernel = norm_shifted_kernel<T, NV, THREADS>;
    else kernel = norm_stream_kernel<T, VEC, NV, THREADS>;
    static std::atomic<uint64_t> ready{0};  // devices on which the kernel's shared memory is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    const int threads = ((vectors + NV - 1) / NV + 31) / 32 * 32;
    const int slot = (a.cols * (int)sizeof(T) + 15) / 16 * 16 + 16, stage = slot * (a.res ? 2 : 1);
    int ctas = 1024 / threads;  // 64 registers a thread
    while (ctas > 1 && RING_BYTES / ctas < 2 * stage) ctas--;
    int stages = RING_BYTES / ctas / stage;
    stages = stages > MAX_STAGES ? MAX_STAGES : stages;
    long long grid = (long long)ctas * sm_count();
    if (SHIFTED) grid = grid / 8 * 8;  // 8 rows of any length are whole vectors
    kernel<<<(int)(a.rows < grid ? a.rows : grid), threads, (size_t)stages * stage, st>>>(a, stages, (uint32_t)slot);
    return cudaSuccess;
}

template <typename T, int VEC>
cudaError_t launch_vec(const NormArgs& a, cudaStream_t st) {
    const int vectors = (a.cols + VEC - 1) / VEC;
    constexpr int E8 = VEC >= 8 ? 1 : 8 / VEC, E16 = 16 / VEC, E32 = 32 / VEC;  // vectors that make so many elements
    if (a.cols <= 1024) {
        // many short rows: 8 lanes a row keep the reductions few (31000 x 256 f32, 8-bit output: 22.5 us, a warp a row 24.6)
        const bool many = a.rows >= 8 * sm_count();
        if (many && vectors <= 8 * E16) launch_group<T, VEC, E16, 8>(a, st);
        else if (many && vectors <= 16 * E16) launch_group<T, VEC, E16, 16>(a, st);
        else if (vectors <= 32 * E8) launch_group<T, VEC, E8, 32>(a, st);
        else launch_group<T, VEC, E32, 32>(a, st);
        return cudaSuccess;
    }
    const int stage = (a.cols * (int)sizeof(T) + 32) * (a.res ? 2 : 1);
    if (a.rows > 4 * sm_count() && stage <= RING_BYTES) {
        if (vectors <= 512 * E16) return launch_stream<T, VEC, E16, 512>(a, vectors, st);
        if (vectors <= 1024 * E16) return launch_stream<T, VEC, E16, 1024>(a, vectors, st);
    }
    if (vectors <= 1024 * E8) launch_block<T, VEC, E8>(a, vectors, st);
    else if (vectors <= 1024 * E16) launch_block<T, VEC, E16>(a, vectors, st);
    else launch_block<T, VEC, E32>(a, vectors, st);
    return cudaSuccess;
}

template <typename T>
cudaError_t launch(const NormArgs& a, cudaStream_t st) {
    constexpr int VEC = 16 / sizeof(T);
    const bool one = a.rows == 1;
    auto fits = [&](const void* p, long long ld, size_t e) { return aligned(p, VEC * e) && (one || ld % VEC == 0); };
    // rows that begin at the same place within 16 bytes, wherever that is
    auto with_x = [&](const void* p, long long ld) {
        return !p || (((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(a.x)) & 15) == 0 && (ld - a.ldx) % VEC == 0);
    };
    const int most = (a.cols + 2 * VEC - 2) / VEC;  // vectors that a row may touch
    const bool vec = a.cols % VEC == 0 && fits(a.x, a.ldx, sizeof(T)) && fits(a.w, 0, sizeof(T)) &&
                     fits(a.res, a.ldr, sizeof(T)) && fits(a.sum, a.lds, sizeof(T)) && fits(a.y, a.ldy, sizeof(T)) &&
                     fits(a.q, a.ldq, 1);
    if (!vec && a.cols > 1024 && most <= 1024 * (16 / VEC) && a.rows > 4 * sm_count() && with_x(a.res, a.ldr) &&
        with_x(a.sum, a.lds) && with_x(a.y, a.ldy) && (!a.q || (aligned(a.q, VEC) && a.ldq % VEC == 0)))
        return most <= 512 * (16 / VEC) ? launch_stream<T, VEC, 16 / VEC, 512, true>(a, most, st)
                                        : launch_stream<T, VEC, 16 / VEC, 1024, true>(a, most, st);
    if (a.cols <= MAX_COLS) return vec ? launch_vec<T, VEC>(a, st) : launch_vec<T, 1>(a, st);
    norm_long_rows_kernel<T><<<a.rows, 1024, 0, st>>>(a);
    return cudaSuccess;
}

rk_status norm_rows(const NormArgs& a, bool norm, int dtype, void* stream, const char* who) {
    if (!dtype_ok(dtype) || !size_ok(a.rows, 0) || !size_ok(a.cols, 1)) return fail(RK_ERR_CANNOT_IMPLEMENT, who);
    if (a.rows == 0) return RK_OK;
    if (!a.x || (norm && !a.w) || (!a.y && !(a.q && a.scale)) || !pitch_ok(a.ldx, a.rows, a.cols) ||
        (a.res && !pitch_ok(a.ldr, a.rows, a.cols)) || (a.sum && !pitch_ok(a.lds, a.rows, a.cols)) ||
        (a.y && !pitch_ok(a.ldy, a.rows, a.cols)) || (a.q && !pitch_ok(a.ldq, a.rows, a.cols)))
        return fail(RK_ERR_CANNOT_IMPLEMENT, who);
    const size_t e = dtype_bytes(dtype);
    if (!aligned(a.x, e) || !aligned(a.res, e) || !aligned(a.w, e) || !aligned(a.sum, e) || !aligned(a.y, e) ||
        !aligned(a.scale, 4))
        return fail(RK_ERR_CANNOT_IMPLEMENT, who);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    NormArgs b = a;
    b.inv_cols = 1.f / (float)a.cols;
    b.xoff = (uint32_t)(reinterpret_cast<uintptr_t>(a.x) & 15);
    b.roff = (uint32_t)(reinterpret_cast<uintptr_t>(a.res) & 15);
    cudaError_t ce = dtype == RK_DTYPE_F32 ? launch<float>(b, st) : dtype == RK_DTYPE_F16 ? launch<__half>(b, st)
                                                                                          : launch<__nv_bfloat16>(b, st);
    const cudaError_t le = cudaGetLastError();
    if (ce == cudaSuccess) ce = le;
    return ce == cudaSuccess ? RK_OK : fail_cuda_err(RK_ERR_LAUNCH, who, ce);
}

}  // namespace

void* norm_err_word() {
    void* p = nullptr;
    return cudaGetSymbolAddress(&p, norm_err) == cudaSuccess ? p : nullptr;
}

}  // namespace rk

using namespace rk;

extern "C" rk_status rk_rms_norm(const void* x, long long ldx, const void* residual, long long ldr,
                                 const void* weight, void* sum_out, long long lds, void* y, long long ldy, int rows,
                                 int cols, float eps, int dtype, void* stream) {
    NormArgs a{x, residual, weight, sum_out, y, nullptr, nullptr, ldx, ldr, lds, ldy, 0, rows, cols, eps};
    return norm_rows(a, true, dtype, stream, "rk_rms_norm: unsupported arguments");
}

extern "C" rk_status rk_rms_norm_q8(const void* x, long long ldx, const void* residual, long long ldr,
                                    const void* weight, void* sum_out, long long lds, void* q, long long ldq,
                                    float* scale, int rows, int cols, float eps, int dtype, void* stream) {
    NormArgs a{x, residual, weight, sum_out, nullptr, static_cast<uint8_t*>(q), scale, ldx, ldr, lds, 0, ldq,
               rows, cols, eps};
    return norm_rows(a, true, dtype, stream, "rk_rms_norm_q8: unsupported arguments");
}

extern "C" rk_status rk_quantize_q8(const void* x, long long ldx, void* q, long long ldq, float* scale, int rows,
                                    int cols, int dtype, void* stream) {
    NormArgs a{x, nullptr, nullptr, nullptr, nullptr, static_cast<uint8_t*>(q), scale, ldx, 0, 0, 0, ldq,
               rows, cols, 0.f};
    return norm_rows(a, false, dtype, stream, "rk_quantize_q8: unsupported arguments");
}
