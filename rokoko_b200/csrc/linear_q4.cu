// linear_q4.cu -- the linear layer with 4-bit weights in groups along the
// reduction, for few rows, and the quantiser that makes such weights:
//
//   y[m][n] = sum_g s[n][g] sum_{k in g} (q[n][k] - z[n][g]) x[m][k] + bias[n] + residual[m][n]
//
// Byte j of a weight row holds columns 2j (low half) and 2j + 1 (high half).
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
};

// Simple form: one warp per weight row, activation rows one after the other.
template <typename T>
__global__ void __launch_bounds__(256) linear_q4_kernel(const Q4Args a) {
    const int n = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (n >= a.n) return;
    const uint8_t* w = a.w + n * a.ldw;
    for (long long m = blockIdx.y; m < a.rows; m += gridDim.y) {
        const T* x = static_cast<const T*>(a.x) + m * a.ldx;
        float acc = 0.f;
        for (int k = lane; k < a.k; k += 32) {
            const size_t g = (size_t)n * a.groups + k / a.group;
            const int q = (w[k >> 1] >> (k & 1) * 4) & 15, z = a.z ? a.z[g] : Q4_ZERO;
            acc += load_as_f32(a.s, g, a.s_dtype) * (float)(q - z) * to_f32(x[k]);
        }
        for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
        if (lane == 0) {
            if (a.bias) acc += a.bias[n];
            if (a.res) acc += to_f32(static_cast<const T*>(a.res)[m * a.ldr + n]);
            static_cast<T*>(a.y)[m * a.ldy + n] = from_f32<T>(acc);
        }
    }
}

template <typename T>
void launch(const Q4Args& a, cudaStream_t st) {
    linear_q4_kernel<T><<<dim3((a.n + 7) / 8, a.rows < 65535 ? a.rows : 65535), 256, 0, st>>>(a);
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
             group, (int)(((long long)k + group - 1) / group), scale_dtype};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case RK_DTYPE_F32: launch<float>(a, st); break;
        case RK_DTYPE_F16: launch<__half>(a, st); break;
        default: launch<__nv_bfloat16>(a, st); break;
    }
    const cudaError_t ce = cudaGetLastError();
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
