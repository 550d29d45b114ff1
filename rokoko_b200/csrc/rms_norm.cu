// rms_norm.cu -- root-mean-square norm with the residual's addition, its output
// in the input's type or in 8 bits with a scale for each row, and the same
// 8-bit rows without the norm.
//
//   h = x + residual            (32 bit)
//   y = h / sqrt(mean(h^2) + eps) * w
//   q = e4m3(y / s),  s = max(max|y|, 1e-30) / 448
#include <cuda_fp8.h>

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
};

// Simple form: one block per row, the row read twice.
template <typename T, bool NORM>
__global__ void __launch_bounds__(256) norm_rows_kernel(const NormArgs a) {
    __shared__ float red_s[8], red_m[8];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* r = a.res ? static_cast<const T*>(a.res) + row * a.ldr : nullptr;
    const T* w = static_cast<const T*>(a.w);
    float ss = 0.f, top = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
        const float h = to_f32(x[c]) + (r ? to_f32(r[c]) : 0.f);
        ss += h * h;
        top = max_nan(top, fabsf(NORM ? h * to_f32(w[c]) : h));
    }
    for (int o = 16; o; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if ((threadIdx.x & 31) == 0) { red_s[threadIdx.x >> 5] = ss; red_m[threadIdx.x >> 5] = top; }
    __syncthreads();
    ss = top = 0.f;
    for (int i = 0; i < 8; i++) { ss += red_s[i]; top = max_nan(top, red_m[i]); }
    const float inv = NORM ? rsqrtf(ss / (float)a.cols + a.eps) : 1.f;
    const float s = max_nan(top * inv, AMAX_FLOOR) / Q8_MAX, is = 1.f / s;
    if (a.q && threadIdx.x == 0) a.scale[row] = s;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
        const float h = to_f32(x[c]) + (r ? to_f32(r[c]) : 0.f);
        const float y = NORM ? h * inv * to_f32(w[c]) : h;
        if (a.sum) static_cast<T*>(a.sum)[row * a.lds + c] = from_f32<T>(h);
        if (a.y) static_cast<T*>(a.y)[row * a.ldy + c] = from_f32<T>(y);
        if (a.q) a.q[row * a.ldq + c] = __nv_cvt_float_to_fp8(y * is, __NV_SATFINITE, __NV_E4M3);
    }
}

template <typename T>
void launch(const NormArgs& a, bool norm, cudaStream_t st) {
    if (norm) norm_rows_kernel<T, true><<<a.rows, 256, 0, st>>>(a);
    else norm_rows_kernel<T, false><<<a.rows, 256, 0, st>>>(a);
}

rk_status norm_rows(const NormArgs& a, bool norm, int dtype, void* stream, const char* who) {
    if (!dtype_ok(dtype) || a.rows < 0 || a.cols < 1) return fail(RK_ERR_CANNOT_IMPLEMENT, who);
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
    switch (dtype) {
        case RK_DTYPE_F32: launch<float>(a, norm, st); break;
        case RK_DTYPE_F16: launch<__half>(a, norm, st); break;
        default: launch<__nv_bfloat16>(a, norm, st); break;
    }
    const cudaError_t e2 = cudaGetLastError();
    return e2 == cudaSuccess ? RK_OK : fail_cuda_err(RK_ERR_LAUNCH, who, e2);
}

}  // namespace
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
