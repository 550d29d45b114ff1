// linear_q8.cu -- the linear layer on 8-bit (e4m3) rows with a scale each:
//
//   y[m][n] = sx[m] sw[n] sum_k xq[m][k] wq[n][k] + bias[n] + residual[m][n]
#include <cuda_fp8.h>

#include "quant.cuh"
#include "status.h"

namespace rk {
namespace {

struct Q8Args {
    const uint8_t *x, *w;
    const float *sx, *sw, *bias;
    const void* res;
    void* y;
    long long ldx, ldw, ldr, ldy;
    int rows, n, k;
};

__device__ __forceinline__ float q8_value(uint8_t q) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3)));
}

// Simple form: 16 x 16 outputs per block, both operands through shared memory.
template <typename T>
__global__ void __launch_bounds__(256) linear_q8_kernel(const Q8Args a) {
    __shared__ float xs[16][17], ws[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const long long n0 = (long long)blockIdx.x * 16;
    for (long long m0 = (long long)blockIdx.y * 16; m0 < a.rows; m0 += (long long)gridDim.y * 16) {
        float acc = 0.f;
        for (int k0 = 0; k0 < a.k; k0 += 16) {
            const bool kin = k0 + tx < a.k;
            xs[ty][tx] = kin && m0 + ty < a.rows ? q8_value(a.x[(m0 + ty) * a.ldx + k0 + tx]) : 0.f;
            ws[ty][tx] = kin && n0 + ty < a.n ? q8_value(a.w[(n0 + ty) * a.ldw + k0 + tx]) : 0.f;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 16; i++) acc += xs[ty][i] * ws[tx][i];
            __syncthreads();
        }
        const long long m = m0 + ty, n = n0 + tx;
        if (m < a.rows && n < a.n) {
            float v = acc * a.sx[m] * a.sw[n];
            if (a.bias) v += a.bias[n];
            if (a.res) v += to_f32(static_cast<const T*>(a.res)[m * a.ldr + n]);
            static_cast<T*>(a.y)[m * a.ldy + n] = from_f32<T>(v);
        }
    }
}

template <typename T>
void launch(const Q8Args& a, cudaStream_t st) {
    const int gy = (a.rows + 15) / 16;
    linear_q8_kernel<T><<<dim3((a.n + 15) / 16, gy < 65535 ? gy : 65535), 256, 0, st>>>(a);
}

__device__ uint32_t q8_err;  // set when a bounded wait of a kernel gives up

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
    Q8Args a{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(w), x_scale, w_scale, bias, residual, y,
             ldx, ldw, ldr, ldy, rows, n, k};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case RK_DTYPE_F32: launch<float>(a, st); break;
        case RK_DTYPE_F16: launch<__half>(a, st); break;
        default: launch<__nv_bfloat16>(a, st); break;
    }
    const cudaError_t ce = cudaGetLastError();
    return ce == cudaSuccess ? RK_OK : fail_cuda_err(RK_ERR_LAUNCH, "rk_linear_q8", ce);
}
