// quant.cuh -- element types, vector access and reductions shared by the
// quantised-serving operators (rms_norm.cu, linear_q8.cu, linear_q4.cu).
//
// Activations come as float, half or bfloat16 (rk_dtype); every sum, norm and
// scale is held in 32 bits and rounded once when a result is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

#include "../../include/rk_b200.h"

namespace rk {

constexpr float Q8_MAX = 448.0f;      // largest finite e4m3 value
constexpr float AMAX_FLOOR = 1e-30f;  // smallest row maximum that sets a scale: 1 / scale stays finite

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Scale vectors come in any of the three types; the choice is uniform over a launch.
__device__ __forceinline__ float load_as_f32(const void* p, size_t i, int dtype) {
    if (dtype == RK_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == RK_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// max that keeps NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// SM count of the current device (148 when it cannot be asked)
int sm_count();

// Device addresses of the error words of the operators' bounded waits, on the current device.
void* norm_err_word();
void* q8_err_word();
void* q4_err_word();

inline size_t dtype_bytes(int dtype) { return dtype == RK_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == RK_DTYPE_F32 || dtype == RK_DTYPE_F16 || dtype == RK_DTYPE_BF16; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
// Rows and columns up to 2^30: the kernels' 32-bit indices may step past an end by a tile or a block's width.
inline bool size_ok(int n, int least) { return n >= least && n <= 1 << 30; }
// a row pitch that holds `cols` elements (the pitch of a single row is never used)
inline bool pitch_ok(long long ld, int rows, int cols) { return rows <= 1 || ld >= cols; }

}  // namespace rk
