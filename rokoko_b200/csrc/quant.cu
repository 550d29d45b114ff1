// quant.cu -- what the quantised-serving operators share on the host: the SM
// count, and rk_linear_check, which reads the device error words of their
// bounded waits.
#include "quant.cuh"

#include <atomic>
#include <cstdio>

#include "status.h"

namespace rk {

int sm_count() {
    static std::atomic<int> cache[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int n = cache[dev].load(std::memory_order_relaxed);
    if (!n) {
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        cache[dev].store(n = n > 0 ? n : 148, std::memory_order_relaxed);
    }
    return n;
}

}  // namespace rk

extern "C" rk_status rk_linear_check(void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    void* words[] = {rk::norm_err_word(), rk::q8_err_word(), rk::q4_err_word()};
    uint32_t seen = 0;
    for (void* p : words) {
        uint32_t e = 0;
        if (!p) return rk::fail_cuda(RK_ERR_CUDA, "rk_linear_check: cudaGetSymbolAddress");
        if (cudaMemcpyAsync(&e, p, 4, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
            cudaStreamSynchronize(st) != cudaSuccess)
            return rk::fail_cuda(RK_ERR_CUDA, "rk_linear_check");
        if (e && (cudaMemsetAsync(p, 0, 4, st) != cudaSuccess || cudaStreamSynchronize(st) != cudaSuccess))
            return rk::fail_cuda(RK_ERR_CUDA, "rk_linear_check: clearing the error word");
        if (e) seen = e;
    }
    if (seen) {
        char buf[96];
        snprintf(buf, sizeof buf, "device wait timed out (code %u)", seen);
        return rk::fail(RK_ERR_DEVICE_TIMEOUT, buf);
    }
    return RK_OK;
}
