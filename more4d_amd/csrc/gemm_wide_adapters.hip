// gemm_bt256w_kernel (gemm_wide.h) with the low-rank adapters' extension and the M4D_EPI_STORE epilogue; adapters.hip dispatches here
#include "gemm_wide.h"

extern "C" __attribute__((visibility("hidden"))) int m4d_launch_gemm_wide_adapters(const void* args, unsigned nwg, hipStream_t st) {
    static PerDeviceOnce configured;
    if (configured.pending()) {
        if (hipFuncSetAttribute((const void*)gemm_bt256w_kernel<0, M4D_EPI_STORE, false, true>, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * W_BUF) != hipSuccess)
            return -3;
        configured.mark();
    }
    hipLaunchKernelGGL((gemm_bt256w_kernel<0, M4D_EPI_STORE, false, true>), dim3(nwg), dim3(256), 2 * W_BUF, st, *(const GemmAdArgs*)args);
    return 0;
}
