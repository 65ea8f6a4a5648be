// Status plumbing of the C ABI: CUDA errors become syn_status values and the
// message is kept per thread for syn_last_error().
#include "common.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include <cstdio>
#include <cstring>
#include <mutex>
#include <utility>
#include <vector>

namespace {
thread_local char g_last_error[256] = "";
thread_local int g_pdl = 0;
}

int syn_pdl_enabled() { return g_pdl; }
void syn_set_pdl(int on) { g_pdl = on; }
// For microbenchmarks that capture kernels as the session does.
extern "C" void syn_set_programmatic_launch(int on) { g_pdl = on; }

int syn_cuda_status(cudaError_t e) {
    if (e == cudaSuccess) return SYN_OK;
    std::snprintf(g_last_error, sizeof g_last_error, "%s: %s", cudaGetErrorName(e), cudaGetErrorString(e));
    return e == cudaErrorMemoryAllocation ? SYN_ERR_NO_MEMORY : SYN_ERR_CUDA;
}

int syn_check_launch() { return syn_cuda_status(cudaGetLastError()); }

void syn_set_error(const char* msg) { std::snprintf(g_last_error, sizeof g_last_error, "%s", msg); }

int syn_num_sms() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    return n;
}

// cuTensorMapEncodeTiled from the driver (looked up once; no libcuda link).
PFN_cuTensorMapEncodeTiled_v12000 syn_tensor_map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
        else
            cudaGetLastError();
    });
    return fn;
}

// The dynamic shared memory opt-in of a kernel, once per device.
int syn_opt_in_smem(const void* kernel, size_t bytes) {
    static std::mutex mu;
    static std::vector<std::pair<const void*, int>> done;
    int dev = 0;
    int st = syn_cuda_status(cudaGetDevice(&dev));
    if (st) return st;
    std::lock_guard<std::mutex> lock(mu);
    for (const auto& d : done)
        if (d.first == kernel && d.second == dev) return SYN_OK;
    st = syn_cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
    if (!st) done.push_back({kernel, dev});
    return st;
}

extern "C" const char* syn_build_info(void) { return "synapse_b200 0.1 sm_100a"; }

extern "C" const char* syn_last_error(void) { return g_last_error; }

extern "C" const char* syn_status_string(int status) {
    switch (status) {
    case SYN_OK: return "ok";
    case SYN_ERR_INVALID: return "invalid argument";
    case SYN_ERR_UNSUPPORTED: return "unsupported";
    case SYN_ERR_CUDA: return "cuda error";
    case SYN_ERR_NO_MEMORY: return "out of device memory";
    case SYN_ERR_TIMEOUT: return "timeout";
    case SYN_ERR_NCCL: return "nccl error";
    case SYN_ERR_FORMAT: return "bad format";
    case SYN_ERR_RANGE: return "out of range";
    default: return "unknown";
    }
}
