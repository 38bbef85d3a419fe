// Error reporting and device queries shared by every entry point.
#include <stdarg.h>
#include <stdio.h>

#include <mutex>

#include "common.cuh"

namespace p2p {

static thread_local char g_error[1024] = "";

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
    return code;
}

int launch_status(const char* what) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(P2P_ECUDA, "%s: %s", what, cudaGetErrorString(e));
    return P2P_OK;
}

// The limit belongs to the kernel and the device, not to the call, so it only ever rises: a smaller request of another
// thread must not take it away between a call's own request and its launch. What was asked so far is kept in a table of
// open addresses (no allocation that could throw across the C ABI); with the table full a request sets the limit itself.
namespace {
struct SmemLimit {
    const void* kernel;
    int device, bytes;
};
constexpr int kSmemLimits = 4096;
SmemLimit g_smem_limits[kSmemLimits];
std::mutex g_smem_mu;
}  // namespace

int allow_smem(const void* kernel, int bytes, const char* what) {
    if (bytes <= 48 * 1024) return P2P_OK;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return fail(P2P_ECUDA, "%s: %s", what, cudaGetErrorString(e));
    const std::lock_guard<std::mutex> lock(g_smem_mu);
    SmemLimit* at = nullptr;
    const uintptr_t start = (reinterpret_cast<uintptr_t>(kernel) >> 4) * 31 + (uintptr_t)dev;
    for (int i = 0; i < kSmemLimits && !at; ++i) {
        SmemLimit* slot = &g_smem_limits[(start + i) % kSmemLimits];
        if (!slot->kernel || (slot->kernel == kernel && slot->device == dev)) at = slot;
    }
    if (at && at->kernel && at->bytes >= bytes) return P2P_OK;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return fail(P2P_ECUDA, "%s: %d bytes of shared memory: %s", what, bytes, cudaGetErrorString(e));
    if (at) *at = {kernel, dev, bytes};
    return P2P_OK;
}

int sm_count() {
    static int counts[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (counts[dev] == 0) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        counts[dev] = n;
    }
    return counts[dev];
}

}  // namespace p2p

extern "C" const char* p2p_last_error(void) { return p2p::g_error; }
extern "C" int p2p_abi_version(void) { return 1; }
