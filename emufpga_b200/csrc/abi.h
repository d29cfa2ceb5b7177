// Shared by the translation units that implement C ABI entry points: every
// entry point runs its body under guarded(), which turns a thrown Error into
// its status code and the thread's spm_last_error() message.
#pragma once
#include <cuda_runtime_api.h>

#include <atomic>
#include <exception>
#include <new>
#include <string>

#include "common.h"

#define CUDA_OK(expr)                                                                        \
    do {                                                                                     \
        cudaError_t e_ = (expr);                                                             \
        if (e_ != cudaSuccess) spm::fail(SPM_E_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e_)); \
    } while (0)

namespace spm {

template <class F>
spm_status guarded(F&& f) {
    try {
        f();
        return SPM_OK;
    } catch (const Error& e) {
        set_error(e.msg);
        return e.code;
    } catch (const std::bad_alloc&) {
        set_error("host allocation failed");
        return SPM_E_ARG;
    } catch (const std::exception& e) {
        set_error(e.what());
        return SPM_E_ARG;
    }
}

struct DeviceBuf {
    void* p = nullptr;
    DeviceBuf() = default;
    DeviceBuf(const DeviceBuf&) = delete;
    DeviceBuf& operator=(const DeviceBuf&) = delete;
    ~DeviceBuf() { if (p) cudaFree(p); }
};

// Makes `device` current for the life of the object and then puts back the
// caller's.  SPM_E_NO_DEVICE where no device is visible.
struct DeviceScope {
    int before = -1;
    explicit DeviceScope(int device) {
        static std::atomic<int> devices{0};
        int n = devices;
        if (n == 0) {
            if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
                cudaGetLastError();
                fail(SPM_E_NO_DEVICE, "no CUDA device is visible");
            }
            devices = n;
        }
        if (device < 0 || device >= n) fail(SPM_E_ARG, "device index out of range");
        CUDA_OK(cudaGetDevice(&before));
        if (before != device) CUDA_OK(cudaSetDevice(device));
        else before = -1;
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    ~DeviceScope() { if (before >= 0) cudaSetDevice(before); }
};

// The multiprocessors of the current device (asked for once per device).
inline int device_sms() {
    static std::atomic<int> sms[64] = {};
    int d = 0;
    CUDA_OK(cudaGetDevice(&d));
    if (d < 64 && sms[d]) return sms[d];
    int v = 0;
    CUDA_OK(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, d));
    if (d < 64) sms[d] = v;
    return v;
}

// Raises a kernel's dynamic shared memory limit on the current device, once
// per device (`done` is the kernel's own bit per device).
template <class K>
void allow_smem(K kernel, size_t bytes, std::atomic<unsigned long long>& done) {
    int d = 0;
    CUDA_OK(cudaGetDevice(&d));
    if (d < 64 && (done >> d & 1)) return;
    CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
    if (d < 64) done |= 1ull << d;
}

// Likewise for clusters of more than eight CTAs.
template <class K>
void allow_wide_clusters(K kernel, std::atomic<unsigned long long>& done) {
    int d = 0;
    CUDA_OK(cudaGetDevice(&d));
    if (d < 64 && (done >> d & 1)) return;
    CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (d < 64) done |= 1ull << d;
}

}  // namespace spm
