// operators.cu -- the device a handle-less operator runs on, and the check of
// what its kernels recorded.
#include "operators.h"

#include <atomic>

namespace gtmoe {

static bool sm100(int device) {
    static std::atomic<int> known[64];  // 0 not asked yet, 1 no, 2 yes
    const int slot = device & 63;
    int v = device < 64 ? known[slot].load(std::memory_order_relaxed) : 0;
    if (!v) {
        int major = 0;
        if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device) != cudaSuccess) {
            cudaGetLastError();
            return false;
        }
        v = major == 10 ? 2 : 1;
        if (device < 64) known[slot].store(v, std::memory_order_relaxed);
    }
    return v == 2;
}

int DeviceScope::enter(std::initializer_list<DevArg> args) {
    for (const DevArg &a : args)
        if ((uintptr_t)a.p % a.align)
            return fail(GTMOE_EINVAL, "%s must start on a multiple of its elements' %zu bytes", a.name, a.align);
    const char *first = nullptr;
    for (const DevArg &a : args) {
        if (!a.p) continue;
        cudaPointerAttributes at;
        const cudaError_t e = cudaPointerGetAttributes(&at, a.p);
        if (e != cudaSuccess) {
            cudaGetLastError();
            int n = 0;
            if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
                cudaGetLastError();
                return fail(GTMOE_ENODEVICE, "no CUDA device");
            }
            return fail(GTMOE_EINVAL, "%s must be device memory", a.name);
        }
        if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
            return fail(GTMOE_EINVAL, "%s must be device memory", a.name);
        if (device_ < 0) {
            device_ = at.device;
            first = a.name;
        } else if (at.device != device_ && at.type == cudaMemoryTypeDevice) {
            return fail(GTMOE_EINVAL, "%s is on device %d but %s is on device %d", a.name, at.device, first, device_);
        }
    }
    if (device_ < 0) return 0;
    if (!sm100(device_))
        return fail(GTMOE_ENODEVICE, "device %d is not an sm_100 device; libgtmoe.so is built for sm_100a only", device_);
    int now = -1;
    GT_CUDA(cudaGetDevice(&now));
    if (now != device_) {
        GT_CUDA(cudaSetDevice(device_));
        previous_ = now;
    }
    return 0;
}

}  // namespace gtmoe

using namespace gtmoe;

extern "C" int gtmoe_operators_check(int device) {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || device < 0 || device >= n) {
        cudaGetLastError();
        return fail(GTMOE_ENODEVICE, "device %d does not exist", device);
    }
    int before = 0, code = 0;
    GT_CUDA(cudaGetDevice(&before));
    GT_CUDA(cudaSetDevice(device));
    int norm = 0;
    int rc = grouped_take_error(&code);
    if (rc == 0) rc = norm_take_error(&norm);
    cudaSetDevice(before);
    GT_CHECK(rc);
    if (norm != 0) return fail(GTMOE_ETIMEOUT, "layer norm: a kernel gave up waiting (barrier %d); results are invalid", norm);
    if (code == kErrBadCounts)
        return fail(GTMOE_EINVAL, "grouped product: a group had a negative count, or the counts' sum was above the rows; "
                                  "the call's results are invalid");
    if (code != 0) return fail(GTMOE_ETIMEOUT, "grouped product: a kernel gave up waiting (barrier %d); results are invalid", code);
    return 0;
}
