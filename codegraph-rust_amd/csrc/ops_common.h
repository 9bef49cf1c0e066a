// ops_common.h - what the entry points of q4scan.hip, lookup.hip and softmax.hip share: error reporting, the device a call
// runs on, 16-bit conversions. These calls enqueue on the CALLER's stream and leave the thread's current device as they found it.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <exception>
#include <new>
#include <string>

#include "../../include/cgvec.h"
#include "common.h"
#include "use_device.h"

extern "C" int cgv_set_error_(int code, const char* msg);  // abi.hip (shared thread-local message)

namespace cgv_ops {

inline int fail(int code, const std::string& m) { return cgv_set_error_(code, m.c_str()); }

#define OPCHK(expr)                                                                             \
    do {                                                                                        \
        hipError_t _e = (expr);                                                                 \
        if (_e != hipSuccess) {                                                                 \
            (void)hipGetLastError();                                                            \
            return cgv_ops::fail(_e == hipErrorOutOfMemory ? CGV_ERR_OOM : CGV_ERR_HIP,         \
                                 std::string(#expr) + ": " + hipGetErrorString(_e));            \
        }                                                                                       \
    } while (0)

// the body of a C entry: nothing is thrown across the boundary
template <class F>
int guarded(F&& body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return cgv_set_error_(CGV_ERR_OOM, "out of host memory");
    } catch (const std::exception& e) {
        return cgv_set_error_(CGV_ERR_INTERNAL, e.what());
    } catch (...) {
        return cgv_set_error_(CGV_ERR_INTERNAL, "unexpected exception");
    }
}

inline int need_gpu(int device_id) {
    static const int n = cgv_device_count();   // does not change while a process lives
    if (n == 0) return fail(CGV_ERR_HIP, "no HIP device visible: libcgvec_hip has no CPU fallback");
    if (device_id < 0 || device_id >= n) return fail(CGV_ERR_INVALID_ARG, "device_id out of range");
    return CGV_OK;
}

// makes `device` current for a call and gives the thread its own device back afterwards
struct DeviceScope {
    int before = -1, device;
    explicit DeviceScope(int d) : device(d) {
        if (hipGetDevice(&before) != hipSuccess) {
            (void)hipGetLastError();
            before = -1;
        }
    }
    hipError_t enter() { return cgv::use_device(device); }
    ~DeviceScope() {
        if (before >= 0 && before != device) (void)hipSetDevice(before);
    }
};

// a kernel's limit of dynamic LDS, raised once per device (it is a property of the kernel on a device); one object per kernel
struct LdsLimit {
    std::atomic<uint64_t> done{0};
    hipError_t raise(const void* kernel, int device, int bytes) {
        const uint64_t bit = 1ull << (device & 63);
        if (device < 64 && (done.load(std::memory_order_acquire) & bit)) return hipSuccess;
        const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == hipSuccess && device < 64) done.fetch_or(bit, std::memory_order_release);
        return e;
    }
};

// a grid of any number of workgroups: a launch holds less than 2^32 threads in each direction, so the second one takes over
constexpr uint64_t MOST_BLOCKS = 65535ull << 20;
inline dim3 wide_grid(uint64_t blocks) {
    const uint64_t x = std::min<uint64_t>(blocks, 1u << 20);
    return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
__device__ inline uint64_t wide_block() { return (uint64_t)blockIdx.y * gridDim.x + blockIdx.x; }   // may be beyond the last one

// 16-bit value -> f32 by storage type (CGV_DTYPE_BF16 / CGV_DTYPE_FP16)
template <int DT>
__device__ inline float half_to_f32(uint16_t v) {
    return DT == cgv::DT_BF16 ? cgv::bf16_to_f32(v) : cgv::f16_to_f32(v);
}
template <int DT>
__device__ inline uint16_t f32_to_half(float v) {
    return DT == cgv::DT_BF16 ? cgv::f32_to_bf16_rne(v) : cgv::f32_to_f16_rne(v);
}
template <int DT>
__device__ inline float load_elem(const void* p, uint64_t i) {
    if (DT == cgv::DT_F32) return ((const float*)p)[i];
    return half_to_f32<DT>(((const uint16_t*)p)[i]);
}
template <int DT>
__device__ inline void store_elem(void* p, uint64_t i, float v) {
    if (DT == cgv::DT_F32)
        ((float*)p)[i] = v;
    else
        ((uint16_t*)p)[i] = f32_to_half<DT>(v);
}

// calls f.template operator()<DT>() for the storage type `dtype`
template <class F>
int by_dtype(int dtype, F&& f) {
    switch (dtype) {
        case CGV_DTYPE_F32: return f(std::integral_constant<int, cgv::DT_F32>());
        case CGV_DTYPE_BF16: return f(std::integral_constant<int, cgv::DT_BF16>());
        case CGV_DTYPE_FP16: return f(std::integral_constant<int, cgv::DT_FP16>());
    }
    return fail(CGV_ERR_INVALID_ARG, "dtype must be f32, bf16 or fp16");
}
inline uint32_t esize(int dtype) { return dtype == CGV_DTYPE_F32 ? 4u : 2u; }

}  // namespace cgv_ops
