// use_device.h - how an entry point starts its GPU work.
#pragma once
#include <hip/hip_runtime.h>

namespace cgv {

// Makes `device` current. An error that an EARLIER HIP call of the same thread left unread (a hipHostRegister that the system
// refused, a failed call of another library) is dropped: the launches that follow are checked with hipGetLastError and must
// not report somebody else's failure as their own.
inline hipError_t use_device(int device) {
    (void)hipGetLastError();
    return hipSetDevice(device);
}

}  // namespace cgv
