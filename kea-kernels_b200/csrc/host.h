// host.h - what the host sides of the library's translation units share: the one-time set-up of a device, the tensor
// map encoder and the library's device error word. Defined in kea_lowbit.cu.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace kea_host {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// What a launch on the current device needs.
struct Device {
    int index = 0;
    int sms = 148;
    uint32_t *error_word = nullptr;   // device address of the library's own error word
    EncodeTiledFn encode = nullptr;
};

// The current device, set up (KEA_OK), or the status that says why not (KEA_ERR_CAPTURE inside a first-use capture).
int device(Device *out, void *stream);

// The 8-bit GEMM's kernel attributes, set once per device with that device current.
int setup_int8_gemm();

inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
inline bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace kea_host
