// operator_common.cuh - device pieces shared by the 8-bit GEMM, the residual-norm and the beam-search kernels: element
// types, their conversions and the error report.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kea_lowbit.h"
#include "ptx.cuh"

namespace kea {

template <typename T> struct TypeCode;
template <> struct TypeCode<float> { static constexpr int value = KEA_TYPE_F32; };
template <> struct TypeCode<__half> { static constexpr int value = KEA_TYPE_F16; };
template <> struct TypeCode<__nv_bfloat16> { static constexpr int value = KEA_TYPE_BF16; };

KEA_DEVI float to_float(float v) { return v; }
KEA_DEVI float to_float(__half v) { return __half2float(v); }
KEA_DEVI float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> KEA_DEVI T from_float(float v);
template <> KEA_DEVI float from_float<float>(float v) { return v; }
template <> KEA_DEVI __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> KEA_DEVI __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two values rounded to nearest even and packed, `lo` in the lower half.
template <typename T> KEA_DEVI uint32_t pack2(float lo, float hi);
template <> KEA_DEVI uint32_t pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> KEA_DEVI uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <typename T> KEA_DEVI float2 unpack2(uint32_t w);
template <> KEA_DEVI float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
template <> KEA_DEVI float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// float has no 16-bit packing; there for code that names it, never called
template <> KEA_DEVI uint32_t pack2<float>(float, float) { return 0u; }
template <> KEA_DEVI float2 unpack2<float>(uint32_t) { return make_float2(0.f, 0.f); }

constexpr long long kOpWaitBudget = 4000000000LL;   // SM clocks (about 2 s) before a wait gives up

KEA_DEVI void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
KEA_DEVI uint4 ld_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

KEA_DEVI ulonglong2 ld_shared_pairs(uint32_t addr) {
    ulonglong2 v;
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(v.x), "=l"(v.y) : "r"(addr) : "memory");
    return v;
}

// Two FP32 values in one 64-bit register: packed multiplications and additions, each rounded as the scalar ones.
KEA_DEVI uint64_t pair_of(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
KEA_DEVI void unpair(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
KEA_DEVI uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
KEA_DEVI uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
KEA_DEVI uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

KEA_DEVI void report_error(uint32_t *word, uint32_t bits) { atomicOr(word, bits); }

}  // namespace kea
