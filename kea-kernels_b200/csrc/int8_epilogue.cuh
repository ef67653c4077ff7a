// int8_epilogue.cuh - what every 8-bit GEMM kernel does with an exact INT32 sum: token and channel scales, bias, SiLU,
// skip connection, one rounding to the output type. Every kernel takes these steps in this order, so all give the same bits. But
// for SiLU each is one IEEE FP32 rounding in the order of the low-bit GEMMs' epilogue; SiLU is this file's own.
#pragma once

#include "operator_common.cuh"

namespace kea {

struct Int8Args {
    const int8_t *q;             // [m][ldq]
    long long ldq;
    const float *qs;             // [m]
    const int8_t *w;             // [n][ldw]
    long long ldw;
    const float *alpha;          // [n]
    const float *bias;           // [n] or null
    void *y;                     // [m][ldy] of y_type
    long long ldy;
    const void *res;             // [m][ld_res] of y_type, or null: y = res + res_scale * value
    long long ld_res;
    int *acc;                    // INT32 [m][ld_acc] or null
    long long ld_acc;
    float res_scale;
    int M, N, K;
    int y_type, silu;
    uint32_t *err;
};

// The bias where there is none: r * alpha + -0 is r * alpha, its sign included.
constexpr float kI8NoBias = -0.0f;

// Two outputs before the skip connection. SiLU: y times the reciprocal of 1 + 2^(-y log2 e), the hardware's approximate exponential
// and reciprocal (2 and 1 units in the last place, subnormals as zero; a denominator above 2^126 gives 0), so that two values
// share the packed operations. (The low-bit epilogue divides, and keeps subnormals.)
template <bool SILU>
KEA_DEVI uint64_t int8_values(int a0, int a1, uint64_t s, uint64_t alpha, uint64_t bias) {
    uint64_t y = fma2(mul2(pair_of(__int2float_rn(a0), __int2float_rn(a1)), s), alpha, bias);
    if constexpr (SILU) {
        float t0, t1;
        unpair(mul2(y, pair_of(-1.4426950408889634f, -1.4426950408889634f)), t0, t1);
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t0));
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t1));
        unpair(add2(pair_of(t0, t1), pair_of(1.0f, 1.0f)), t0, t1);
        asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(t0));
        asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(t1));
        y = mul2(y, pair_of(t0, t1));
    }
    return y;
}

template <typename T>
KEA_DEVI void int8_store(const Int8Args &a, int m, int n, float v) {
    if (a.res)
        v = __fadd_rn(to_float(static_cast<const T *>(a.res)[(long long)m * a.ld_res + n]), __fmul_rn(a.res_scale, v));
    static_cast<T *>(a.y)[(long long)m * a.ldy + n] = from_float<T>(v);
}

}  // namespace kea
