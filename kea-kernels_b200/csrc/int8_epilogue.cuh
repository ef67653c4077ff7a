// int8_epilogue.cuh - what every 8-bit GEMM kernel does with an exact INT32 sum: token and channel scales, bias, SiLU,
// skip connection, one rounding to the output type. Each operation is one IEEE FP32 rounding in the order of the
// low-bit GEMMs' epilogue, so all kernels give the same bits.
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

// value of one output before the skip connection; has_bias as the caller's constant
KEA_DEVI float int8_value(int acc, float s, float alpha, bool has_bias, float bias, bool silu) {
    const float r = __fmul_rn(__int2float_rn(acc), s);
    const float v = has_bias ? __fmaf_rn(r, alpha, bias) : __fmul_rn(r, alpha);
    return silu ? silu_approx(v) : v;
}

template <typename T>
KEA_DEVI void int8_store(const Int8Args &a, int m, int n, float v) {
    if (a.res)
        v = __fadd_rn(to_float(static_cast<const T *>(a.res)[(long long)m * a.ld_res + n]), __fmul_rn(a.res_scale, v));
    static_cast<T *>(a.y)[(long long)m * a.ldy + n] = from_float<T>(v);
}

}  // namespace kea
