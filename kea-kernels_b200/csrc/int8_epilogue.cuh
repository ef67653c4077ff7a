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

// y / (1 + 2^(-y log2 e)) with the hardware's approximate exponential and division (2 units in the last place each; a
// denominator above 2^126 gives 0).
KEA_DEVI float int8_silu(float y) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(y, -1.4426950408889634f)));
    return __fdividef(y, __fadd_rn(1.0f, e));
}

// RN(a) without the conversion instruction, whose pipe is a quarter as wide as the SiLU's exponential and reciprocal
// leave free: with a = 65536 h + l, the float of bits 0x4B000000 | (h + 2^15) is 2^23 + 2^15 + h and that of 0x4B000000 | l
// is 2^23 + l; the fma is exact (a multiple of 65536 below 2^40), the addition rounds once.
KEA_DEVI float int_to_float(int a) {
    const float h = __uint_as_float(__byte_perm((uint32_t)a ^ 0x80000000u, 0x4B000000u, 0x7632));
    const float l = __uint_as_float(__byte_perm((uint32_t)a, 0x4B000000u, 0x7610));
    return __fadd_rn(__fmaf_rn(h, 65536.0f, -551911686144.0f), l);   // 65536 (2^23 + 2^15 + 128)
}

// One output before the skip connection.
template <bool SILU>
KEA_DEVI float int8_value(int acc, float s, float alpha, bool has_bias, float bias) {
    const float r = __fmul_rn(SILU ? int_to_float(acc) : __int2float_rn(acc), s);
    const float v = has_bias ? __fmaf_rn(r, alpha, bias) : __fmul_rn(r, alpha);
    return SILU ? int8_silu(v) : v;
}
KEA_DEVI float int8_value(int acc, float s, float alpha, bool has_bias, float bias, bool silu) {
    return silu ? int8_value<true>(acc, s, alpha, has_bias, bias) : int8_value<false>(acc, s, alpha, has_bias, bias);
}

template <typename T>
KEA_DEVI void int8_store(const Int8Args &a, int m, int n, float v) {
    if (a.res)
        v = __fadd_rn(to_float(static_cast<const T *>(a.res)[(long long)m * a.ld_res + n]), __fmul_rn(a.res_scale, v));
    static_cast<T *>(a.y)[(long long)m * a.ldy + n] = from_float<T>(v);
}

}  // namespace kea
