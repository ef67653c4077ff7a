// residual_norm_kernel.cuh - the step between two blocks of a residual network in one pass over its rows:
//   u = post(y)                     LayerNorm, root-mean-square norm or nothing, over the block's output row
//   r = x + scale * act(gate) * u   the residual stream's next value (stored in x's type)
//   h = pre(r)                      the next block's norm, taken of r before its rounding; stored as FP32 / FP16 / BF16, or
//                                   as INT8 codes with one scale per row (the quantizer's formula)
// Statistics and every intermediate value are FP32; a value is rounded to a shorter type only where it is stored.
//
// `tpr` threads (32 .. 512) hold one row in registers, VPT values each, so every input is read and every output written
// once; a LayerNorm takes two group sums (mean, then centred squares), a root-mean-square norm one, the codes one maximum.
// VEC: eight consecutive values per chunk (32-byte FP32 or 16-byte loads); otherwise thread i holds values i, i + tpr, ...
#pragma once

#include "operator_common.cuh"
#include "quant_common.cuh"

namespace kea {

struct ResidualNormArgs {
    const void *x, *y, *gate;
    long long ldx, ldy;
    long long gate_clip, gate_row;       // gate strides: per clip, per row of a clip (0: shared)
    int frames;                          // rows per clip
    int gate_act, post, pre;
    float scale, post_eps, pre_eps;
    const float *post_w, *post_b, *pre_w, *pre_b;
    void *r, *h;
    long long ldr, ldh;
    int h_type;
    int8_t *q;
    int ldq;
    float *qs;
    int M, D;
};

constexpr int kRnThreads = 256;
constexpr int kRnMaxThreads = 512;
constexpr int kRnSlots = 5;   // group reductions of one launch

KEA_DEVI void load8(const float *p, float *v) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(p)
                 : "memory");
}
template <typename T>
KEA_DEVI void load8(const T *p, float *v) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(u[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
KEA_DEVI void store8(float *p, const float *v) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                 "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}
template <typename T>
KEA_DEVI void store8(T *p, const float *v) {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

// Sum or maximum over a row group's threads in a fixed order; `slot`: kRnMaxThreads / 32 floats used by this reduction
// alone. Every thread of the CTA calls it.
template <bool MAX>
KEA_DEVI float row_reduce(float v, int tpr, float *slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xFFFFFFFFu, v, o);
        v = MAX ? fmaxf(v, u) : v + u;
    }
    if (tpr == 32) return v;
    const int warp = threadIdx.x >> 5, per = tpr >> 5;
    if ((threadIdx.x & 31) == 0) slot[warp] = v;
    __syncthreads();
    const int first = warp - warp % per;
    float r = slot[first];
    for (int w = 1; w < per; ++w) r = MAX ? fmaxf(r, slot[first + w]) : r + slot[first + w];
    return r;
}

template <typename TX, typename TY, int VPT, bool VEC>
struct RowStep {
    static constexpr int C = VEC ? VPT / 8 : VPT, W = VEC ? 8 : 1;
    int gt, tpr, D;
    KEA_DEVI int at(int c) const { return (c * tpr + gt) * W; }   // first value of chunk c
    KEA_DEVI bool in(int c) const { return at(c) < D; }

    template <typename T>
    KEA_DEVI void load(const T *row, float (&v)[VPT]) const {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (in(c)) {
                if constexpr (VEC) load8(row + at(c), v + 8 * c);
                else v[c] = to_float(row[at(c)]);
            } else {
#pragma unroll
                for (int i = 0; i < W; ++i) v[W * c + i] = 0.f;
            }
        }
    }
    template <typename T>
    KEA_DEVI void store(T *row, const float (&v)[VPT]) const {
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (in(c)) {
                if constexpr (VEC) store8(row + at(c), v + 8 * c);
                else row[at(c)] = from_float<T>(v[c]);
            }
    }
    KEA_DEVI void norm(float (&v)[VPT], int kind, const float *w, const float *b, float eps, float *slots) const {
        float mean = 0.f;
        if (kind == KEA_NORM_LAYER) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < VPT; ++i) s += v[i];
            mean = __fdiv_rn(row_reduce<false>(s, tpr, slots), (float)D);
        }
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (in(c)) {
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    v[W * c + i] -= mean;
                    ss = fmaf(v[W * c + i], v[W * c + i], ss);
                }
            }
        const float inv = rsqrtf(__fdiv_rn(row_reduce<false>(ss, tpr, slots + kRnMaxThreads / 32), (float)D) + eps);
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (in(c)) {
                float wv[W], bv[W];
                if constexpr (VEC) {
                    load8(w + at(c), wv);
                    if (b) load8(b + at(c), bv);
                } else {
                    wv[0] = w[at(c)];
                    if (b) bv[0] = b[at(c)];
                }
#pragma unroll
                for (int i = 0; i < W; ++i) v[W * c + i] = fmaf(v[W * c + i] * inv, wv[i], b ? bv[i] : 0.f);
            }
    }
};

template <typename TX, typename TY, int VPT, bool VEC>
__global__ void __launch_bounds__(kRnMaxThreads) residual_norm_kernel(const ResidualNormArgs a, int tpr) {
    __shared__ float slots[kRnSlots * (kRnMaxThreads / 32)];
    const int rows = blockDim.x / tpr;
    const int m = blockIdx.x * rows + threadIdx.x / tpr;
    const bool live = m < a.M;
    const RowStep<TX, TY, VPT, VEC> row{(int)(threadIdx.x % tpr), tpr, live ? a.D : 0};
    using Row = RowStep<TX, TY, VPT, VEC>;
    const long long mr = live ? m : 0;
    grid_dependency_wait();
    grid_launch_dependents();
    float u[VPT], x[VPT];
    row.load(static_cast<const TY *>(a.y) + mr * a.ldy, u);
    row.load(static_cast<const TX *>(a.x) + mr * a.ldx, x);
    constexpr int S = kRnMaxThreads / 32;
    RowStep<TX, TY, VPT, VEC> full = row;
    full.D = a.D;   // statistics divide by the row's width; a dead group's values are zeros
    if (a.post) full.norm(u, a.post, a.post_w, a.post_b, a.post_eps, slots);
    if (a.gate) {
        const TY *gate = static_cast<const TY *>(a.gate) + (mr / a.frames) * a.gate_clip + (mr % a.frames) * a.gate_row;
#pragma unroll
        for (int c = 0; c < Row::C; ++c)
            if (row.in(c)) {
                float g[Row::W];
                if constexpr (VEC) load8(gate + row.at(c), g);
                else g[0] = to_float(gate[row.at(c)]);
#pragma unroll
                for (int i = 0; i < Row::W; ++i) {
                    if (a.gate_act == KEA_GATE_SIGMOID) g[i] = __fdividef(1.0f, 1.0f + __expf(-g[i]));
                    u[Row::W * c + i] *= g[i];
                }
            }
    }
#pragma unroll
    for (int c = 0; c < Row::C; ++c)
        if (row.in(c)) {
#pragma unroll
            for (int i = 0; i < Row::W; ++i) x[Row::W * c + i] = fmaf(a.scale, u[Row::W * c + i], x[Row::W * c + i]);
        }
    row.store(static_cast<TX *>(a.r) + mr * a.ldr, x);
    if (a.pre) full.norm(x, a.pre, a.pre_w, a.pre_b, a.pre_eps, slots + 2 * S);
    if (a.h) {
        if (a.h_type == KEA_TYPE_F32) row.store(static_cast<float *>(a.h) + mr * a.ldh, x);
        else if (a.h_type == KEA_TYPE_F16) row.store(static_cast<__half *>(a.h) + mr * a.ldh, x);
        else row.store(static_cast<__nv_bfloat16 *>(a.h) + mr * a.ldh, x);
    }
    if (a.q) {
        float amax = 0.f;
#pragma unroll
        for (int c = 0; c < Row::C; ++c)
            if (row.in(c)) {
#pragma unroll
                for (int i = 0; i < Row::W; ++i) amax = fmaxf(amax, fabsf(x[Row::W * c + i]));
            }
        amax = row_reduce<true>(amax, tpr, slots + 4 * S);
        const float s = fmaxf(__fdiv_rn(amax, 127.0f), 1.0e-30f), inv = __frcp_rn(s);
        int8_t *q = a.q + mr * a.ldq;
#pragma unroll
        for (int c = 0; c < Row::C; ++c)
            if (row.in(c)) {
                if constexpr (VEC) {
                    float t[4];
                    uint2 w;
                    w.x = quantize4(x + 8 * c, s, inv, t);
                    w.y = quantize4(x + 8 * c + 4, s, inv, t);
                    *reinterpret_cast<uint2 *>(q + row.at(c)) = w;
                } else {
                    q[row.at(c)] = (int8_t)(int)round_quotient(x[c], s, inv);
                }
            }
        if (live) {
            for (int i = a.D + row.gt; i < a.ldq; i += tpr) q[i] = 0;   // padding columns
            if (row.gt == 0) a.qs[m] = s;
        }
    }
}

}  // namespace kea
