// residual_norm_kernel.cuh - the step between two blocks of a residual network in one pass over its rows:
//   u = post(y)                     LayerNorm, root-mean-square norm or nothing, over the block's output row
//   r = x + scale * act(gate) * u   the residual stream's next value (stored in x's type)
//   h = pre(r)                      the next block's norm, taken of r before its rounding; stored as FP32 / FP16 / BF16, or
//                                   as INT8 codes with one scale per row (the quantizer's formula)
// Statistics and every intermediate value are FP32; a value is rounded to a shorter type only where it is stored.
//
// `tpr` threads (32 .. 512) hold one row in registers, VPT values each, so every input is read and every output written
// once; a LayerNorm takes two group sums (mean, then centred squares), a root-mean-square norm one, the codes one maximum.
// VEC: whole vectors per chunk; otherwise thread i holds values i, i + tpr, ...
//
// Two kernels: residual_norm_kernel for rows at any stride, a group of threads to a row; residual_norm_flat_kernel (below) for
// many contiguous rows whose width no vector fits.
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
    int ldq;                             // rows times it pass 32 bits: multiplied in 64
    float *qs;
    int M, D;
};

constexpr int kRnMaxThreads = 512;
constexpr int kRnSlots = 5;   // group reductions of one launch

// W consecutive values (1, or whole vectors of 4 or 8) to and from FP32 registers.
template <int W, typename T>
KEA_DEVI void get(const T *p, float *v) {
    if constexpr (W == 1) {
        v[0] = to_float(*p);
    } else if constexpr (sizeof(T) == 4 && W == 8) {   // a 32-byte load; ordered after griddepcontrol.wait (volatile)
        asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                     : "l"(p));
    } else if constexpr (sizeof(T) == 4) {
        const float4 f = *reinterpret_cast<const float4 *>(p);
        v[0] = f.x;
        v[1] = f.y;
        v[2] = f.z;
        v[3] = f.w;
    } else {
        uint32_t u[W / 2];
        if constexpr (W == 8) *reinterpret_cast<uint4 *>(u) = *reinterpret_cast<const uint4 *>(p);
        else *reinterpret_cast<uint2 *>(u) = *reinterpret_cast<const uint2 *>(p);
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
            const float2 f = unpack2<T>(u[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
template <int W, typename T>
KEA_DEVI void put(T *p, const float *v) {
    if constexpr (W == 1) {
        *p = from_float<T>(v[0]);
    } else if constexpr (sizeof(T) == 4 && W == 8) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                     "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                     : "memory");
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        uint32_t u[W / 2];
#pragma unroll
        for (int i = 0; i < W / 2; ++i) u[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
        if constexpr (W == 8) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(u);
        else *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(u);
    }
}

// W values as they came from memory: 16-bit types stay packed until they are used (half the registers).
template <typename T, int W>
struct RawValues {
    static constexpr bool kPacked = sizeof(T) == 2 && W == 8;
    uint4 words;
    float v[kPacked ? 1 : W];
    KEA_DEVI void load(const T *p) {
        if constexpr (kPacked) words = *reinterpret_cast<const uint4 *>(p);
        else get<W>(p, v);
    }
    KEA_DEVI void values(float *f) const {
        if constexpr (kPacked) {
            const uint32_t u[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 t = unpack2<T>(u[i]);
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) f[i] = v[i];
        }
    }
};

// The larger of two values; not a number where one of them is none.
KEA_DEVI float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The largest size of three values, the same way.
KEA_DEVI float max_size_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Sum or maximum (max_nan) over a row group's threads in a fixed order; `slot`: kRnMaxThreads / 32 floats used by this reduction
// alone. Every thread of the CTA calls it.
template <bool MAX>
KEA_DEVI float row_reduce(float v, int tpr, float *slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xFFFFFFFFu, v, o);
        v = MAX ? max_nan(v, u) : v + u;
    }
    if (tpr == 32) return v;
    const int warp = threadIdx.x >> 5, per = tpr >> 5;
    if ((threadIdx.x & 31) == 0) slot[warp] = v;
    __syncthreads();
    const int first = warp - warp % per;
    float r = slot[first];
    for (int w = 1; w < per; ++w) r = MAX ? max_nan(r, slot[first + w]) : r + slot[first + w];
    return r;
}

// One thread's share of a row: VPT values in chunks of W, chunk c at (c * tpr + gt) * W. Nothing here branches on a chunk
// being inside the row: chunks past its end read the last one and count as zeros (a branch per chunk would make every
// chunk wait for its own loads: rows of 1001 values took six times as long).
template <int VPT, int W>
struct RowPart {
    static constexpr int C = VPT / W;
    int gt, tpr, D;
    KEA_DEVI int at(int c) const { return (c * tpr + gt) * W; }
    KEA_DEVI bool in(int c) const { return at(c) < D; }
    KEA_DEVI int safe(int c) const { return min(at(c), D - W); }

    template <typename T>
    KEA_DEVI void load(const T *row, float (&v)[VPT]) const {
#pragma unroll
        for (int c = 0; c < C; ++c) get<W>(row + safe(c), v + W * c);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < W; ++i) v[W * c + i] = in(c) ? v[W * c + i] : 0.f;
    }
    template <typename T>
    KEA_DEVI void store(T *row, const float (&v)[VPT], bool live) const {
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (live && in(c)) put<W>(row + at(c), v + W * c);
    }
    KEA_DEVI void norm(float (&v)[VPT], int kind, const float *w, const float *b, float eps, float *slots) const {
        if (kind == KEA_NORM_LAYER) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < VPT; ++i) s += v[i];
            const float mean = __fdiv_rn(row_reduce<false>(s, tpr, slots), (float)D);
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < W; ++i) v[W * c + i] = in(c) ? v[W * c + i] - mean : 0.f;
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) ss = fmaf(v[i], v[i], ss);
        const float inv = rsqrtf(__fdiv_rn(row_reduce<false>(ss, tpr, slots + kRnMaxThreads / 32), (float)D) + eps);
        if (b) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float wv[W], bv[W];
                get<W>(w + safe(c), wv);
                get<W>(b + safe(c), bv);
#pragma unroll
                for (int i = 0; i < W; ++i) v[W * c + i] = fmaf(v[W * c + i] * inv, wv[i], bv[i]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float wv[W];
                get<W>(w + safe(c), wv);
#pragma unroll
                for (int i = 0; i < W; ++i) v[W * c + i] = v[W * c + i] * inv * wv[i];
            }
        }
    }
    // h as INT8 codes with one scale, as the quantizer's single part; codes hold no NaN, so a row with one has scale NaN (and
    // codes 0), and the product after it is not a number either
    KEA_DEVI void codes(const float (&v)[VPT], int8_t *q, int ldq, float *qs, bool live, float *slot) const {
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; i += 2) amax = max_size_nan(amax, in(i / W) ? v[i] : 0.f, in((i + 1) / W) ? v[i + 1] : 0.f);
        amax = row_reduce<true>(amax, tpr, slot);
        const float s = max_nan(__fdiv_rn(amax, 127.0f), 1.0e-30f), inv = __frcp_rn(s);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if constexpr (W == 1) {
                if (live && in(c)) q[at(c)] = (int8_t)(int)round_quotient(v[c], s, inv);
            } else {
                float t[4];
                uint32_t word[W / 4];
#pragma unroll
                for (int h = 0; h < W / 4; ++h) word[h] = quantize4(v + W * c + 4 * h, s, inv, t);
                if (live && in(c)) {
                    if constexpr (W == 8) *reinterpret_cast<uint2 *>(q + at(c)) = make_uint2(word[0], word[1]);
                    else *reinterpret_cast<uint32_t *>(q + at(c)) = word[0];
                }
            }
        }
        if (live) {
            for (int e = D + gt; e < ldq; e += tpr) q[e] = 0;   // padding columns
            if (gt == 0) *qs = s;
        }
    }
};

// THREADS: the largest CTA. With 128 (rows of up to 4096 values) four CTAs share an SM (five spill registers: 70 instead of
// 64 us for 32000 rows of 1024 BF16 values).
template <typename TX, typename TY, int VPT, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 128 ? 4 : 1) residual_norm_kernel(const ResidualNormArgs a, int tpr) {
    __shared__ float slots[kRnSlots * (kRnMaxThreads / 32)];
    constexpr int S = kRnMaxThreads / 32, W = VEC ? 8 : 1, C = VPT / W;
    const int rows = blockDim.x / tpr;
    const int row = blockIdx.x * rows + threadIdx.x / tpr;
    const bool live = row < a.M;
    const int m = live ? row : a.M - 1;   // a group past the last row does that one again and stores nothing
    const RowPart<VPT, W> part{(int)(threadIdx.x % tpr), tpr, a.D};
    grid_dependency_wait();
    grid_launch_dependents();
    // everything is asked for at once: the stream and the gate wait, as they came, for the block's norm. (Not an FP32 gate
    // beside 32 FP32 values of each: the registers spill, 32000 rows of 1024 take 139 us instead of 98.)
    constexpr bool kGateAhead = VPT < 32 || sizeof(TY) == 2;
    RawValues<TX, W> xr[C];
    RawValues<TY, W> gr[C];
    float u[VPT], x[VPT];
    const TX *const xp = static_cast<const TX *>(a.x) + m * a.ldx;
    const TY *const gp = static_cast<const TY *>(a.gate) + (long long)(m / a.frames) * a.gate_clip + (long long)(m % a.frames) * a.gate_row;
    {
        RawValues<TY, W> yr[C];
        const TY *const yp = static_cast<const TY *>(a.y) + m * a.ldy;
#pragma unroll
        for (int c = 0; c < C; ++c) yr[c].load(yp + part.safe(c));
#pragma unroll
        for (int c = 0; c < C; ++c) xr[c].load(xp + part.safe(c));
        if (kGateAhead && a.gate)
#pragma unroll
            for (int c = 0; c < C; ++c) gr[c].load(gp + part.safe(c));
#pragma unroll
        for (int c = 0; c < C; ++c) {
            yr[c].values(u + W * c);
#pragma unroll
            for (int i = 0; i < W; ++i) u[W * c + i] = part.in(c) ? u[W * c + i] : 0.f;
        }
    }
    if (a.post) part.norm(u, a.post, a.post_w, a.post_b, a.post_eps, slots);
    if (a.gate) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float g[W];
            if constexpr (kGateAhead) gr[c].values(g);
            else get<W>(gp + part.safe(c), g);
#pragma unroll
            for (int i = 0; i < W; ++i) u[W * c + i] *= a.gate_act == KEA_GATE_SIGMOID ? __fdividef(1.0f, 1.0f + __expf(-g[i])) : g[i];
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        xr[c].values(x + W * c);
#pragma unroll
        for (int i = 0; i < W; ++i) x[W * c + i] = part.in(c) ? fmaf(a.scale, u[W * c + i], x[W * c + i]) : 0.f;
    }
    part.store(static_cast<TX *>(a.r) + m * a.ldr, x, live);
    if (a.pre) part.norm(x, a.pre, a.pre_w, a.pre_b, a.pre_eps, slots + 2 * S);
    if (a.h) {
        if (a.h_type == KEA_TYPE_F32) part.store(static_cast<float *>(a.h) + m * a.ldh, x, live);
        else if (a.h_type == KEA_TYPE_F16) part.store(static_cast<__half *>(a.h) + m * a.ldh, x, live);
        else part.store(static_cast<__nv_bfloat16 *>(a.h) + m * a.ldh, x, live);
    }
    if (a.q) part.codes(x, a.q + (long long)m * a.ldq, a.ldq, a.qs + m, live, slots + 4 * S);
}

// ---- many contiguous rows of any width -----------------------------------------------------------------------------------
// Rows whose width is no multiple of eight start at any address. Read value by value they cost a memory instruction per 32
// values (12024 rows of 1001 values, FP32 stream and BF16 block: 66 us in registers, 79 and 136 us through shared memory,
// against 22 us of traffic; 3000 instructions a row bound it). But in one contiguous buffer the groups of eight values
// that start at a multiple of eight are aligned in x, y, r, h and a gate of x's shape alike, wherever the rows begin: a
// thread takes such groups, the two at a row's ends in part. What does not line up is the parameters: value i of a row
// sits in its group at (i + o) % 8 with the row's own o. They are held in shared memory four times, shifted by 0 .. 3
// values, so that every group finds its parameters in two aligned vectors of one of the copies. One CTA of 16 warps per
// SM shares the copies and takes rows in turn.
constexpr int kFlatThreads = 512, kFlatVpt = 32, kFlatGroups = kFlatVpt / 8;

struct FlatArgs {
    ResidualNormArgs a;
    int padded;               // floats of one shifted copy: whole rows of groups and eight more
    long long gate_end;       // values of a gate of other strides, from its 16-byte aligned base; 0: not aligned
    int params;               // bit k: parameter k (post weight, post bias, pre weight, pre bias, shared gate) is held
};

// Eight values of a row: groups of the flat buffer, `lo` .. `hi` of each inside the row.
template <int TPR>
struct FlatRow {
    long long first;          // flat index of this thread's first group
    long long total;
    int i0, D;                // index in the row of that group's first value (negative before the row)
    KEA_DEVI int index(int c) const { return i0 + 8 * TPR * c; }
    KEA_DEVI bool whole(int c) const { return index(c) >= 0 && index(c) + 8 <= D; }
    KEA_DEVI bool some(int c) const { return index(c) + 8 > 0 && index(c) < D; }
    KEA_DEVI bool has(int c, int e) const { return (unsigned)(index(c) + e) < (unsigned)D; }

    template <typename T>
    KEA_DEVI void load(const T *p, float (&v)[kFlatVpt]) const {
#pragma unroll
        for (int c = 0; c < kFlatGroups; ++c) {
            const long long f = first + 8LL * TPR * c;
            if (f + 8 <= total) {
                get<8>(p + f, v + 8 * c);
            } else {   // the buffer's end
#pragma unroll
                for (int e = 0; e < 8; ++e) v[8 * c + e] = f + e < total ? to_float(p[f + e]) : 0.f;
            }
        }
    }
    // Values of a row at p + g0 that the groups do not line up with: its own 16-byte pieces, moved by the row's shift
    // (12024 rows of 1001 values with a BF16 gate per clip: 49.7 us value by value, 48.2 so; 4008 of 4089: 66.6 and 58.4.
    // Asking for them ahead with an L1 prefetch: 50.4, the instructions cost more than the wait). A piece is read where it
    // holds a value of the row; the caller has seen that the row's last piece ends in the buffer.
    template <typename T>
    KEA_DEVI void load_shifted(const T *p, long long g0, float (&v)[kFlatVpt]) const {
        constexpr int CH = 16 / (int)sizeof(T), N = 8 / CH + 1;
        const int shift = (int)((g0 + i0) & (CH - 1));
#pragma unroll
        for (int c = 0; c < kFlatGroups; ++c) {
            const long long at = g0 + index(c) - shift;
            uint32_t w[4 * N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const long long piece = at + CH * k;
                uint4 u = make_uint4(0u, 0u, 0u, 0u);
                if (piece + CH > g0 && piece < g0 + D) u = *reinterpret_cast<const uint4 *>(p + piece);
                w[4 * k] = u.x, w[4 * k + 1] = u.y, w[4 * k + 2] = u.z, w[4 * k + 3] = u.w;
            }
            const int words = shift * (int)sizeof(T) / 4;
#pragma unroll
            for (int by = 2; by > 0; by >>= 1)
#pragma unroll
                for (int i = 0; i + by < 4 * N; ++i) w[i] = words & by ? w[i + by] : w[i];
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 t = unpack2<T>(shift & 1 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i]);
                    v[8 * c + 2 * i] = t.x;
                    v[8 * c + 2 * i + 1] = t.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * c + i] = __uint_as_float(w[i]);
            }
        }
    }
    KEA_DEVI void clear(float (&v)[kFlatVpt]) const {   // zeros where a group reaches out of the row
#pragma unroll
        for (int c = 0; c < kFlatGroups; ++c)
            if (!whole(c)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[8 * c + e] = has(c, e) ? v[8 * c + e] : 0.f;
            }
    }
    template <typename T>
    KEA_DEVI void store(T *p, const float (&v)[kFlatVpt]) const {
#pragma unroll
        for (int c = 0; c < kFlatGroups; ++c) {
            T *const at = p + first + 8LL * TPR * c;
            if (whole(c)) {
                put<8>(at, v + 8 * c);
            } else if (some(c)) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (has(c, e)) at[e] = from_float<T>(v[8 * c + e]);
            }
        }
    }
    // `w`: this row's shifted copy at this thread's first group
    KEA_DEVI static void scaled(float (&v)[kFlatVpt], float by, const float *w, const float *b) {
#pragma unroll
        for (int c = 0; c < kFlatGroups; ++c) {
            float wv[8], bv[8];
            get<4>(w + 8 * TPR * c, wv);
            get<4>(w + 8 * TPR * c + 4, wv + 4);
            if (b) {
                get<4>(b + 8 * TPR * c, bv);
                get<4>(b + 8 * TPR * c + 4, bv + 4);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float t = v[8 * c + e] * by;
                v[8 * c + e] = b ? fmaf(t, wv[e], bv[e]) : t * wv[e];
            }
        }
    }
    KEA_DEVI void norm(float (&v)[kFlatVpt], int kind, float eps, const float *w, const float *b, float *slots) const {
        if (kind == KEA_NORM_LAYER) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < kFlatVpt; ++i) s += v[i];
            const float mean = __fdiv_rn(row_reduce<false>(s, TPR, slots), (float)D);
#pragma unroll
            for (int i = 0; i < kFlatVpt; ++i) v[i] -= mean;
            clear(v);
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < kFlatVpt; ++i) ss = fmaf(v[i], v[i], ss);
        const float inv = rsqrtf(__fdiv_rn(row_reduce<false>(ss, TPR, slots + kRnMaxThreads / 32), (float)D) + eps);
        scaled(v, inv, w, b);
    }
};

template <typename TX, typename TY, int TPR>
__global__ void __launch_bounds__(kFlatThreads, 1) residual_norm_flat_kernel(const __grid_constant__ FlatArgs p) {
    extern __shared__ __align__(16) float copies[];   // [held parameters][4 shifts][padded]
    __shared__ float slots[kRnSlots * (kRnMaxThreads / 32)];
    constexpr int SL = kRnMaxThreads / 32, GROUPS = kFlatThreads / TPR;
    const ResidualNormArgs &a = p.a;
    const int D = a.D, group = (int)threadIdx.x / TPR, gt = (int)threadIdx.x % TPR;
    const long long total = (long long)a.M * D;
    const float *const source[4] = {a.post_w, a.post_b, a.pre_w, a.pre_b};
    const float *held[5];
    int n = 0;
#pragma unroll
    for (int k = 0; k < 5; ++k) {
        held[k] = nullptr;
        if (p.params >> k & 1) held[k] = copies + (size_t)4 * p.padded * n++;
    }
    // copy s holds value i at i + 8 + s: the group with row index i0 = 8 t - o finds its values at i0 + 8 + (o % 4)
    const auto fill = [&](float *to, auto value) {
        for (int i = threadIdx.x; i < 4 * p.padded; i += kFlatThreads) {
            const int s = i / p.padded, at = i - s * p.padded - 8 - s;
            to[i] = at >= 0 && at < D ? value(at) : 0.f;
        }
    };
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (held[k]) fill(const_cast<float *>(held[k]), [&](int i) { return __ldg(source[k] + i); });
    grid_dependency_wait();
    grid_launch_dependents();
    if (held[4])
        fill(const_cast<float *>(held[4]), [&](int i) {
            const float g = to_float(static_cast<const TY *>(a.gate)[i]);
            return a.gate_act == KEA_GATE_SIGMOID ? __fdividef(1.0f, 1.0f + __expf(-g)) : g;
        });
    __syncthreads();

    const int turns = (a.M + (int)gridDim.x * GROUPS - 1) / ((int)gridDim.x * GROUPS);
    for (int turn = 0; turn < turns; ++turn) {   // every thread takes every turn (row_reduce has barriers)
        const long long wanted = ((long long)turn * gridDim.x + blockIdx.x) * GROUPS + group;
        const bool live = wanted < a.M;
        if (TPR == 32 && !live) break;
        const int m = live ? (int)wanted : 0;
        const long long start = (long long)m * D;
        const int o = (int)(start & 7);
        const FlatRow<TPR> row{start - o + 8LL * gt, total, 8 * gt - o, D};
        const int at = row.i0 + 8 + (o & 3);   // of this thread's first group in the row's copy, a multiple of four
        const auto mine = [&](int k) { return held[k] ? held[k] + (o & 3) * p.padded + at : nullptr; };
        float u[kFlatVpt], x[kFlatVpt];
        row.load(static_cast<const TY *>(a.y), u);
        row.load(static_cast<const TX *>(a.x), x);
        row.clear(u);
        if (a.post) row.norm(u, a.post, a.post_eps, mine(0), mine(1), slots);
        if (held[4]) {
            row.scaled(u, 1.0f, mine(4), nullptr);
        } else if (a.gate) {
            float g[kFlatVpt];
            if (a.gate_row == D && a.gate_clip == (long long)a.frames * D) {
                row.load(static_cast<const TY *>(a.gate), g);
            } else {   // one row per clip
                constexpr int CH = 16 / (int)sizeof(TY);
                const long long g0 = (long long)(m / a.frames) * a.gate_clip + (long long)(m % a.frames) * a.gate_row;
                if (((g0 + D + CH - 1) & ~(long long)(CH - 1)) <= p.gate_end) {
                    row.load_shifted(static_cast<const TY *>(a.gate), g0, g);
                } else {   // the buffer's end, or no alignment: value by value
                    const TY *const gr = static_cast<const TY *>(a.gate) + g0;
#pragma unroll
                    for (int c = 0; c < kFlatGroups; ++c)
#pragma unroll
                        for (int e = 0; e < 8; ++e) g[8 * c + e] = row.has(c, e) ? to_float(gr[row.index(c) + e]) : 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < kFlatVpt; ++i) u[i] *= a.gate_act == KEA_GATE_SIGMOID ? __fdividef(1.0f, 1.0f + __expf(-g[i])) : g[i];
        }
#pragma unroll
        for (int i = 0; i < kFlatVpt; ++i) x[i] = fmaf(a.scale, u[i], x[i]);
        row.clear(x);
        if (live) row.store(static_cast<TX *>(a.r), x);
        if (a.pre) row.norm(x, a.pre, a.pre_eps, mine(2), mine(3), slots + 2 * SL);
        if (a.h && live) {
            if (a.h_type == KEA_TYPE_F32) row.store(static_cast<float *>(a.h), x);
            else if (a.h_type == KEA_TYPE_F16) row.store(static_cast<__half *>(a.h), x);
            else row.store(static_cast<__nv_bfloat16 *>(a.h), x);
        }
        if (a.q) {   // codes with one scale, as the quantizer's single part
            row.clear(x);
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < kFlatVpt; i += 2) amax = max_size_nan(amax, x[i], x[i + 1]);
            amax = row_reduce<true>(amax, TPR, slots + 4 * SL);
            const float s = max_nan(__fdiv_rn(amax, 127.0f), 1.0e-30f), inv = __frcp_rn(s);
            int8_t *const q = a.q + (long long)m * a.ldq;
#pragma unroll
            for (int c = 0; c < kFlatGroups; ++c) {
                float t[4];
                const uint32_t word[2] = {quantize4(x + 8 * c, s, inv, t), quantize4(x + 8 * c + 4, s, inv, t)};
                if (live && row.some(c)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (row.has(c, e)) q[row.index(c) + e] = (int8_t)(word[e / 4] >> (8 * (e % 4)));
                }
            }
            if (live) {
                for (int e = D + gt; e < a.ldq; e += TPR) q[e] = 0;   // padding columns
                if (gt == 0) a.qs[m] = s;
            }
        }
        if (TPR > 32) __syncthreads();   // the reductions' slots serve the next rows
    }
}

}  // namespace kea
