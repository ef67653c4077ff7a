// int8_reg_kernel.cuh - the 8-bit GEMM for few tokens: warp-level tensor-core MMAs (mma.sync m16n8k32, INT8 x INT8 ->
// INT32) on operands loaded straight from global memory into registers.
//
// With a handful of tokens the weights are nearly all that is read (N x K bytes for 2 M N K operations), and a launch
// lasts a few microseconds: what counts is that every byte is requested at once and that nothing is set up first. So no
// shared-memory staging, no barriers before the sums: a warp asks for its operands a few steps ahead, in 16-byte loads.
//
// Operands. The weights are the MMA's A operand (16 channels x 32 k), the tokens B (32 k x 8 rows). An integer sum does
// not depend on the order of its terms as long as both operands use the same one, so k is walked in steps of 64 (two
// MMAs): lane (g, t) (g = lane / 4, t = lane % 4) holds bytes 16 t .. 16 t + 15 of rows g and g + 8 of its 16 channels and of
// token row g; bytes 0-3 / 4-7 of a 16-byte group are the first MMA's two k registers, 8-11 / 12-15 the second's.
//
// Work split. A CTA owns 16 channels (8 where that leaves SMs without one: the MMA's upper rows stay empty) x 8 RG tokens; its
// 8 warps are slices of K, whose INT32 sums meet in shared memory, are added in slice order (exact) and finished. A warp
// keeps D steps in flight, so with K <= 512 D its whole share is asked for at once.
// Weights do not depend on the previous kernel of the stream (KEA_INT8_PDL promises it): the first loads are issued before
// griddepcontrol.wait.
//
// Measured on a B200 (launches back to back, without programmatic launch): 1 x 4096 x 1024 3.4 us (1.2 TB/s of weights; the
// library's smallest kernels take 2.1 us), 8 x 1024 x 4096 3.7 us, 32 x 4096 x 1024 4.4 us. The first form of this kernel
// (two steps in flight) took 6.5, 13.6 and 9.0 us. From some 64 tokens on every further 32 read all the weights again from L2
// (128 x 4096 x 1024: 13.4 us), and the tcgen05 tiles, which share them, take over.
#pragma once

#include "int8_epilogue.cuh"

namespace kea {

constexpr int kI8RegThreads = 256, kI8RegWarps = 8, kI8RegPad = 4;

KEA_DEVI void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes at column k of a row of K valid bytes (16-byte aligned): zeros past K, and nothing past K is read.
template <bool CONST>
KEA_DEVI uint4 load_codes(const int8_t *row, int k, int K) {
    if (row == nullptr || k >= K) return make_uint4(0u, 0u, 0u, 0u);
    const uint4 *p = reinterpret_cast<const uint4 *>(row + k);
    if (k + 16 <= K) return CONST ? __ldg(p) : *p;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 15; ++i)
        if (k + i < K) w[i >> 2] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int RG, int D, bool HALF>
__global__ void __launch_bounds__(kI8RegThreads, 2) int8_gemm_reg_kernel(const Int8Args a) {
    constexpr int R = 8 * RG, H = HALF ? 1 : 2, CN = 8 * H, KS = kI8RegWarps, LD = 16 + kI8RegPad;
    __shared__ int part[KS * R * LD];   // [slice][token][channel]
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int c0 = blockIdx.x * CN, m0 = blockIdx.y * R;
    const int steps = (a.K + 63) / 64, per = (steps + KS - 1) / KS;
    const int s0 = min(steps, warp * per), s1 = min(steps, s0 + per);

    const int8_t *wrow[H], *qrow[RG];
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const int n = c0 + g + 8 * h;
        wrow[h] = n < a.N ? a.w + (long long)n * a.ldw : nullptr;
    }
#pragma unroll
    for (int r = 0; r < RG; ++r) {
        const int m = m0 + 8 * r + g;
        qrow[r] = m < a.M ? a.q + (long long)m * a.ldq : nullptr;
    }

    uint4 wr[D][H], br[D][RG];
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int h = 0; h < H; ++h) wr[d][h] = load_codes<true>(wrow[h], s0 + d < s1 ? 64 * (s0 + d) + 16 * t : a.K, a.K);
    grid_dependency_wait();
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int r = 0; r < RG; ++r) br[d][r] = load_codes<false>(qrow[r], s0 + d < s1 ? 64 * (s0 + d) + 16 * t : a.K, a.K);

    int acc[RG][4];
#pragma unroll
    for (int r = 0; r < RG; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][i] = 0;

    for (int base = s0; base < s1; base += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int s = base + d;
            if (s >= s1) break;
            const uint4 lo = wr[d][0], hi = HALF ? make_uint4(0u, 0u, 0u, 0u) : wr[d][H - 1];
#pragma unroll
            for (int r = 0; r < RG; ++r) {
                mma_s8(acc[r], lo.x, hi.x, lo.y, hi.y, br[d][r].x, br[d][r].y);
                mma_s8(acc[r], lo.z, hi.z, lo.w, hi.w, br[d][r].z, br[d][r].w);
            }
            if (base + D < s1) {   // this slot's next step
                const int k = s + D < s1 ? 64 * (s + D) + 16 * t : a.K;
#pragma unroll
                for (int h = 0; h < H; ++h) wr[d][h] = load_codes<true>(wrow[h], k, a.K);
#pragma unroll
                for (int r = 0; r < RG; ++r) br[d][r] = load_codes<false>(qrow[r], k, a.K);
            }
        }
    }

    // the D fragment: channels g / g + 8, token rows 2 t / 2 t + 1
    int *own = part + warp * R * LD;
#pragma unroll
    for (int r = 0; r < RG; ++r) {
        const int row = 8 * r + 2 * t;
        own[row * LD + g] = acc[r][0];
        own[(row + 1) * LD + g] = acc[r][1];
        if (!HALF) {
            own[row * LD + g + 8] = acc[r][2];
            own[(row + 1) * LD + g + 8] = acc[r][3];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * CN; i += kI8RegThreads) {
        const int row = i / CN, ch = i % CN, m = m0 + row, n = c0 + ch;
        if (m >= a.M || n >= a.N) continue;
        const uint64_t s = pair_of(a.qs[m], 0.f), alpha = pair_of(__ldg(a.alpha + n), 0.f);
        const uint64_t bias = pair_of(a.bias ? __ldg(a.bias + n) : kI8NoBias, 0.f);
        int v = 0;
#pragma unroll
        for (int w = 0; w < KS; ++w) v += part[(w * R + row) * LD + ch];
        if (a.acc) a.acc[(long long)m * a.ld_acc + n] = v;
        float y, unused;
        unpair(a.silu ? int8_values<true>(v, 0, s, alpha, bias) : int8_values<false>(v, 0, s, alpha, bias), y, unused);
        int8_store<T>(a, m, n, y);
    }
}

}  // namespace kea
