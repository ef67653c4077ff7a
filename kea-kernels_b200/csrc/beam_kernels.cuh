// beam_kernels.cuh - one step of a beam search: the best continuations over a clip's hypotheses and the vocabulary, and the
// reordering of the hypotheses' states.
//
// Selection. c[k, v] = score_k + (x[k, v] - lse_k), lse_k = log sum_v exp x[k, v]. Within a hypothesis c falls with x, so
// its `width` largest logits are all it can contribute, and they can be found in the same pass that sums the
// exponentials, before lse_k is known: the logits are read once. One thread-block cluster serves a clip; each of its
// warps takes a unit (a hypothesis, or a segment of one) and keeps, while it streams the logits,
//   * per lane a running maximum m and the sum of 2^(x log2 e - off), off = m log2 e rounded, in FP32; the log-sum is
//     (off + log2 of the sum) / log2 e, so the rounding of off cancels. Where that is not finite - a logit that is not a
//     number, or one so large that off overflows - the unit is summed again with its maximum known, masking what is not
//     a number;
//   * across its lanes the unit's best logits, lane i the i-th best with its index. A logit enters only if it is above
//     the last of them, which after the first few hundred values is rare, so the common path is one maximum per value and
//     one vote per tile. Where many lanes of a tile pass, the width-th largest of the lane maxima is a bound below which
//     no value of the tile can enter.
// The units' sums and lists meet in the first CTA of the cluster (distributed shared memory), which forms every lse_k and
// merges the lists by (c, flat index). No scratch memory, one launch.
#pragma once

#include "operator_common.cuh"

namespace kea {

constexpr int kBeamThreads = 256, kBeamWarps = 8;
constexpr int kBeamMax = 32;          // hypotheses and width
constexpr int kBeamCluster = 8;       // CTAs per clip at most
constexpr int kBeamRounds = 4;        // units per warp at most: kBeamMax hypotheses / 8 warps
constexpr int kBeamNone = 0x7FFFFFFF; // index of an empty place

struct BeamArgs {
    const void *logits;
    long long ld_clip, ld_beam;
    const float *scores;
    const uint8_t *ended;
    float *out_scores;
    int *parents, *labels;
    uint8_t *out_ended;
    int beams, vocab, width, end;
    int ctas;                         // CTAs per clip: the cluster's size
    int segs, units, rounds;          // segments per hypothesis, beams * segs, units per warp
};

// Order of the list: larger values first, equal ones by index.
KEA_DEVI bool beam_before(float av, int ai, float bv, int bi) { return av > bv || (av == bv && ai < bi); }

// Enters (v, i) (the same in every lane) into the warp's sorted list, lane j holding the j-th.
KEA_DEVI void beam_insert(float v, int i, int lane, float &lv, int &li) {
    const uint32_t ahead = __ballot_sync(0xFFFFFFFFu, beam_before(lv, li, v, i));
    const int pos = __popc(ahead);
    const float uv = __shfl_up_sync(0xFFFFFFFFu, lv, 1);
    const int ui = __shfl_up_sync(0xFFFFFFFFu, li, 1);
    if (lane > pos) {
        lv = uv;
        li = ui;
    } else if (lane == pos) {
        lv = v;
        li = i;
    }
}

// An unsigned key in the order of the floats (no NaN).
KEA_DEVI uint32_t float_key(float v) {
    const uint32_t u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
KEA_DEVI float key_float(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }

// The n-th largest of the lanes' values.
KEA_DEVI float nth_largest(float v, int n, int lane) {
    uint32_t key = float_key(v), top = 0;
    for (int i = 0; i < n; ++i) {
        top = __reduce_max_sync(0xFFFFFFFFu, key);
        const uint32_t at = __ballot_sync(0xFFFFFFFFu, key == top);
        if (lane == __ffs(at) - 1) key = 0;
    }
    return key_float(top);
}

struct BeamScan {
    float m = -INFINITY, off = 0.f;   // this lane's maximum and m log2 e (0 while there is none)
    float s = 0.f;                    // sum of 2^(x log2 e - off)
    float lv = -INFINITY;             // the list
    int li = kBeamNone;
};

constexpr float kLog2e = 1.4426950408889634f;

KEA_DEVI float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// E values per lane of one tile, x[e] at row index `index(e)` (ascending in the tile for ascending (e / EPV, lane, e %
// EPV)); absent ones are -inf.
template <typename T, int E, typename Index>
KEA_DEVI void beam_tile(BeamScan &c, const float (&x)[E], const T *row, int width, int lane, Index index) {
    float tm = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) tm = fmaxf(tm, x[e]);
    if (tm > c.m) {
        const float off = tm * kLog2e;
        c.s *= exp2_approx(c.off - off);   // 0 before the first finite logit
        c.m = tm;
        c.off = off;
    }
    const float off = c.off;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        s0 += exp2_approx(fmaf(x[e], kLog2e, -off));
        if (e + 1 < E) s1 += exp2_approx(fmaf(x[e + 1], kLog2e, -off));
    }
    c.s += s0 + s1;

    const float worst = __shfl_sync(0xFFFFFFFFu, c.lv, width - 1);
    const uint32_t pass = __ballot_sync(0xFFFFFFFFu, tm > worst);
    if (pass == 0) return;
    const float bound = __popc(pass) >= width ? nth_largest(tm, width, lane) : -INFINITY;
    uint32_t mask = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) mask |= (x[e] > worst && x[e] >= bound) ? 1u << e : 0u;
    int entered = 0;
    while (true) {
        const uint32_t mine = mask ? (uint32_t)index(__ffs(mask) - 1) : 0xFFFFFFFFu;
        const uint32_t next = __reduce_min_sync(0xFFFFFFFFu, mine);
        if (next == 0xFFFFFFFFu) break;
        const float v = to_float(row[next]);
        if (mine == next) mask &= mask - 1;
        const float lw = __shfl_sync(0xFFFFFFFFu, c.lv, width - 1);
        const int iw = __shfl_sync(0xFFFFFFFFu, c.li, width - 1);
        if (!beam_before(v, (int)next, lw, iw)) continue;
        beam_insert(v, (int)next, lane, c.lv, c.li);
        if (++entered == width) {   // the tile has filled the list: drop what is no longer above its end
            entered = 0;
            const float nw = __shfl_sync(0xFFFFFFFFu, c.lv, width - 1);
            uint32_t keep = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) keep |= (x[e] > nw) ? 1u << e : 0u;   // equal ones come later: behind
            mask &= keep;
        }
    }
}

template <typename T> struct BeamVec;   // a 16-byte vector of logits
template <> struct BeamVec<float> {
    static constexpr int N = 4;
    static KEA_DEVI void get(const float *p, float *v) {
        const float4 w = *reinterpret_cast<const float4 *>(p);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    }
};
template <typename T> struct BeamVec {
    static constexpr int N = 8;
    static KEA_DEVI void get(const T *p, float *v) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(u[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};

// One value per lane at lo + lane < hi.
template <typename T>
KEA_DEVI void beam_edge(BeamScan &c, const T *row, int lo, int hi, int width, int lane) {
    if (lo >= hi) return;
    float x[1] = {-INFINITY};
    if (lo + lane < hi) {
        x[0] = to_float(row[lo + lane]);
    }
    beam_tile<T, 1>(c, x, row, width, lane, [&](int) { return lo + lane; });
}

// Logits lo .. hi - 1 of a row.
template <typename T>
KEA_DEVI void beam_scan(BeamScan &c, const T *row, int lo, int hi, int width, int lane) {
    constexpr int N = BeamVec<T>::N, V = 4, E = N * V;
    const int head = min(hi - lo, (int)((16u - ((uint32_t)(reinterpret_cast<uintptr_t>(row + lo)) & 15u)) & 15u) / (int)sizeof(T));
    beam_edge(c, row, lo, lo + head, width, lane);
    lo += head;
    const int vecs = (hi - lo) / N;
    for (int v0 = 0; v0 < vecs; v0 += 32 * V) {
        float x[E];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int v = v0 + 32 * j + lane;
            if (v < vecs) {
                BeamVec<T>::get(row + lo + v * N, x + j * N);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) x[j * N + i] = -INFINITY;
            }
        }
        beam_tile<T, E>(c, x, row, width, lane, [&](int e) { return lo + (v0 + 32 * (e / N) + lane) * N + e % N; });
    }
    beam_edge(c, row, lo + vecs * N, hi, width, lane);
}

// log sum exp of logits lo .. hi - 1, the warp's lanes having scanned them; not a number: a logit of +inf.
template <typename T>
KEA_DEVI double beam_log_sum(const BeamScan &c, const T *row, int lo, int hi, int lane) {
    constexpr double kLn2 = 0.6931471805599453;
    float m = c.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (m == -INFINITY) return -INFINITY;
    float off = c.m == -INFINITY ? -INFINITY : c.off;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) off = fmaxf(off, __shfl_xor_sync(0xFFFFFFFFu, off, o));
    float s = c.m == -INFINITY ? c.s : c.s * exp2_approx(c.off - off);   // a lane of NaN alone keeps its NaN
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (s < INFINITY && fabsf(off) < INFINITY) return (double)off * kLn2 + (double)logf(s);
    s = 0.f;
    for (int i = lo + lane; i < hi; i += 32) {
        const float x = to_float(row[i]);
        if (x == x) s += expf(x - m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    return (double)m + (double)logf(s);
}

KEA_DEVI float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

KEA_DEVI double ld_cluster_f64(uint32_t addr) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kBeamThreads) beam_select_kernel(const BeamArgs a) {
    constexpr int SLOTS = kBeamRounds * kBeamWarps;
    __shared__ double ul[SLOTS];                                      // the units' log-sums
    __shared__ float uv[SLOTS * kBeamMax];                            // and lists: [slot][width]
    __shared__ int ui[SLOTS * kBeamMax];
    __shared__ float lse[kBeamMax];                                   // first CTA: per hypothesis, NaN: offers nothing
    __shared__ float wv[kBeamWarps * kBeamMax];                       // first CTA: the warps' merged lists
    __shared__ int wi[kBeamWarps * kBeamMax];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ctas = a.ctas, rank = (int)blockIdx.x % ctas, b = (int)blockIdx.x / ctas;   // a cluster is `ctas` consecutive CTAs
    const int warps = ctas * kBeamWarps, K = a.beams, W = a.width;
    grid_dependency_wait();
    grid_launch_dependents();

    for (int r = 0; r < a.rounds; ++r) {
        const int unit = r * warps + rank * kBeamWarps + warp, slot = r * kBeamWarps + warp;
        if (unit >= a.units) break;
        const int k = unit / a.segs, seg = unit - k * a.segs;
        BeamScan c;
        if (a.ended && a.ended[(long long)b * K + k]) {
            if (seg == 0 && lane == 0) {
                c.lv = 0.f;
                c.li = a.end;
            }
        } else {
            const T *row = static_cast<const T *>(a.logits) + (long long)b * a.ld_clip + (long long)k * a.ld_beam;
            const int per = (a.vocab + a.segs - 1) / a.segs;
            const int lo = min(a.vocab, seg * per);
            const int hi = min(a.vocab, lo + per);
            beam_scan(c, row, lo, hi, W, lane);
            const double sum = beam_log_sum(c, row, lo, hi, lane);
            if (lane == 0) ul[slot] = sum;
        }
        if (lane < W) {
            uv[slot * W + lane] = c.lv;
            ui[slot * W + lane] = c.li;
        }
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();

    if (rank == 0) {
        // where unit u's results lie: CTA (u % warps) / 8, slot (u / warps) * 8 + u % 8
        const auto at = [&](const void *base, int u, int words, int i) {
            const int r = u / warps, w = u - r * warps;
            return map_to_rank(smem_u32(base) + 4u * (uint32_t)((r * kBeamWarps + (w & (kBeamWarps - 1))) * words + i),
                               (uint32_t)(w / kBeamWarps));
        };
        for (int k = warp; k < K; k += kBeamWarps) {
            // an ended hypothesis needs none
            if (a.ended && a.ended[(long long)b * K + k]) {
                if (lane == 0) lse[k] = 0.f;
                continue;
            }
            double top = -INFINITY;
            for (int g = lane; g < a.segs; g += 32) top = fmax(top, ld_cluster_f64(at(ul, k * a.segs + g, 2, 0)));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            float s = 0.f;   // a segment with a logit of +inf is not a number, and makes the whole so
            for (int g = lane; g < a.segs; g += 32) s += expf((float)(ld_cluster_f64(at(ul, k * a.segs + g, 2, 0)) - top));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            if (lane == 0) {
                // nothing is offered where it is infinite (no label left) or not a number
                const float l = (float)(top + (double)logf(s));
                lse[k] = fabsf(l) < INFINITY ? l : __int_as_float(0x7FC00000);
            }
        }
        __syncthreads();
        float lv = -INFINITY;
        int li = kBeamNone;
        const int entries = a.units * W;
        for (int e0 = warp * 32; e0 < entries; e0 += kBeamThreads) {
            const int e = e0 + lane;
            float v = -INFINITY;
            int i = kBeamNone;
            if (e < entries) {
                const int u = e / W, k = u / a.segs, p = e - u * W;
                i = ld_cluster_s32(at(ui, u, W, p));
                const float l = lse[k];
                const float score = a.scores[(long long)b * K + k];
                if (i != kBeamNone && l == l && fabsf(score) < INFINITY) {
                    const float x = ld_cluster_f32(at(uv, u, W, p));
                    v = (a.ended && a.ended[(long long)b * K + k]) ? score : __fadd_rn(__fsub_rn(x, l), score);
                    i += k * a.vocab;
                } else {
                    i = kBeamNone;
                }
            }
            while (true) {
                const float lw = __shfl_sync(0xFFFFFFFFu, lv, W - 1);
                const int iw = __shfl_sync(0xFFFFFFFFu, li, W - 1);
                const uint32_t pass = __ballot_sync(0xFFFFFFFFu, i != kBeamNone && beam_before(v, i, lw, iw));
                if (pass == 0) break;
                const int src = __ffs(pass) - 1;
                beam_insert(__shfl_sync(0xFFFFFFFFu, v, src), __shfl_sync(0xFFFFFFFFu, i, src), lane, lv, li);
                if (lane == src) i = kBeamNone;
            }
        }
        wv[warp * kBeamMax + lane] = lv;
        wi[warp * kBeamMax + lane] = li;
        __syncthreads();
        if (warp == 0) {
            const int lists = min(kBeamWarps, (entries + 31) / 32);
            for (int w = 1; w < lists; ++w) {
                float v = wv[w * kBeamMax + lane];
                int i = lane < W ? wi[w * kBeamMax + lane] : kBeamNone;
                while (true) {
                    const float lw = __shfl_sync(0xFFFFFFFFu, lv, W - 1);
                    const int iw = __shfl_sync(0xFFFFFFFFu, li, W - 1);
                    const uint32_t pass = __ballot_sync(0xFFFFFFFFu, i != kBeamNone && beam_before(v, i, lw, iw));
                    if (pass == 0) break;
                    const int src = __ffs(pass) - 1;
                    beam_insert(__shfl_sync(0xFFFFFFFFu, v, src), __shfl_sync(0xFFFFFFFFu, i, src), lane, lv, li);
                    if (lane == src) i = kBeamNone;
                }
            }
            // Places left over take what is not offered, by flat index: the lowest numbers that the list does not hold
            // (at most 31 are taken, so 63 numbers are enough).
            const uint32_t some = __ballot_sync(0xFFFFFFFFu, lane < W && li != kBeamNone);
            if (__popc(some) < W) {
                uint32_t low = 0, high = 0;   // flat indices 0 .. 31 and 32 .. 63 that the list holds
                if (lane < W && li < 32) low = 1u << li;
                else if (lane < W && li < 64) high = 1u << (li - 32);
                uint64_t open = ~(((uint64_t)__reduce_or_sync(0xFFFFFFFFu, high) << 32) | __reduce_or_sync(0xFFFFFFFFu, low));
                for (int i = __popc(some); i < lane; ++i) open &= open - 1;
                if (lane < W && lane >= __popc(some)) {
                    lv = -INFINITY;
                    li = __ffsll((long long)open) - 1;
                }
            }
            if (lane < W) {
                const long long o = (long long)b * W + lane;
                const int k = li / a.vocab, v = li - k * a.vocab;
                a.out_scores[o] = lv;
                a.parents[o] = k;
                a.labels[o] = v;
                if (a.out_ended)
                    a.out_ended[o] = v == a.end || (a.ended && a.ended[(long long)b * K + k]) ? 1 : 0;
            }
        }
    }
    if (ctas > 1) cluster_sync_all();   // the first CTA has read the others' shared memory
}

// ---- reordering ----------------------------------------------------------------------------------------------------
struct ReorderItem {
    const uint8_t *src;
    uint8_t *dst;
    long long src_group, src_clip, src_beam, dst_group, dst_clip, dst_beam;
    int unit;                 // bytes per access: 16, 8, 4, 2 or 1
    int row;                  // row length in units
    int rows_per_block;       // > 0: whole rows per block; 0: a block takes kReorderUnits units of one row
    int blocks_per_row;
    unsigned first_block;     // this item's first block
    unsigned rows;            // groups * clips * width
};
constexpr int kReorderThreads = 256, kReorderEach = 4, kReorderUnits = kReorderThreads * kReorderEach;

struct ReorderArgs {
    const int *parents;
    int count, clips, beams, width;
    uint32_t *err;
    ReorderItem item[KEA_REORDER_MAX];
};

template <typename V>
KEA_DEVI void reorder_block(const ReorderArgs &a, const ReorderItem &it, unsigned block) {
    unsigned row0;
    int off, n;   // units this block copies, from unit `off` of row row0 on
    if (it.rows_per_block) {
        row0 = block * it.rows_per_block;
        off = 0;
        n = (int)min((unsigned)it.rows_per_block, it.rows - row0) * it.row;
    } else {
        row0 = block / it.blocks_per_row;
        off = (int)(block - row0 * it.blocks_per_row) * kReorderUnits;
        n = min(kReorderUnits, it.row - off);
    }
    V v[kReorderEach];
    V *dst[kReorderEach];
    const V zero = {};
#pragma unroll
    for (int j = 0; j < kReorderEach; ++j) {
        const int i = (int)threadIdx.x + j * kReorderThreads;
        dst[j] = nullptr;
        if (i >= n) continue;
        const int r = it.rows_per_block ? i / it.row : 0;
        const int u = it.rows_per_block ? i - r * it.row : off + i;
        const unsigned row = row0 + r, w = row % (unsigned)a.width, gb = row / (unsigned)a.width;
        const unsigned b = gb % (unsigned)a.clips, g = gb / (unsigned)a.clips;
        const int p = a.parents[(size_t)b * a.width + w];
        dst[j] = reinterpret_cast<V *>(it.dst + g * it.dst_group + b * it.dst_clip + w * it.dst_beam) + u;
        if (p >= 0 && p < a.beams) {
            v[j] = reinterpret_cast<const V *>(it.src + g * it.src_group + b * it.src_clip + p * it.src_beam)[u];
        } else {
            v[j] = zero;
            if (u == 0) report_error(a.err, KEA_DEVERR_INDEX);
        }
    }
#pragma unroll
    for (int j = 0; j < kReorderEach; ++j)
        if (dst[j]) *dst[j] = v[j];
}

__global__ void __launch_bounds__(kReorderThreads) beam_reorder_kernel(const __grid_constant__ ReorderArgs a) {
    grid_dependency_wait();
    grid_launch_dependents();
    int k = 0;
    while (k + 1 < a.count && blockIdx.x >= a.item[k + 1].first_block) ++k;
    const ReorderItem &it = a.item[k];
    const unsigned block = blockIdx.x - it.first_block;
    switch (it.unit) {
        case 16: reorder_block<uint4>(a, it, block); break;
        case 8: reorder_block<uint2>(a, it, block); break;
        case 4: reorder_block<uint32_t>(a, it, block); break;
        case 2: reorder_block<uint16_t>(a, it, block); break;
        default: reorder_block<uint8_t>(a, it, block); break;
    }
}

}  // namespace kea
