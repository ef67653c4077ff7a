// beam_kernels.cuh - one step of a beam search: the best continuations over a clip's hypotheses and the vocabulary, and the
// reordering of the hypotheses' states.
//
// Selection. c[k, v] = score_k + (x[k, v] - lse_k), lse_k = log sum_v exp x[k, v]. Within a hypothesis c falls with x, so
// its `width` largest logits are all it can contribute, and they can be found while the exponentials are summed, before
// lse_k is known. One thread-block cluster serves a clip; each of its warps takes a unit (a hypothesis, or a segment of
// one) and streams its logits once, a tile ahead, keeping
//   * per lane a running maximum m and the sum of 2^((x - m) log2 e), in FP32: x - m is at most zero and loses nothing where
//     it counts, at any level of the logits (masks of the type's lowest value, log-probabilities). (One FMA with m log2 e
//     rounded saves an addition, but that rounding passes the exponential's range below about -2^30.) Where the sum is not
//     a number - a logit that is not one beside others in a lane's tile, or +inf - the unit is summed again with its maximum
//     known, masking what is not a number;
//   * the maximum of every tile.
// The width-th largest of the lane maxima of all the CTA's warps at a hypothesis bounds its best logits from below: only
// the few tiles whose maximum reaches it are read again (from the caches), and what reaches it in them, a little more
// than `width` values in all, enters the warp's list. (Keeping the lists up to date while streaming made every warp pay
// for its own `width` best: 3300 instructions for 2048 logits; one clip of 8 x 131072 FP32 logits 43 us, 20 so.) Candidates are
// gathered in shared memory and enter 32 at a time: every lane counts how many candidates and list entries are ahead of
// its own, independent comparisons.
// The units' sums and lists meet in the first CTA of the cluster (distributed shared memory), which forms every lse_k, merges
// each hypothesis' lists by (logit, label) and then the hypotheses' by (c, hypothesis, place). Many logits can have one c:
// ordering the units' lists by c and label would choose by how a row was split, a unit's list being by logit. No scratch
// memory, one launch.
#pragma once

#include "operator_common.cuh"

namespace kea {

constexpr int kBeamMax = 32;          // hypotheses and width
constexpr int kBeamCluster = 16;      // CTAs per clip at most
constexpr int kBeamSlots = 32;        // units per CTA at most: 32 hypotheses, or 32 warps with one each

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

// An unsigned key in the order of the floats (no NaN; -0 as 0).
KEA_DEVI uint32_t float_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
KEA_DEVI float key_float(uint32_t k) { return __uint_as_float(k ^ ((uint32_t)((int)~k >> 31) | 0x80000000u)); }

// An entry of a list: larger values first, equal ones by index, as one number to compare; 0: an empty place.
KEA_DEVI uint64_t beam_entry(float v, int i) { return (uint64_t)float_key(v) << 32 | (uint32_t)~i; }
KEA_DEVI float entry_value(uint64_t e) { return key_float((uint32_t)(e >> 32)); }
KEA_DEVI int entry_index(uint64_t e) { return (int)~(uint32_t)e; }

// The lanes' values in descending order.
KEA_DEVI float sorted(float v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const float u = __shfl_xor_sync(0xFFFFFFFFu, v, j);
            v = ((lane & k) == 0) == ((lane & j) == 0) ? fmaxf(v, u) : fminf(v, u);
        }
    return v;
}

// A warp's scratch: candidates on their way into its list, and the list while it is put together.
struct __align__(16) BeamScratch {
    uint64_t cand[64 + 2];
    uint64_t list[kBeamMax + 2];
};

// Merges the first n <= 32 candidates of s.cand into the warp's sorted list: lane j < width holds the j-th entry, the
// others nothing (0). Every lane counts what is ahead of its own entry and of its own candidate.
KEA_DEVI void beam_merge(BeamScratch &s, int n, int width, int lane, uint64_t &list) {
    const uint64_t mine = lane < n ? s.cand[lane] : 0;
    s.list[lane] = list;
    if (lane == 0) {   // the loops take two at a time
        if (n & 1) s.cand[n] = 0;
        if (width & 1) s.list[width] = 0;
    }
    __syncwarp();
    int place = lane, rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 2) {
        const ulonglong2 c = *reinterpret_cast<const ulonglong2 *>(s.cand + j);
        place += (c.x > list) + (c.y > list);
        rank += (c.x > mine) + (c.y > mine);
    }
#pragma unroll 4
    for (int j = 0; j < width; j += 2) {
        const ulonglong2 l = *reinterpret_cast<const ulonglong2 *>(s.list + j);
        rank += (l.x > mine) + (l.y > mine);
    }
    __syncwarp();
    if (lane < width && place < width) s.list[place] = list;
    if (mine && rank < width) s.list[rank] = mine;
    __syncwarp();
    if (lane < width) list = s.list[lane];
    __syncwarp();
}

KEA_DEVI uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

// A sequence that falls and rises (or the other way round) over each group of P lanes, P a power of two, in descending order.
KEA_DEVI uint64_t beam_order(uint64_t v, int P, int lane) {
    for (int j = P / 2; j > 0; j /= 2) {
        const uint64_t u = __shfl_xor_sync(0xFFFFFFFFu, v, j);
        v = ((lane & j) == 0) == (u > v) ? u : v;
    }
    return v;
}

// Merges `lists` sorted lists, list i in lanes i P .. i P + P - 1 of e, into the warp's (in the first P lanes): the larger of one
// list's entry and the other's from its end are the best P of both.
KEA_DEVI void beam_merge_lists(uint64_t e, int lists, int P, int lane, uint64_t &list) {
    for (int w = P; w < P * lists; w *= 2) e = beam_order(larger(e, __shfl_xor_sync(0xFFFFFFFFu, e, w | (P - 1))), P, lane);
    if (__any_sync(0xFFFFFFFFu, list != 0)) list = beam_order(larger(list, __shfl_xor_sync(0xFFFFFFFFu, e, P - 1)), P, lane);
    else list = e;
}

struct BeamScan {
    float m = -INFINITY, from = 0.f;  // this lane's maximum; the same, 0 while there is none
    float s = 0.f;                    // sum of 2^((x - from) log2 e)
    uint32_t tiles = 0;               // key of the largest logit in this lane's group of tiles
    float side = -INFINITY;           // this lane's value before the first or after the last vector
    uint64_t list = 0;                // lane i: the i-th best logit
};

constexpr float kLog2e = 1.4426950408889634f;

KEA_DEVI float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Adds E values per lane (absent ones -inf) to the lane's maximum and sum; returns their maximum (no NaN).
template <int E>
KEA_DEVI float beam_add(BeamScan &c, const float (&x)[E]) {
    float tm = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) tm = fmaxf(tm, x[e]);
    if (tm > c.m) {
        c.s = c.m == -INFINITY ? 0.f : c.s * exp2_approx((c.m - tm) * kLog2e);   // nothing counts before the first finite logit
        c.m = c.from = tm;
    }
    if constexpr (E == 1) {
        c.s += exp2_approx((x[0] - c.from) * kLog2e);
    } else {
        const uint64_t scale = pair_of(kLog2e, kLog2e), from = pair_of(-c.from, -c.from);
        uint64_t sum = pair_of(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float a, b;
            unpair(mul2(add2(pair_of(x[e], x[e + 1]), from), scale), a, b);
            sum = add2(sum, pair_of(exp2_approx(a), exp2_approx(b)));
        }
        float a, b;
        unpair(sum, a, b);
        c.s += a + b;
    }
    return tm;
}

// A warp's candidates on their way into its list.
struct BeamGather {
    BeamScratch &s;
    uint64_t &list;
    int width, lane, n = 0;
    KEA_DEVI BeamGather(BeamScratch &scratch, uint64_t &l, int w, int ln) : s(scratch), list(l), width(w), lane(ln) {}
    KEA_DEVI void flush(int k) {
        __syncwarp();
        beam_merge(s, k, width, lane, list);
    }
    KEA_DEVI void offer(bool good, uint64_t entry) {
        const uint64_t end = __shfl_sync(0xFFFFFFFFu, list, width - 1);
        good = good && entry > end;
        const uint32_t votes = __ballot_sync(0xFFFFFFFFu, good);
        if (votes == 0) return;
        if (good) s.cand[n + __popc(votes & ((1u << lane) - 1u))] = entry;
        n += __popc(votes);
        if (n > 32) {
            flush(32);
            const uint64_t e = lane + 32 < n ? s.cand[32 + lane] : 0;
            __syncwarp();
            if (lane + 32 < n) s.cand[lane] = e;   // what is left moves down
            __syncwarp();
            n -= 32;
        }
    }
    KEA_DEVI void finish() {
        if (n) flush(n);
    }
};

template <typename T> struct BeamVec;   // a 16-byte vector of logits
template <> struct BeamVec<float> {
    static constexpr int N = 4;
    static constexpr uint32_t kNone = 0xFF800000u;   // -inf
    static KEA_DEVI void get(const uint4 &w, float *v) {
        v[0] = __uint_as_float(w.x);
        v[1] = __uint_as_float(w.y);
        v[2] = __uint_as_float(w.z);
        v[3] = __uint_as_float(w.w);
    }
};
template <typename T> struct BeamVec {
    static constexpr int N = 8;
    static constexpr uint32_t kNone = sizeof(T) == 2 && TypeCode<T>::value == KEA_TYPE_F16 ? 0xFC00FC00u : 0xFF80FF80u;
    static KEA_DEVI void get(const uint4 &w, float *v) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(u[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};

// A unit: logits lo .. hi - 1 of a row, as whole 16-byte vectors in tiles and the values before the first and after the
// last vector (one per lane).
template <typename T>
struct BeamUnit {
    using Vec = BeamVec<T>;
    static constexpr int N = Vec::N, V = sizeof(T) == 4 ? 4 : 2, E = N * V, TILE = 32 * V;   // vectors per tile
    const T *row;
    int lane, first, vecs, edge, group;   // group: tiles that share a lane's maximum
    bool at_edge;
    KEA_DEVI BeamUnit(const T *r, int lo, int hi, int l) : row(r), lane(l) {
        const int head = min(hi - lo, (int)((16u - ((uint32_t)(reinterpret_cast<uintptr_t>(row + lo)) & 15u)) & 15u) / (int)sizeof(T));
        first = lo + head;
        vecs = (hi - first) / N;
        const int last = first + vecs * N;
        edge = lane < 16 ? lo + lane : last + lane - 16;   // at most 7 values on either side
        at_edge = lane < 16 ? lane < head : edge < hi;
        group = ((vecs + TILE - 1) / TILE + 31) / 32;
    }
    KEA_DEVI void load(int v0, uint4 (&w)[V]) const {
        const uint4 *p = reinterpret_cast<const uint4 *>(row + first);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int v = v0 + 32 * j + lane;
            w[j] = make_uint4(Vec::kNone, Vec::kNone, Vec::kNone, Vec::kNone);
            if (v < vecs) w[j] = p[v];
        }
    }
    KEA_DEVI void values(const uint4 (&w)[V], float (&x)[E]) const {
#pragma unroll
        for (int j = 0; j < V; ++j) Vec::get(w[j], x + j * N);
    }
    KEA_DEVI void scan(BeamScan &c) const {
        if (at_edge) c.side = to_float(row[edge]);
        uint4 next[V];
        load(0, next);
        int left = group, owner = 0;
        for (int v0 = 0; v0 < vecs; v0 += TILE) {
            float x[E];
            values(next, x);
            load(v0 + TILE, next);
            const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, float_key(beam_add(c, x)));
            if (lane == owner) c.tiles = max(c.tiles, top);
            if (--left == 0) {
                left = group;
                ++owner;
            }
        }
        const float side[1] = {c.side};
        beam_add(c, side);
    }
    // the values that reach `low`, into the list; tiles come by index, so once the list is full a later value has to exceed
    // its last (a row of one value, or a segment that is masked whole, would be offered value by value)
    KEA_DEVI void gather(BeamScan &c, float low, int width, BeamScratch &s) const {
        BeamGather g(s, c.list, width, lane);
        uint32_t need = max(float_key(low), float_key(-INFINITY) + 1);   // key of the least value that can enter
        uint32_t todo = __ballot_sync(0xFFFFFFFFu, c.tiles >= need);
        while (todo) {
            const int owner = __ffs(todo) - 1, v1 = (owner + 1) * group * TILE;
            todo &= todo - 1;
            if (__shfl_sync(0xFFFFFFFFu, c.tiles, owner) < need) continue;
            for (int v0 = v1 - group * TILE; v0 < min(v1, vecs); v0 += TILE) {
                uint4 w[V];
                load(v0, w);
                float x[E];
                values(w, x);
                const float least = key_float(need);
                uint32_t mask = 0;   // this lane's values that do
#pragma unroll
                for (int e = 0; e < E; ++e) mask |= (x[e] >= least ? 1u : 0u) << e;
                while (__any_sync(0xFFFFFFFFu, mask != 0)) {   // one of every lane at a time, hardly ever more than one
                    const int e = mask ? __ffs(mask) - 1 : 0;
                    const int i = first + (v0 + 32 * (e / N) + lane) * N + e % N;
                    g.offer(mask != 0, mask ? beam_entry(to_float(row[i]), i) : 0);
                    mask &= mask - 1;
                }
                const uint64_t end = __shfl_sync(0xFFFFFFFFu, c.list, width - 1);
                if (end) need = max(need, (uint32_t)(end >> 32) + 1);
            }
        }
        g.offer(c.side >= low && c.side > -INFINITY, beam_entry(c.side, edge));
        g.finish();
    }
};

// log sum exp of logits lo .. hi - 1, the warp's lanes having scanned them; not a number: a logit of +inf.
template <typename T>
KEA_DEVI double beam_log_sum(const BeamScan &c, const T *row, int lo, int hi, int lane) {
    float m = c.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (m == -INFINITY) return -INFINITY;
    float s = c.m == -INFINITY ? 0.f : c.s * exp2_approx((c.m - m) * kLog2e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (s < INFINITY) return (double)m + (double)logf(s);
    s = 0.f;
    for (int i = lo + lane; i < hi; i += 32) {
        const float x = to_float(row[i]);
        if (x == x) s += expf(x - m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    return (double)m + (double)logf(s);
}

KEA_DEVI double ld_cluster_f64(uint32_t addr) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}
KEA_DEVI uint64_t ld_cluster_u64(uint32_t addr) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}

// CTAs of 8 warps: four share an SM (with the 80 registers that the compiler would take for FP32, three: 256 x 8 x 1025 is then a
// second wave, 16.5 instead of 12.2 us).
template <typename T, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 32 / WARPS) beam_select_kernel(const BeamArgs a) {
    __shared__ double ul[kBeamSlots];                  // the units' log-sums
    __shared__ uint64_t ue[kBeamSlots * kBeamMax];     // and lists: [slot][width]
    __shared__ uint64_t lists[kBeamMax * kBeamMax];    // (first CTA) the hypotheses' lists: [hypothesis][width]
    __shared__ float tops[2 * WARPS];                  // per warp: two of its largest lane maxima
    __shared__ float score[kBeamMax], lse[kBeamMax];   // per hypothesis; lse not a number: it offers nothing
    __shared__ bool over[kBeamMax];                    // it has ended
    __shared__ BeamScratch scratch[WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ctas = a.ctas, rank = (int)blockIdx.x % ctas, b = (int)blockIdx.x / ctas;   // a cluster is `ctas` consecutive CTAs
    const int warps = ctas * WARPS, K = a.beams, W = a.width;
    BeamScratch &own = scratch[warp];
    grid_dependency_wait();
    grid_launch_dependents();
    if (threadIdx.x < K) {
        score[threadIdx.x] = a.scores[(long long)b * K + threadIdx.x];
        over[threadIdx.x] = a.ended && a.ended[(long long)b * K + threadIdx.x];
    }
    __syncthreads();

    // Several rounds only where every unit is a whole hypothesis; segments of one have one round, in which the warps of a
    // CTA at the same hypothesis agree on its bound.
    for (int r = 0; r < a.rounds; ++r) {
        const int unit = r * warps + rank * WARPS + warp, slot = r * WARPS + warp;
        const bool some = unit < a.units;
        const int k = some ? unit / a.segs : 0, seg = unit - k * a.segs;
        const bool scans = some && !over[k];
        const T *row = static_cast<const T *>(a.logits) + (long long)b * a.ld_clip + (long long)k * a.ld_beam;
        const int per = (a.vocab + a.segs - 1) / a.segs, lo = scans ? min(a.vocab, seg * per) : 0, hi = scans ? min(a.vocab, lo + per) : 0;
        BeamScan c;
        const BeamUnit<T> u(row, lo, hi, lane);
        if (scans) {
            u.scan(c);
            const double sum = beam_log_sum(c, row, lo, hi, lane);
            if (lane == 0) ul[slot] = sum;
        } else if (some && seg == 0 && lane == 0) {
            c.list = beam_entry(0.f, a.end);
        }
        // `width` lanes of this warp reach low; of the n warps of this CTA at the hypothesis each has ceil(width / n) lanes
        // that reach its own such value, so `width` lanes of them all reach the least of those
        const float best = sorted(c.m, lane);
        float low = __shfl_sync(0xFFFFFFFFu, best, W - 1);
        if (a.segs > 1) {
            const int w0 = max(0, warp - seg), n = max(1, min(WARPS, warp - seg + a.segs) - w0);   // its first warp, their number
            const float few = __shfl_sync(0xFFFFFFFFu, best, (W + n - 1) / n - 1);
            if (lane == 0) {
                tops[warp] = low;
                tops[WARPS + warp] = few;
            }
            __syncthreads();
            const float other = lane < n ? tops[w0 + lane] : -INFINITY, least = lane < n ? tops[WARPS + w0 + lane] : INFINITY;
            low = fmaxf(key_float(__reduce_max_sync(0xFFFFFFFFu, float_key(other))),
                        key_float(__reduce_min_sync(0xFFFFFFFFu, float_key(least))));
        }
        if (scans) u.gather(c, low, W, own);
        if (some && lane < W) ue[slot * W + lane] = c.list;
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();

    if (rank == 0) {
        // where unit u's results lie: CTA (u % warps) / WARPS, slot (u / warps) * WARPS + u % WARPS
        const auto at = [&](const void *base, int u, int each, int i) {
            const int r = a.rounds == 1 ? 0 : u / warps, w = u - r * warps;
            return map_to_rank(smem_u32(base) + 8u * (uint32_t)((r * WARPS + w % WARPS) * each + i), (uint32_t)(w / WARPS));
        };
        int P = 1;   // lists come in P places, `each` per turn; this lane's list and place in it
        while (P < W) P *= 2;
        const int each = 32 / P, mine = lane / P, q = lane - mine * P;
        uint64_t list = 0;
        // The hypotheses' log-sums, and their lists (by logit and label), shared by `parts` warps where they are few and long:
        // as many as leave every warp one job.
        const int parts = min(max(1, WARPS / K - 1), (a.segs + each - 1) / each);
        for (int job = warp; job < K + K * parts; job += WARPS) {
            if (job < K) {
                const int k = job;
                if (over[k]) continue;   // it needs none
                const double own_sum = lane < a.segs ? ld_cluster_f64(at(ul, k * a.segs + lane, 1, 0)) : (double)-INFINITY;
                double top = fmax((double)-INFINITY, own_sum);   // (a number)
                for (int g = lane + 32; g < a.segs; g += 32) top = fmax(top, ld_cluster_f64(at(ul, k * a.segs + g, 1, 0)));
                for (int o = 1; o < min(a.segs, 32); o *= 2) top = fmax(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                top = __shfl_sync(0xFFFFFFFFu, top, 0);
                // a segment with a logit of +inf is not a number, and makes the whole so
                float s = lane < a.segs ? expf((float)(own_sum - top)) : 0.f;
                for (int g = lane + 32; g < a.segs; g += 32) s += expf((float)(ld_cluster_f64(at(ul, k * a.segs + g, 1, 0)) - top));
                for (int o = 1; o < min(a.segs, 32); o *= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
                if (lane == 0) {
                    // nothing is offered where it is infinite (no label left) or not a number
                    const float l = (float)(top + (double)logf(s));
                    lse[k] = fabsf(l) < INFINITY ? l : __int_as_float(0x7FC00000);
                }
            } else {
                const int k = (job - K) / parts, part = job - K - k * parts;
                list = 0;
                if (a.segs == 1) {
                    if (lane < W) list = ld_cluster_u64(at(ue, k, W, lane));
                } else {
                    for (int g0 = part * each; g0 < a.segs; g0 += parts * each) {
                        const int g = g0 + mine;
                        beam_merge_lists(g < a.segs && q < W ? ld_cluster_u64(at(ue, k * a.segs + g, W, q)) : 0, min(each, a.segs - g0), P,
                                         lane, list);
                    }
                }
                if (lane < W) lists[(parts == 1 ? k : job) * W + lane] = list;
            }
        }
        __syncthreads();
        if (parts > 1) {   // slots K .. K (1 + parts) - 1, below WARPS, hold the parts
            if (warp < K) {
                const int first = K + warp * parts;
                list = lane < W ? lists[first * W + lane] : 0;
                for (int p = 1; p < parts; p += each) {
                    const int from = p + mine;
                    beam_merge_lists(from < parts && q < W ? lists[(first + from) * W + q] : 0, min(each, parts - p), P, lane, list);
                }
                if (lane < W) lists[warp * W + lane] = list;
            }
            __syncthreads();
        }
        // The hypotheses' lists by c, hypothesis and place in the list: c does not rise along a list, so each stays in its order.
        // Where one warp would take more than two turns, up to eight do and the first takes theirs.
        const int turns = (K + each - 1) / each, takers = turns <= 2 ? 1 : min(min(WARPS, 8), turns);
        list = 0;
        if (warp < takers)
            for (int k0 = warp * each; k0 < K; k0 += takers * each) {
                const int k = k0 + mine;
                uint64_t e = 0;
                if (k < K && q < W) {
                    const float s = score[k], l = over[k] ? 0.f : lse[k];
                    e = lists[k * W + q];
                    const float c = over[k] ? s : __fadd_rn(__fsub_rn(entry_value(e), l), s);
                    e = e && l == l && fabsf(s) < INFINITY && c > -INFINITY ? beam_entry(c, k * kBeamMax + q) : 0;
                }
                beam_merge_lists(e, min(each, K - k0), P, lane, list);
            }
        if (takers > 1) {
            __syncwarp();
            own.list[lane] = list;
            __syncthreads();
            if (warp == 0)
                for (int w = 1; w < takers; w += each) {
                    const int from = w + mine;
                    beam_merge_lists(from < takers && q < W ? scratch[from].list[q] : 0, min(each, takers - w), P, lane, list);
                }
        }
        if (warp == 0) {
            // Places left over take what is not offered, by flat index: the lowest numbers that the list does not hold
            // (at most 31 are taken, so 63 numbers are enough).
            const uint32_t some = __ballot_sync(0xFFFFFFFFu, lane < W && list != 0);
            float v = entry_value(list);
            int i = 0;   // the flat index
            if (some >> lane & 1) {
                const int place = entry_index(list), k = place / kBeamMax;
                i = k * a.vocab + entry_index(lists[k * W + place % kBeamMax]);
            }
            if (__popc(some) < W) {
                uint32_t low = 0, high = 0;   // flat indices 0 .. 31 and 32 .. 63 that the list holds
                if (some >> lane & 1) {
                    if (i < 32) low = 1u << i;
                    else if (i < 64) high = 1u << (i - 32);
                }
                uint64_t open = ~(((uint64_t)__reduce_or_sync(0xFFFFFFFFu, high) << 32) | __reduce_or_sync(0xFFFFFFFFu, low));
                for (int j = __popc(some); j < lane; ++j) open &= open - 1;
                if (lane < W && lane >= __popc(some)) {
                    v = -INFINITY;
                    i = __ffsll((long long)open) - 1;
                }
            }
            if (lane < W) {
                const long long o = (long long)b * W + lane;
                const int k = i / a.vocab, label = i - k * a.vocab;
                a.out_scores[o] = v;
                a.parents[o] = k;
                a.labels[o] = label;
                if (a.out_ended) a.out_ended[o] = label == a.end || over[k] ? 1 : 0;
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
