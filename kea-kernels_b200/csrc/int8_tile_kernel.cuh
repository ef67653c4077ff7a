// int8_tile_kernel.cuh - the 8-bit GEMM on the tcgen05 tensor cores: both operands by TMA, INT32 accumulators in tensor
// memory, persistent CTAs (CTAS = 1) or CTA pairs (CTAS = 2, tcgen05 cta_group::2).
//
// A tile is 128 CTAS tokens x BN channels. A CTA holds 128 token rows of it and BN / CTAS channel rows; for a pair the even
// CTA issues the MMAs of both (M 256 x N 256 x K 32), each SM reading only its own shared memory, so a byte of either
// operand serves 256 products. K goes by in blocks of 128 bytes (rows of 128 bytes in the 128-byte swizzle, K-major);
// rows and columns past M, N and K are filled with zeros by the copies. Tensor memory holds two accumulators, so the
// epilogue of one tile runs while the MMAs of the next fill the other.
//
// Warps: 0 producer (one lane: TMA loads); 1 tensor memory and MMA issue; 2 .. epilogue, warp pair (w % 4) reading the
// 32 tensor-memory lanes it may and 64 columns: TMEM -> scales, bias, SiLU, skip connection -> boxes of 32 rows
// x 128 bytes staged in shared memory (128-byte swizzle) -> TMA stores, or row-wise stores where the output's rows are
// not 16-byte aligned. Every wait is bounded; one that runs out is reported in the error word and the kernel ends.
//
// SPLIT (single CTAs, 64 channels): few tiles and a long K. A cluster of 2, 4 or 8 CTAs shares a tile, each taking a slice of
// K (a CTA issues about 100 clocks per MMA whatever its N, so the length of K, not its products, sets a launch's time);
// each sends every other the INT32 sums of the channels that one finishes (distributed shared memory), and after a cluster
// barrier adds the slices' sums of its own, exactly.
//
// Measured on a B200 (M x N x K, launches back to back): pairs, FP16 out, 8192 x 4096 x 1024 31.0 us = 2220 TOPS, with SiLU
// 34.4 us, FP32 out 37.7 us; 32000 x 1024 x 4096 94.4 us = 2840 TOPS, 0.92 of the INT8 rate measured with a library product
// of 8192^3 (3102). With K 1024 the outputs bound it: leaving the stores out (a diagnostic build of an earlier form) gave
// 28.5 instead of 32.0 us. Under load for seconds the power cap lowers the clock (8192 x 1024 x 4096: 28.2 us alone, up to
// 38 us right after a run of larger products). What helped: 128-byte boxes, one per epilogue warp, and five
// stages instead of two boxes and four stages (K 4096: 31.2 -> 28.7 us); the rolled epilogue loop and packed FP32
// arithmetic (below). Sixteen epilogue warps instead of eight: 34.8 us, with SiLU 35.4 (shared memory for four stages
// only). The next 32 columns on their way from tensor memory meanwhile: no gain without SiLU, 40.6 us with.
#pragma once

#include "int8_epilogue.cuh"

namespace kea {

constexpr int kI8K = 128;                 // bytes of K per stage
constexpr uint32_t kI8Half = 128u * kI8K; // 128 rows of a stage
constexpr uint32_t kI8Box = 4096;         // one output box: 32 rows x 128 bytes
constexpr int kI8MaxStages = 8;

template <int CTAS, int BN>
struct Int8Tile {
    static constexpr int CW = BN == 256 ? 128 : 64;                       // columns per epilogue warp
    static constexpr int EPI_WARPS = 4 * (BN / CW), THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int BUFS = BN == 256 ? 1 : 2;                         // staging boxes per epilogue warp
    static constexpr uint32_t B_BYTES = (uint32_t)(BN / CTAS) * kI8K, STAGE = kI8Half + B_BYTES;
    static constexpr uint32_t STAGING = EPI_WARPS * BUFS * kI8Box, CONSTS = EPI_WARPS * CW * 8u;
    static constexpr uint32_t smem(int stages) { return 1024u + (uint32_t)stages * STAGE + STAGING + CONSTS; }
};

struct Int8TileArgs {
    Int8Args a;
    int n_tiles, tiles, kbs, stages;
    int tma_store, res_vec;
    int splits, per_split;    // CTAs that share a tile, blocks of K each takes (SPLIT)
};

KEA_DEVI void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}

KEA_DEVI void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    tmem_ld16(taddr, *reinterpret_cast<uint32_t(*)[16]>(&v[0]));
    tmem_ld16(taddr + 16u, *reinterpret_cast<uint32_t(*)[16]>(&v[16]));
}

// The skip connection's 32 rows x 128 bytes in front of a box: row-wise loads into registers (ahead of their use), then
// into the staging space (swizzled).
template <typename T>
KEA_DEVI void int8_load_residual(const Int8Args &a, uint4 (&v)[8], int row0, int n0) {
    const int lane = threadIdx.x & 31, n = n0 + (lane & 7) * (16 / (int)sizeof(T));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int t = row0 + 4 * i + (lane >> 3);
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (t < a.M && n < a.N)
            v[i] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.res) + (long long)t * a.ld_res + n);
    }
}
KEA_DEVI void int8_stage_residual(const uint4 (&v)[8], uint32_t stg) {
    const int lane = threadIdx.x & 31, piece = lane & 7;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3);
        st_shared16(stg + (uint32_t)r * 128u + (uint32_t)((piece ^ (r & 7)) << 4), v[i].x, v[i].y, v[i].z, v[i].w);
    }
}

// A staged box written row by row: one row's 128 bytes per warp store.
template <typename T>
KEA_DEVI void int8_store_rows(const Int8Args &a, uint32_t stg, int row0, int n0) {
    const int lane = threadIdx.x & 31;
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
        if (row0 + r >= a.M) break;
        uint32_t w;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(stg + (uint32_t)r * 128u + (uint32_t)(((lane >> 2) ^ (r & 7)) << 4) + (uint32_t)(lane & 3) * 4u) : "memory");
        T *dst = static_cast<T *>(a.y) + (long long)(row0 + r) * a.ldy;
        if constexpr (sizeof(T) == 4) {
            if (n0 + lane < a.N) reinterpret_cast<uint32_t *>(dst)[n0 + lane] = w;
        } else {
            uint16_t *d16 = reinterpret_cast<uint16_t *>(dst);
            if (n0 + 2 * lane < a.N) d16[n0 + 2 * lane] = (uint16_t)w;
            if (n0 + 2 * lane + 1 < a.N) d16[n0 + 2 * lane + 1] = (uint16_t)(w >> 16);
        }
    }
}

// One epilogue warp's 32 rows x CW columns of a finished tile, 32 columns at a time. The loop is not unrolled: eight warps run
// its body at different places, and four copies of it missed the instruction cache (the largest stall of the kernel:
// 8192 x 4096 x 1024 with SiLU 58 us, 39 rolled, 34 with packed arithmetic). `ahead` holds the first box's skip connection
// (res_vec), `release` hands the accumulator back. EXTRA: the sums are wanted too, or the skip connection's rows are not
// 16-byte aligned.
template <typename T, bool SILU, bool EXTRA, int CW, int BUFS, typename Release>
KEA_DEVI void int8_epilogue_tile(const Int8TileArgs &p, const CUtensorMap *ymap, uint32_t taddr, uint32_t stg0, uint32_t consts,
                                 int row0, int n0, uint64_t sq, int &box, uint4 (&ahead)[8], Release release) {
    const Int8Args &a = p.a;
    const int lane = threadIdx.x & 31, t = row0 + lane;
    constexpr int NC = 128 / (int)sizeof(T), CHUNKS = CW / 32, PER = NC / 32;   // columns per box, chunks, chunks per box
    constexpr int PIECES = 32 * (int)sizeof(T) / 16, E = 16 / (int)sizeof(T);   // 16-byte pieces of a chunk, values in one
    const bool has_res = a.res != nullptr, staged = has_res && (!EXTRA || p.res_vec);
#pragma unroll 1
    for (int i = 0; i < CHUNKS; ++i) {
        const uint32_t stg = stg0 + (uint32_t)(box % BUFS) * kI8Box, rowaddr = stg + (uint32_t)lane * 128u;
        const int c = 32 * i, nb = n0 + i / PER * NC, piece0 = i % PER * PIECES;
        uint32_t v[32];
        tmem_ld32(taddr + (uint32_t)c, v);
        if (i % PER == 0) {
            if (lane == 0) {   // the store that last read this space is done with it
                if constexpr (BUFS == 2) bulk_wait_group_read1();
                else bulk_wait_group_read0();
            }
            __syncwarp();
            if (staged) {
                int8_stage_residual(ahead, stg);
                if (i + PER < CHUNKS) int8_load_residual<T>(a, ahead, row0, nb + NC);
                __syncwarp();
            }
        }
        tmem_wait_ld();
        tmem_regs_ready(v);
        if (i + 1 == CHUNKS) release();
        if constexpr (EXTRA) {
            if (a.acc && t < a.M) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (n0 + c + j < a.N) a.acc[(long long)t * a.ld_acc + n0 + c + j] = (int)v[j];
            }
        }
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            const ulonglong2 al = ld_shared_pairs(consts + (uint32_t)(c + 4 * g) * 4u);
            const ulonglong2 bi = ld_shared_pairs(consts + (uint32_t)(CW + c + 4 * g) * 4u);
            float f[4];
            unpair(int8_values<SILU>((int)v[4 * g], (int)v[4 * g + 1], sq, al.x, bi.x), f[0], f[1]);
            unpair(int8_values<SILU>((int)v[4 * g + 2], (int)v[4 * g + 3], sq, al.y, bi.y), f[2], f[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * g + j] = __float_as_uint(f[j]);
        }
        if (has_res) {
#pragma unroll
            for (int h = 0; h < PIECES; ++h) {
                float r[E];
                if (staged) {
                    const uint4 u = ld_shared16(rowaddr + (uint32_t)(((piece0 + h) ^ (lane & 7)) << 4));
                    const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if constexpr (sizeof(T) == 4) {
                            r[j] = __uint_as_float(uw[j]);
                        } else {
                            const float2 q = unpack2<T>(uw[j]);
                            r[2 * j] = q.x;
                            r[2 * j + 1] = q.y;
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        const int n = n0 + c + h * E + j;
                        r[j] = t < a.M && n < a.N ? to_float(static_cast<const T *>(a.res)[(long long)t * a.ld_res + n]) : 0.f;
                    }
                }
#pragma unroll
                for (int j = 0; j < E; ++j)
                    v[h * E + j] = __float_as_uint(__fadd_rn(r[j], __fmul_rn(a.res_scale, __uint_as_float(v[h * E + j]))));
            }
        }
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
            const uint32_t at = rowaddr + (uint32_t)(((piece0 + h) ^ (lane & 7)) << 4);
            if constexpr (sizeof(T) == 4) {
                st_shared16(at, v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
            } else {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    w[j] = pack2<T>(__uint_as_float(v[8 * h + 2 * j]), __uint_as_float(v[8 * h + 2 * j + 1]));
                st_shared16(at, w[0], w[1], w[2], w[3]);
            }
        }
        if (i % PER == PER - 1) {
            if (p.tma_store) {
                fence_async_shared();
                __syncwarp();
                if (lane == 0) {
                    if (nb < a.N && row0 < a.M) tma_store_2d(ymap, stg, nb, row0);
                    bulk_commit_group();
                }
            } else {
                __syncwarp();
                int8_store_rows<T>(a, stg, row0, nb);
                __syncwarp();
            }
            ++box;
        }
    }
}

// Split tiles: this warp's 32 rows of every rank's channels to their owners' receive space, [source][128 rows][cw].
KEA_DEVI void int8_send_sums(uint32_t taddr, uint32_t recv, int cw, int splits, uint32_t rank, int quad) {
    const int row = quad * 32 + (int)(threadIdx.x & 31);
#pragma unroll 1
    for (int c = 0; c < 64; c += 8) {
        uint32_t v[8];
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                     : "r"(taddr + (uint32_t)c)
                     : "memory");
        tmem_wait_ld();
        asm volatile("" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]) : : "memory");
        const int owner = c / cw;
        const uint32_t at = map_to_rank(recv + (uint32_t)(((int)rank * 128 + row) * cw + c - owner * cw) * 4u, (uint32_t)owner);
        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + 16u), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
    }
}

// The slices' sums of this CTA's cw channels, added and finished: eight channels of a row per lane at a time.
template <typename T, bool SILU>
KEA_DEVI void int8_finish_split(const Int8TileArgs &p, uint32_t recv, uint32_t consts, int cw, uint32_t rank, int quad, int m0, int n0,
                                uint64_t sq) {
    const Int8Args &a = p.a;
    const int row = quad * 32 + (int)(threadIdx.x & 31), m = m0 + row;
    if (m >= a.M) return;
#pragma unroll 1
    for (int c = 0; c < cw; c += 8) {
        const int col = (int)rank * cw + c, n = n0 + col;   // in the tile, in the output
        if (n >= a.N) break;
        int v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int s = 0; s < p.splits; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 u = ld_shared16(recv + (uint32_t)((s * 128 + row) * cw + c + 4 * h) * 4u);
                v[4 * h] += (int)u.x;
                v[4 * h + 1] += (int)u.y;
                v[4 * h + 2] += (int)u.z;
                v[4 * h + 3] += (int)u.w;
            }
        float f[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const ulonglong2 al = ld_shared_pairs(consts + (uint32_t)(col + 4 * h) * 4u);
            const ulonglong2 bi = ld_shared_pairs(consts + (uint32_t)(64 + col + 4 * h) * 4u);
            unpair(int8_values<SILU>(v[4 * h], v[4 * h + 1], sq, al.x, bi.x), f[4 * h], f[4 * h + 1]);
            unpair(int8_values<SILU>(v[4 * h + 2], v[4 * h + 3], sq, al.y, bi.y), f[4 * h + 2], f[4 * h + 3]);
        }
        const bool whole = n + 8 <= a.N;
        if (a.res) {
            const T *r = static_cast<const T *>(a.res) + (long long)m * a.ld_res + n;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (n + j < a.N) f[j] = __fadd_rn(to_float(r[j]), __fmul_rn(a.res_scale, f[j]));
        }
        if (a.acc) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (n + j < a.N) a.acc[(long long)m * a.ld_acc + n + j] = v[j];
        }
        T *y = static_cast<T *>(a.y) + (long long)m * a.ldy + n;
        if (whole && p.tma_store) {   // rows 16-byte aligned
            if constexpr (sizeof(T) == 4) {
                reinterpret_cast<float4 *>(y)[0] = make_float4(f[0], f[1], f[2], f[3]);
                reinterpret_cast<float4 *>(y)[1] = make_float4(f[4], f[5], f[6], f[7]);
            } else {
                *reinterpret_cast<uint4 *>(y) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (n + j < a.N) y[j] = from_float<T>(f[j]);
        }
    }
}

template <typename T, bool SILU, bool EXTRA, int CTAS, int BN, bool SPLIT = false>
__global__ void __launch_bounds__(Int8Tile<CTAS, BN>::THREADS, 1)
int8_gemm_tile_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap wmap,
                      const __grid_constant__ CUtensorMap ymap, const Int8TileArgs p) {
    static_assert(!SPLIT || (CTAS == 1 && BN == 64), "split tiles are single CTAs' of 64 channels");
    using Tile = Int8Tile<CTAS, BN>;
    extern __shared__ uint8_t dyn_smem[];
    __shared__ __align__(8) uint64_t bar_full[kI8MaxStages];    // (pairs: in the even CTA) both operands of a stage landed
    __shared__ __align__(8) uint64_t bar_empty[kI8MaxStages];   // the MMAs are done with the stage
    __shared__ __align__(8) uint64_t bar_acc_full[2];           // accumulator complete
    __shared__ __align__(8) uint64_t bar_acc_empty[2];          // (pairs: in the even CTA) accumulator read by every epilogue warp
    __shared__ __align__(8) uint64_t bar_drain;
    __shared__ uint32_t tmem_slot;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a pair's CTA, or the slice of K a split tile's CTA takes
    const uint32_t rank = CTAS == 2 ? cluster_ctarank() : 0u, slice = SPLIT ? cluster_ctarank() : 0u;
    const int worker = (int)blockIdx.x / (SPLIT ? p.splits : CTAS), workers = (int)gridDim.x / (SPLIT ? p.splits : CTAS);
    const int kb0 = SPLIT ? (int)slice * p.per_split : 0, kb1 = SPLIT ? min(p.kbs, kb0 + p.per_split) : p.kbs;
    const uint32_t base = (smem_u32(dyn_smem) + 1023u) & ~1023u;
    const int S = p.stages;
    const uint32_t A0 = base, B0 = base + (uint32_t)S * kI8Half;
    const uint32_t STG0 = B0 + (uint32_t)S * Tile::B_BYTES, CONST0 = STG0 + Tile::STAGING;
    constexpr uint32_t kCols = 2u * BN;   // two accumulators

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&bar_acc_full[b]), 1);
            mbar_init(smem_u32(&bar_acc_empty[b]), CTAS * Tile::EPI_WARPS);
        }
        mbar_init(smem_u32(&bar_drain), 1);
        fence_barrier_init();
        prefetch_tensormap(&qmap);
        prefetch_tensormap(&wmap);
        prefetch_tensormap(&ymap);
    }
    if (warp == 1) {
        if constexpr (CTAS == 2) {
            tmem_alloc_pair(smem_u32(&tmem_slot), kCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(&tmem_slot), kCols);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    if constexpr (CTAS == 2 || SPLIT) cluster_sync_all();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    grid_dependency_wait();

    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            int s = 0, issued = 0;
            uint32_t ph = 0;
            for (int tile = worker; tile < p.tiles && ok; tile += workers) {
                const int mt = tile / p.n_tiles, nt = tile - mt * p.n_tiles;
                const int t0 = mt * 128 * CTAS + (int)rank * 128, n0 = nt * BN + (int)rank * (BN / CTAS);
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (issued >= S && !mbar_wait(smem_u32(&bar_empty[s]), ph ^ 1u, kOpWaitBudget)) {
                        ok = false;
                        break;
                    }
                    const uint32_t as = A0 + (uint32_t)s * kI8Half, bs = B0 + (uint32_t)s * Tile::B_BYTES;
                    const uint32_t full = smem_u32(&bar_full[s]);
                    if constexpr (CTAS == 2) {
                        const uint32_t even = map_to_rank(full, 0u);
                        if (rank == 0) mbar_arrive_expect_tx(full, 2u * Tile::STAGE);   // the bytes of both CTAs
                        tma_load_2d_pair(as, &qmap, even, kb * kI8K, t0);
                        tma_load_2d_pair(bs, &wmap, even, kb * kI8K, n0);
                    } else {
                        mbar_arrive_expect_tx(full, Tile::STAGE);
                        tma_load_2d(as, &qmap, full, kb * kI8K, t0);
                        tma_load_2d(bs, &wmap, full, kb * kI8K, n0);
                    }
                    if (issued < S) ++issued;
                    if (++s == S) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            // on failure the copies still in flight were issued before a wait that has lasted its whole bound (about 2 s)
            if (!ok) report_error(p.a.err, KEA_DEVERR_TIMEOUT);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = idesc_i8(128u * CTAS, (uint32_t)BN);
            const uint64_t ad0 = sw128_kmajor_desc(A0), bd0 = sw128_kmajor_desc(B0);
            int j = 0, s = 0;
            uint32_t ph = 0;
            for (int tile = worker; tile < p.tiles; tile += workers, ++j) {
                const int buf = j & 1;
                const uint32_t use = (uint32_t)(j >> 1);
                if (j >= 2) {
                    const bool drained = CTAS == 2 ? mbar_wait_cluster(smem_u32(&bar_acc_empty[buf]), (use & 1u) ^ 1u, kOpWaitBudget)
                                                   : mbar_wait(smem_u32(&bar_acc_empty[buf]), (use & 1u) ^ 1u, kOpWaitBudget);
                    if (!__all_sync(0xFFFFFFFFu, drained)) {
                        ok = false;
                        break;
                    }
                }
                tc_fence_after();
                const uint32_t dcol = tmem + (uint32_t)buf * BN;
                for (int kb = kb0; kb < kb1; ++kb) {
                    const bool ready = CTAS == 2 ? mbar_wait_cluster(smem_u32(&bar_full[s]), ph, kOpWaitBudget)
                                                 : mbar_wait(smem_u32(&bar_full[s]), ph, kOpWaitBudget);
                    if (!__all_sync(0xFFFFFFFFu, ready)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t ad = ad0 + (uint64_t)(((uint32_t)s * kI8Half) >> 4);
                    const uint64_t bd = bd0 + (uint64_t)(((uint32_t)s * Tile::B_BYTES) >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < kI8K / 32; ++kk) {   // K = 32 per MMA: + 32 bytes = 2 descriptor units
                            const uint32_t more = (kb > kb0 || kk > 0) ? 1u : 0u;
                            if constexpr (CTAS == 2) mma_i8_pair(dcol, ad + (uint64_t)(2 * kk), bd + (uint64_t)(2 * kk), idesc, more);
                            else mma_i8(dcol, ad + (uint64_t)(2 * kk), bd + (uint64_t)(2 * kk), idesc, more);
                        }
                        if constexpr (CTAS == 2) mma_commit_pair(smem_u32(&bar_empty[s]), (uint16_t)3);
                        else mma_commit(smem_u32(&bar_empty[s]));
                    }
                    __syncwarp();
                    if (++s == S) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                if (!ok) break;
                if (elect_one()) {
                    if constexpr (CTAS == 2) mma_commit_pair(smem_u32(&bar_acc_full[buf]), (uint16_t)3);
                    else mma_commit(smem_u32(&bar_acc_full[buf]));
                }
                __syncwarp();
            }
            if (!ok && lane == 0) report_error(p.a.err, KEA_DEVERR_TIMEOUT);
            // every MMA this warp issued completes before shared and tensor memory are given up
            if (elect_one()) {
                if constexpr (CTAS == 2) mma_commit_pair(smem_u32(&bar_drain), (uint16_t)1);
                else mma_commit(smem_u32(&bar_drain));
            }
            __syncwarp();
            mbar_wait(smem_u32(&bar_drain), 0u, kOpWaitBudget);
            __syncwarp();
        }
    } else if constexpr (SPLIT) {   // one tile per cluster
        const int ew = warp - 2, quad = warp & 3, n0 = worker % p.n_tiles * BN;
        const uint32_t consts = CONST0 + (uint32_t)(ew * Tile::CW) * 8u;
#pragma unroll
        for (int i = 0; i < Tile::CW; i += 32) {
            const int n = n0 + i + lane;
            const float al = n < p.a.N ? __ldg(p.a.alpha + n) : 0.f;
            const float bi = p.a.bias && n < p.a.N ? __ldg(p.a.bias + n) : kI8NoBias;
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(consts + (uint32_t)(i + lane) * 4u), "f"(al) : "memory");
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(consts + (uint32_t)(Tile::CW + i + lane) * 4u), "f"(bi) : "memory");
        }
        __syncwarp();
        const bool done = mbar_wait_sleep(smem_u32(&bar_acc_full[0]), 0u, kOpWaitBudget, 64);
        if (__all_sync(0xFFFFFFFFu, done)) {
            tc_fence_after();
            int8_send_sums(tmem + ((uint32_t)(quad * 32) << 16), STG0, BN / p.splits, p.splits, slice, quad);
        } else if (lane == 0) {
            report_error(p.a.err, KEA_DEVERR_TIMEOUT);
        }
    } else {
        const int ew = warp - 2, quad = warp & 3, part = ew >> 2;
        const uint32_t stg = STG0 + (uint32_t)(ew * Tile::BUFS) * kI8Box;
        const uint32_t consts = CONST0 + (uint32_t)(ew * Tile::CW) * 8u;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(part * Tile::CW);
        int j = 0, box = 0;
        for (int tile = worker; tile < p.tiles; tile += workers, ++j) {
            const int buf = j & 1;
            const int mt = tile / p.n_tiles, nt = tile - mt * p.n_tiles;
            const int row0 = mt * 128 * CTAS + (int)rank * 128 + quad * 32, n0 = nt * BN + part * Tile::CW;
#pragma unroll
            for (int i = 0; i < Tile::CW; i += 32) {   // this warp's channel constants, while the accumulator fills
                const int n = n0 + i + lane;
                const float al = n < p.a.N ? __ldg(p.a.alpha + n) : 0.f;
                const float bi = p.a.bias && n < p.a.N ? __ldg(p.a.bias + n) : kI8NoBias;
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(consts + (uint32_t)(i + lane) * 4u), "f"(al) : "memory");
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(consts + (uint32_t)(Tile::CW + i + lane) * 4u), "f"(bi) : "memory");
            }
            const float s = row0 + lane < p.a.M ? p.a.qs[row0 + lane] : 0.f;
            const uint64_t sq = pair_of(s, s);
            uint4 ahead[8];
            if (p.a.res && p.res_vec) int8_load_residual<T>(p.a, ahead, row0, n0);
            __syncwarp();
            const bool done = mbar_wait_sleep(smem_u32(&bar_acc_full[buf]), (uint32_t)((j >> 1) & 1), kOpWaitBudget, 64);
            if (!__all_sync(0xFFFFFFFFu, done)) {
                if (lane == 0) report_error(p.a.err, KEA_DEVERR_TIMEOUT);
                break;
            }
            tc_fence_after();
            const uint32_t acc_empty = smem_u32(&bar_acc_empty[buf]);
            int8_epilogue_tile<T, SILU, EXTRA, Tile::CW, Tile::BUFS>(p, &ymap, lanes + (uint32_t)(buf * BN), stg, consts, row0, n0, sq,
                                                              box, ahead, [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CTAS == 2) mbar_arrive_cluster(map_to_rank(acc_empty, 0u));
                    else mbar_arrive(acc_empty);
                }
            });
        }
        if (lane == 0) bulk_wait_group_read0();   // the staging space outlives the stores' reads of it
        __syncwarp();
    }

    grid_launch_dependents();
    tc_fence_before();
    if constexpr (CTAS == 2 || SPLIT) cluster_sync_relaxed_paths();
    else __syncthreads();
    if constexpr (SPLIT) {
        if (warp >= 2) {   // every slice's sums have arrived
            const int ew = warp - 2, quad = warp & 3, mt = worker / p.n_tiles, m0 = mt * 128, n0 = (worker - mt * p.n_tiles) * BN;   // the cluster's tile
            const int m = m0 + quad * 32 + lane;
            const float s = m < p.a.M ? p.a.qs[m] : 0.f;
            int8_finish_split<T, SILU>(p, STG0, CONST0 + (uint32_t)(ew * Tile::CW) * 8u, BN / p.splits, slice, quad, m0, n0, pair_of(s, s));
        }
    }
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CTAS == 2) tmem_dealloc_pair(tmem, kCols);
        else tmem_dealloc(tmem, kCols);
    }
}

}  // namespace kea
