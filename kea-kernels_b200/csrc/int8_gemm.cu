// int8_gemm.cu - host side of the 8-bit linear map (kea_lowbit_int8_gemm): argument checks, the choice of kernel and the
// launches.
#include <algorithm>

#include "host.h"
#include "int8_reg_kernel.cuh"
#include "int8_tile_kernel.cuh"
#include "kea_lowbit.h"

namespace {

using kea_host::aligned;
using kea_host::ceil_div;

constexpr int kMaxK = 131071;   // 128 * 128 * k < 2^31
constexpr int kMaxDynSmem = 227 * 1024 - 1024;   // the kernels' static shared memory is a few hundred bytes

int validate(const KeaInt8Desc *d) {
    if (!d || d->m < 0 || d->n < 1 || d->k < 1 || d->y_type < KEA_TYPE_F32 || d->y_type > KEA_TYPE_BF16 ||
        (d->flags & ~(KEA_INT8_SILU | KEA_INT8_PDL)) || d->kernel < 0 || d->kernel > KEA_INT8_KERNEL_SPLIT)
        return KEA_ERR_INVALID_VALUE;
    if (d->m == 0) return KEA_OK;
    if (!d->q || !d->qs || !d->w || !d->alpha || !d->y || d->ldq < d->k || d->ldw < d->k || d->ldy < d->n)
        return KEA_ERR_INVALID_VALUE;
    if ((d->residual && d->ld_residual < d->n) || (d->acc && d->ld_acc < d->n)) return KEA_ERR_INVALID_VALUE;
    if (d->k > kMaxK) return KEA_ERR_UNSUPPORTED;
    if (!aligned(d->q, 16) || !aligned(d->w, 16) || d->ldq % 16 || d->ldw % 16) return KEA_ERR_ALIGNMENT;
    const size_t size = d->y_type == KEA_TYPE_F32 ? 4 : 2;
    if (!aligned(d->y, size) || (d->residual && !aligned(d->residual, size)) || (d->acc && !aligned(d->acc, 4)) ||
        !aligned(d->qs, 4) || !aligned(d->alpha, 4) || (d->bias && !aligned(d->bias, 4)))
        return KEA_ERR_ALIGNMENT;
    return KEA_OK;
}

kea::Int8Args arguments(const KeaInt8Desc *d, const kea_host::Device &dev) {
    kea::Int8Args a{};
    a.q = d->q;
    a.ldq = d->ldq;
    a.qs = d->qs;
    a.w = d->w;
    a.ldw = d->ldw;
    a.alpha = d->alpha;
    a.bias = d->bias;
    a.y = d->y;
    a.ldy = d->ldy;
    a.res = d->residual;
    a.ld_res = d->ld_residual;
    a.acc = d->acc;
    a.ld_acc = d->ld_acc;
    a.res_scale = d->residual_scale;
    a.M = d->m;
    a.N = d->n;
    a.K = d->k;
    a.y_type = d->y_type;
    a.silu = (d->flags & KEA_INT8_SILU) ? 1 : 0;
    a.err = d->error_word ? d->error_word : dev.error_word;
    return a;
}

struct Launch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attrs[2];
    Launch(dim3 grid, int threads, size_t smem, void *stream, bool pdl, int cluster = 1) {
        cfg.gridDim = grid;
        cfg.blockDim = dim3((unsigned)threads, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = (cudaStream_t)stream;
        cfg.attrs = attrs;
        if (cluster > 1) {
            attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
            attrs[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
            attrs[cfg.numAttrs].val.clusterDim.y = 1;
            attrs[cfg.numAttrs].val.clusterDim.z = 1;
            ++cfg.numAttrs;
        }
        if (pdl) {
            attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attrs[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
            ++cfg.numAttrs;
        }
    }
};

// ---- register-operand kernel ---------------------------------------------------------------------------------------
template <typename T, int RG, int D>
cudaError_t launch_reg_as(const kea::Int8Args &a, int sms, bool pdl, void *stream) {
    // eight channels per CTA as long as sixteen do not give every SM one
    const bool half = ceil_div(a.N, 16) * ceil_div(a.M, 8 * RG) < sms;
    const Launch l(dim3((unsigned)ceil_div(a.N, half ? 8 : 16), (unsigned)ceil_div(a.M, 8 * RG), 1), kea::kI8RegThreads, 0, stream, pdl);
    return half ? cudaLaunchKernelEx(&l.cfg, kea::int8_gemm_reg_kernel<T, RG, D, true>, a)
                : cudaLaunchKernelEx(&l.cfg, kea::int8_gemm_reg_kernel<T, RG, D, false>, a);
}

template <typename T>
cudaError_t launch_reg(const kea::Int8Args &a, int sms, bool pdl, void *stream) {
    return a.M <= 8    ? launch_reg_as<T, 1, 8>(a, sms, pdl, stream)
           : a.M <= 16 ? launch_reg_as<T, 2, 6>(a, sms, pdl, stream) : launch_reg_as<T, 4, 4>(a, sms, pdl, stream);
}

// ---- tcgen05 kernels -----------------------------------------------------------------------------------------------
// Row-major matrix of 8-bit codes -> boxes of 128 bytes of K x `rows` rows, 128-byte swizzle; zeros outside.
bool map_codes(const kea_host::Device &dev, CUtensorMap *map, const int8_t *p, long long ld, int rows_total, int k, int rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows_total};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {(cuuint32_t)kea::kI8K, (cuuint32_t)rows}, step[2] = {1, 1};
    return dev.encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(p), dims, strides, box, step,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The output as boxes of 32 rows x 128 bytes, where its rows are 16-byte aligned.
bool map_output(const kea_host::Device &dev, CUtensorMap *map, const kea::Int8Args &a) {
    const int size = a.y_type == KEA_TYPE_F32 ? 4 : 2;
    if (!aligned(a.y, 16) || (a.ldy * size) % 16) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)a.N, (cuuint64_t)a.M};
    const cuuint64_t strides[1] = {(cuuint64_t)(a.ldy * size)};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / size), 32}, step[2] = {1, 1};
    const CUtensorMapDataType type = a.y_type == KEA_TYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : a.y_type == KEA_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return dev.encode(map, type, 2, a.y, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int CTAS, int BN>
int stages_for(int kbs, int tiles_per_worker) {
    int s = kea::kI8MaxStages;
    while (s > 2 && kea::Int8Tile<CTAS, BN>::smem(s) > kMaxDynSmem) --s;
    return std::max(2, std::min<int>(s, kbs * tiles_per_worker));
}

template <typename T, bool SILU, int CTAS, int BN>
cudaError_t launch_tile_as(const kea_host::Device &dev, const kea::Int8Args &a, bool pdl, void *stream) {
    using Tile = kea::Int8Tile<CTAS, BN>;
    kea::Int8TileArgs p{};
    p.a = a;
    p.n_tiles = ceil_div(a.N, BN);
    const long long tiles = (long long)p.n_tiles * ceil_div(a.M, 128 * CTAS);
    if (tiles >= (1LL << 30)) return cudaErrorInvalidValue;
    p.tiles = (int)tiles;
    p.kbs = ceil_div(a.K, kea::kI8K);
    const int workers = std::min(p.tiles, std::max(1, dev.sms / CTAS));
    p.stages = stages_for<CTAS, BN>(p.kbs, ceil_div(p.tiles, workers));
    CUtensorMap qmap, wmap, ymap{};
    if (!map_codes(dev, &qmap, a.q, a.ldq, a.M, a.K, 128) || !map_codes(dev, &wmap, a.w, a.ldw, a.N, a.K, BN / CTAS))
        return cudaErrorInvalidValue;
    const size_t size = sizeof(T);
    p.tma_store = map_output(dev, &ymap, a) ? 1 : 0;
    p.res_vec = a.res && aligned(a.res, 16) && (a.ld_res * (long long)size) % 16 == 0 && ((size_t)a.N * size) % 16 == 0;
    const Launch l(dim3((unsigned)(workers * CTAS), 1, 1), Tile::THREADS, Tile::smem(p.stages), stream, pdl, CTAS);
    if (a.acc || (a.res && !p.res_vec))
        return cudaLaunchKernelEx(&l.cfg, kea::int8_gemm_tile_kernel<T, SILU, true, CTAS, BN>, qmap, wmap, ymap, p);
    return cudaLaunchKernelEx(&l.cfg, kea::int8_gemm_tile_kernel<T, SILU, false, CTAS, BN>, qmap, wmap, ymap, p);
}

// How many CTAs share a 128 x 64 tile: as many as find an SM of their own, each with two blocks of K at least.
int tile_splits(int m, int n, int k, int sms) {
    const long long tiles = (long long)ceil_div(m, 128) * ceil_div(n, 64);
    const int kbs = ceil_div(k, kea::kI8K);
    int s = 1;
    while (s < 8 && 2 * s * tiles <= sms && 4 * s <= kbs) s *= 2;
    return ceil_div(kbs, ceil_div(kbs, s)) == s ? s : 1;   // (a power of two) no slice without work
}

template <typename T, bool SILU>
cudaError_t launch_split(const kea_host::Device &dev, const kea::Int8Args &a, int splits, bool pdl, void *stream) {
    using Tile = kea::Int8Tile<1, 64>;
    kea::Int8TileArgs p{};
    p.a = a;
    p.n_tiles = ceil_div(a.N, 64);
    p.tiles = p.n_tiles * ceil_div(a.M, 128);
    p.kbs = ceil_div(a.K, kea::kI8K);
    p.splits = splits;
    p.per_split = ceil_div(p.kbs, splits);
    // three stages at most: two CTAs per SM, so that 16 clusters of 8 run at once (one per SM leaves room for 15: a second
    // wave, 13.4 instead of 10.3 us at 128 x 1024 x 4096)
    p.stages = std::min(3, stages_for<1, 64>(p.per_split, 1));
    CUtensorMap qmap, wmap, ymap{};
    if (!map_codes(dev, &qmap, a.q, a.ldq, a.M, a.K, 128) || !map_codes(dev, &wmap, a.w, a.ldw, a.N, a.K, 64)) return cudaErrorInvalidValue;
    p.tma_store = aligned(a.y, 16) && (a.ldy * (long long)sizeof(T)) % 16 == 0;   // here: rows take 16-byte stores
    const Launch l(dim3((unsigned)(p.tiles * splits), 1, 1), Tile::THREADS, Tile::smem(p.stages), stream, pdl, splits);
    return cudaLaunchKernelEx(&l.cfg, kea::int8_gemm_tile_kernel<T, SILU, false, 1, 64, true>, qmap, wmap, ymap, p);
}

template <typename T>
cudaError_t launch_typed(const kea_host::Device &dev, const kea::Int8Args &a, int kernel, bool pdl, void *stream) {
    switch (kernel) {
        case KEA_INT8_KERNEL_SPLIT: {
            const int splits = tile_splits(a.M, a.N, a.K, dev.sms);
            if (splits > 1) return a.silu ? launch_split<T, true>(dev, a, splits, pdl, stream) : launch_split<T, false>(dev, a, splits, pdl, stream);
            [[fallthrough]];   // nothing to split: the same tiles, one CTA each
        }
        case KEA_INT8_KERNEL_TILE64:
            return a.silu ? launch_tile_as<T, true, 1, 64>(dev, a, pdl, stream) : launch_tile_as<T, false, 1, 64>(dev, a, pdl, stream);
        case KEA_INT8_KERNEL_TILE128:
            return a.silu ? launch_tile_as<T, true, 1, 128>(dev, a, pdl, stream) : launch_tile_as<T, false, 1, 128>(dev, a, pdl, stream);
        case KEA_INT8_KERNEL_PAIR:
            return a.silu ? launch_tile_as<T, true, 2, 256>(dev, a, pdl, stream) : launch_tile_as<T, false, 2, 256>(dev, a, pdl, stream);
        default: return launch_reg<T>(a, dev.sms, pdl, stream);
    }
}

// Which kernel, by the microseconds each is expected to take. A launch of the tile kernels lasts as long as its waves of
// tiles: a fixed part, then per wave a part that grows with K (a CTA's MMAs are issue-paced, about 100 clocks per 32
// columns of K). Fitted to launches back to back on a B200, measured / expected at M x N x K, us:
//   register operands  32 x 4096 x 1024  4.4 / 4.4   128 x 1024 x 4096 11.1 / 11.6   512 x 640 x 640   9.3 / 9.8
//   128 x 64 tiles    128 x 2048 x 256   4.1 / 3.9  1024 x 1024 x 1024  6.2 / 5.7   1024 x 4096 x 1024 14.2 / 14.1
//   split tiles       128 x 1024 x 4096 10.3 / 10.1  256 x 1024 x 4096  9.1 / 10.1   512 x 1024 x 4096 12.6 / 12.0
//   128 x 128 tiles   512 x 4096 x 1024  7.5 / 6.3  1024 x 4096 x 1024 10.7 / 9.5   1024 x 4096 x 4096 25.0 / 23.4
//   pairs            1024 x 4096 x 1024 10.1 / 8.6  2048 x 4096 x 1024 13.3 / 11.9  1024 x 4096 x 4096 18.0 / 16.4
// Over 40 random shapes the chosen kernel takes 1.045 times the best one's time in geometric mean. It is off most for 70 to 540
// tokens with K below 700, where the register form is expected too early: 209 x 714 x 427 9.4 us (5.8 with 128 x 64 tiles).
int choose(const kea::Int8Args &a, int sms) {
    const auto tiles = [&](int rows, int cols) { return (long long)ceil_div(a.M, rows) * ceil_div(a.N, cols); };
    const double k = a.K;
    const size_t size = a.y_type == KEA_TYPE_F32 ? 4 : 2;
    // rows that TMA cannot store, or a skip connection it cannot be read beside, go out value by value
    const double odd = !aligned(a.y, 16) || (a.ldy * size) % 16 || (a.res && ((a.ld_res * size) % 16 || (a.N * size) % 16)) ? 2.0 : 0.0;
    const auto waves = [&](long long n, int at_once) { return (double)((n + at_once - 1) / at_once); };
    int best = KEA_INT8_KERNEL_TILE64;
    double least = 3.3 + 0.00235 * k + odd + (waves(tiles(128, 64), sms) - 1) * (0.6 + 0.00215 * k);
    const auto offer = [&](int kernel, double us) {
        if (us < least) {
            least = us;
            best = kernel;
        }
    };
    if (a.M <= 4096)
        offer(KEA_INT8_KERNEL_REG, std::max(2.9, 0.8 + 0.0047 * (double)tiles(a.M <= 16 ? 8 : 32, 16) * (a.M <= 16 ? 0.5 : 1.0) *
                                                           (ceil_div(a.K, 512) + 1)));
    const int s = tile_splits(a.M, a.N, a.K, sms);
    if (s > 1) offer(KEA_INT8_KERNEL_SPLIT, 6.4 + 0.00245 * k / s + 0.3 * s);
    offer(KEA_INT8_KERNEL_TILE128, 3.9 + 0.00235 * k + odd + (waves(tiles(128, 128), sms) - 1) * (0.9 + 0.0022 * k));
    offer(KEA_INT8_KERNEL_PAIR, 6.0 + 0.00255 * k + odd + (waves(tiles(256, 256), sms / 2) - 1) * (1.05 + 0.0022 * k));
    return best;
}

template <typename T, bool SILU, bool EXTRA>
bool attributes() {
    const auto set = [](const void *kernel) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynSmem) == cudaSuccess;
    };
    return set((const void *)kea::int8_gemm_tile_kernel<T, SILU, EXTRA, 1, 64>) &&
           set((const void *)kea::int8_gemm_tile_kernel<T, SILU, EXTRA, 1, 128>) &&
           set((const void *)kea::int8_gemm_tile_kernel<T, SILU, EXTRA, 2, 256>) &&
           (EXTRA || set((const void *)kea::int8_gemm_tile_kernel<T, SILU, false, 1, 64, true>));
}
template <typename T>
bool attributes() {
    return attributes<T, false, false>() && attributes<T, false, true>() && attributes<T, true, false>() && attributes<T, true, true>();
}

}  // namespace

int kea_host::setup_int8_gemm() {
    return attributes<float>() && attributes<__half>() && attributes<__nv_bfloat16>() ? KEA_OK : KEA_ERR_CUDA;
}

extern "C" int kea_lowbit_int8_gemm(const KeaInt8Desc *d, void *stream) {
    const int v = validate(d);
    if (v != KEA_OK || d->m == 0) return v;
    kea_host::Device dev;
    const int st = kea_host::device(&dev, stream);
    if (st != KEA_OK) return st;
    const kea::Int8Args a = arguments(d, dev);
    const bool pdl = (d->flags & KEA_INT8_PDL) != 0;
    const int kernel = d->kernel ? d->kernel : choose(a, dev.sms);
    if (kernel == KEA_INT8_KERNEL_REG && ceil_div(a.M, 32) > 65535) return KEA_ERR_UNSUPPORTED;
    const cudaError_t e = a.y_type == KEA_TYPE_F32   ? launch_typed<float>(dev, a, kernel, pdl, stream)
                          : a.y_type == KEA_TYPE_F16 ? launch_typed<__half>(dev, a, kernel, pdl, stream)
                                                     : launch_typed<__nv_bfloat16>(dev, a, kernel, pdl, stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return KEA_ERR_CUDA;
    }
    return KEA_OK;
}
