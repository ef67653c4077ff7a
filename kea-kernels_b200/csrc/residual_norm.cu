// residual_norm.cu - host side of the gated norm step between two blocks (kea_lowbit_residual_norm).
#include <algorithm>
#include <atomic>

#include "host.h"
#include "kea_lowbit.h"
#include "residual_norm_kernel.cuh"

namespace {

using kea_host::aligned;
using kea_host::ceil_div;

constexpr int kMaxWidth = kea::kRnMaxThreads * 32;

size_t type_size(int type) { return type == KEA_TYPE_F32 ? 4 : 2; }
bool type_ok(int type) { return type >= KEA_TYPE_F32 && type <= KEA_TYPE_BF16; }
bool norm_ok(int kind, const float *w) {
    return kind == KEA_NORM_NONE || ((kind == KEA_NORM_LAYER || kind == KEA_NORM_RMS) && w);
}

int validate(const KeaResidualNormDesc *d) {
    if (!d || d->m < 0 || d->d < 1 || !type_ok(d->x_type) || !type_ok(d->y_type) || !type_ok(d->h_type) ||
        !norm_ok(d->post, d->post_weight) || !norm_ok(d->pre, d->pre_weight) || d->frames < 1 ||
        (d->gate_act != KEA_GATE_NONE && d->gate_act != KEA_GATE_SIGMOID) || (d->flags & ~KEA_RNORM_PDL))
        return KEA_ERR_INVALID_VALUE;
    if (d->m == 0) return KEA_OK;
    if (!d->x || !d->y || !d->r || (!d->h && !d->q) || (d->q && !d->qs)) return KEA_ERR_INVALID_VALUE;
    if (d->ldx < d->d || d->ldy < d->d || d->ldr < d->d || (d->h && d->ldh < d->d) || (d->q && d->ldq < d->d))
        return KEA_ERR_INVALID_VALUE;
    if (d->d > kMaxWidth) return KEA_ERR_UNSUPPORTED;
    if (!aligned(d->x, type_size(d->x_type)) || !aligned(d->r, type_size(d->x_type)) ||
        !aligned(d->y, type_size(d->y_type)) || (d->gate && !aligned(d->gate, type_size(d->y_type))) ||
        (d->h && !aligned(d->h, type_size(d->h_type))) || (d->qs && !aligned(d->qs, 4)))
        return KEA_ERR_ALIGNMENT;
    return KEA_OK;
}

// Rows and parameters in whole chunks of eight values: 32-byte FP32 or 16-byte loads and stores.
bool whole(const void *p, int64_t ld, int type) { return !p || (aligned(p, 8 * type_size(type)) && ld % 8 == 0); }
bool vectors(const KeaResidualNormDesc *d) {
    return d->d % 8 == 0 && whole(d->x, d->ldx, d->x_type) && whole(d->r, d->ldr, d->x_type) &&
           whole(d->y, d->ldy, d->y_type) && whole(d->h, d->ldh, d->h_type) && whole(d->gate, d->gate_clip_stride, d->y_type) &&
           whole(d->gate, d->gate_row_stride, d->y_type) && whole(d->post_weight, 0, KEA_TYPE_F32) &&
           whole(d->post_bias, 0, KEA_TYPE_F32) && whole(d->pre_weight, 0, KEA_TYPE_F32) &&
           whole(d->pre_bias, 0, KEA_TYPE_F32) && (!d->q || (aligned(d->q, 8) && d->ldq % 8 == 0));
}

int threads_for(int d, int vpt) {
    int t = 32;
    while (t * vpt < d) t *= 2;
    return t;
}

struct Launch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    Launch(int grid, int threads, size_t smem, bool pdl, void *stream) {
        cfg.gridDim = dim3((unsigned)grid, 1, 1);
        cfg.blockDim = dim3((unsigned)threads, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = (cudaStream_t)stream;
        cfg.attrs = attr;
        if (pdl) {
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[0].val.programmaticStreamSerializationAllowed = 1;
            cfg.numAttrs = 1;
        }
    }
};

constexpr int kFlatMaxSmem = 220 * 1024;

// ---- contiguous rows of any width ----------------------------------------------------------------------------------
struct FlatPlan {
    kea::FlatArgs p;
    int tpr, grid;
    size_t smem;
};

// Whether the rows are contiguous in aligned buffers, enough to give every SM's warps one, and their parameters fit.
bool plan_flat(const KeaResidualNormDesc *d, const kea::ResidualNormArgs &a, const kea_host::Device &dev, FlatPlan *f) {
    const bool gate_shared = d->gate && d->gate_row_stride == 0 && (d->gate_clip_stride == 0 || d->m <= d->frames);
    const auto contiguous = [&](const void *p, int64_t ld, int type) { return !p || (ld == d->d && aligned(p, 8 * type_size(type))); };
    if (!contiguous(d->x, d->ldx, d->x_type) || !contiguous(d->r, d->ldr, d->x_type) || !contiguous(d->y, d->ldy, d->y_type) ||
        !contiguous(d->h, d->ldh, d->h_type))
        return false;
    if (d->gate && !gate_shared && d->gate_row_stride == d->d && !aligned(d->gate, 8 * type_size(d->y_type))) return false;
    f->tpr = threads_for(d->d + 7, kea::kFlatVpt);   // a row may begin up to seven values into its first group
    const int groups = kea::kFlatThreads / std::max(f->tpr, 1);
    // narrower rows leave most of a warp's 128 groups empty (8000 rows of 100 values: 29 us against 14 us straight)
    if (d->d <= 512 || f->tpr > 128 || d->m < groups * dev.sms) return false;
    f->p.a = a;
    f->p.gate_end = 0;
    if (d->gate && d->gate_clip_stride >= 0 && d->gate_row_stride >= 0 && aligned(d->gate, 16))
        f->p.gate_end = (d->m - 1) / d->frames * d->gate_clip_stride + (d->m - 1) % d->frames * d->gate_row_stride + d->d;
    f->p.padded = f->tpr * kea::kFlatVpt + 16;
    const bool held[5] = {d->post != KEA_NORM_NONE, d->post != KEA_NORM_NONE && d->post_bias, d->pre != KEA_NORM_NONE,
                          d->pre != KEA_NORM_NONE && d->pre_bias, gate_shared};
    int n = 0;
    f->p.params = 0;
    for (int k = 0; k < 5; ++k)
        if (held[k]) {
            f->p.params |= 1 << k;
            ++n;
        }
    f->smem = (size_t)n * 4 * f->p.padded * sizeof(float);
    f->grid = dev.sms;
    return f->smem <= (size_t)kFlatMaxSmem;
}

template <typename TX, typename TY, int TPR>
cudaError_t launch_flat_as(const FlatPlan &f, int device, bool pdl, void *stream) {
    const auto kernel = kea::residual_norm_flat_kernel<TX, TY, TPR>;
    static std::atomic<uint64_t> ready{0};   // devices this kernel's shared memory limit is set on
    if (!(ready.load(std::memory_order_acquire) >> device & 1)) {
        const cudaError_t e = cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFlatMaxSmem);
        if (e != cudaSuccess) return e;
        ready.fetch_or(1ULL << device, std::memory_order_release);
    }
    const Launch l(f.grid, kea::kFlatThreads, f.smem, pdl, stream);
    return cudaLaunchKernelEx(&l.cfg, kernel, f.p);
}

template <typename TX, typename TY>
cudaError_t launch_flat(const FlatPlan &f, int device, bool pdl, void *stream) {
    return f.tpr == 32   ? launch_flat_as<TX, TY, 32>(f, device, pdl, stream)
           : f.tpr == 64 ? launch_flat_as<TX, TY, 64>(f, device, pdl, stream)
                         : launch_flat_as<TX, TY, 128>(f, device, pdl, stream);
}

// ---- rows straight from global memory ------------------------------------------------------------------------------
template <typename TX, typename TY>
cudaError_t launch_direct(const kea::ResidualNormArgs &a, const kea_host::Device &dev, bool vec, bool pdl, void *stream) {
    // One warp per row, up to 32 values per thread, as long as that gives every SM eight warps: no barriers, and the
    // loads of 16 rows are in flight on an SM (32000 rows of 1024 FP32 values: 83 us, against 129 and 128 us with two and
    // four warps per row). Value by value at most 16 per thread: more is straight-line code that misses the instruction
    // cache (8000 rows of 4095 values: 225-233 us, 464 with 32). Fewer rows: eight, the shortest chain of loads and sums.
    const int most = vec || threads_for(a.D, 16) > kea::kRnMaxThreads ? 32 : 16;
    const bool many = (long long)a.M * threads_for(a.D, most) >= 32LL * 8 * dev.sms;
    int vpt = most;
    while (vpt > 8 && (!many || threads_for(a.D, vpt / 2) == threads_for(a.D, vpt)) && threads_for(a.D, vpt / 2) <= kea::kRnMaxThreads)
        vpt /= 2;
    const int tpr = threads_for(a.D, vpt), threads = std::max(tpr, 128);
    if (vec && vpt == 32 && tpr * 24 >= a.D && threads == 128) vpt = 24;   // a quarter of the registers would be empty
    const Launch l(ceil_div(a.M, threads / tpr), threads, 0, pdl, stream);
#define KEA_RN(VPT, VEC, THREADS) cudaLaunchKernelEx(&l.cfg, kea::residual_norm_kernel<TX, TY, VPT, VEC, THREADS>, a, tpr)
    if (vec)
        return vpt == 8 ? KEA_RN(8, true, 512) : vpt == 16 ? (threads == 128 ? KEA_RN(16, true, 128) : KEA_RN(16, true, 512))
               : vpt == 24 ? KEA_RN(24, true, 128) : threads == 128 ? KEA_RN(32, true, 128) : KEA_RN(32, true, 512);
    return vpt == 8 ? KEA_RN(8, false, 512) : vpt == 16 ? KEA_RN(16, false, 512) : KEA_RN(32, false, 512);
#undef KEA_RN
}

template <typename TX, typename TY>
cudaError_t launch(const KeaResidualNormDesc *d, const kea::ResidualNormArgs &a, const kea_host::Device &dev, bool pdl, void *stream) {
    const bool vec = vectors(d);
    FlatPlan f{};
    if (!vec && plan_flat(d, a, dev, &f)) return launch_flat<TX, TY>(f, dev.index, pdl, stream);
    return launch_direct<TX, TY>(a, dev, vec, pdl, stream);
}

template <typename TX>
cudaError_t launch_for(const KeaResidualNormDesc *d, const kea::ResidualNormArgs &a, const kea_host::Device &dev, bool pdl, void *stream) {
    switch (d->y_type) {
        case KEA_TYPE_F32: return launch<TX, float>(d, a, dev, pdl, stream);
        case KEA_TYPE_F16: return launch<TX, __half>(d, a, dev, pdl, stream);
        default: return launch<TX, __nv_bfloat16>(d, a, dev, pdl, stream);
    }
}

}  // namespace

extern "C" int kea_lowbit_residual_norm(const KeaResidualNormDesc *d, void *stream) {
    const int v = validate(d);
    if (v != KEA_OK || d->m == 0) return v;
    kea_host::Device dev;
    const int st = kea_host::device(&dev, stream);
    if (st != KEA_OK) return st;
    kea::ResidualNormArgs a{};
    a.x = d->x;
    a.y = d->y;
    a.gate = d->gate;
    a.ldx = d->ldx;
    a.ldy = d->ldy;
    a.gate_clip = d->gate_clip_stride;
    a.gate_row = d->gate_row_stride;
    a.frames = d->frames;
    a.gate_act = d->gate_act;
    a.post = d->post;
    a.pre = d->pre;
    a.scale = d->scale;
    a.post_eps = d->post_eps;
    a.pre_eps = d->pre_eps;
    a.post_w = d->post_weight;
    a.post_b = d->post_bias;
    a.pre_w = d->pre_weight;
    a.pre_b = d->pre_bias;
    a.r = d->r;
    a.h = d->h;
    a.ldr = d->ldr;
    a.ldh = d->ldh;
    a.h_type = d->h_type;
    a.q = d->q;
    a.ldq = d->ldq;
    a.qs = d->qs;
    a.M = d->m;
    a.D = d->d;
    const bool pdl = (d->flags & KEA_RNORM_PDL) != 0;
    const cudaError_t e = d->x_type == KEA_TYPE_F32   ? launch_for<float>(d, a, dev, pdl, stream)
                          : d->x_type == KEA_TYPE_F16 ? launch_for<__half>(d, a, dev, pdl, stream)
                                                      : launch_for<__nv_bfloat16>(d, a, dev, pdl, stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return KEA_ERR_CUDA;
    }
    return KEA_OK;
}
