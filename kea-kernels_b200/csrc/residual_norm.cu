// residual_norm.cu - host side of the gated norm step between two blocks (kea_lowbit_residual_norm).
#include <algorithm>

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

template <typename TX, typename TY>
cudaError_t launch(const kea::ResidualNormArgs &a, bool vec, bool pdl, int sms, void *stream) {
    // As few threads per row as 32 values each allow, with no more values than that takes; while that leaves an SM
    // fewer than eight warps, twice the threads with half the values (a shorter chain of loads and sums).
    const auto threads_for = [&](int vpt) {
        int t = 32;
        while (t * vpt < a.D) t *= 2;
        return t;
    };
    int vpt = 32;
    while (vpt > 8 && threads_for(vpt / 2) == threads_for(vpt)) vpt /= 2;
    while (vpt > 8 && threads_for(vpt / 2) <= kea::kRnMaxThreads && (long long)a.M * threads_for(vpt) < 32LL * 8 * sms)
        vpt /= 2;
    const int tpr = threads_for(vpt);
    const int threads = std::max(kea::kRnThreads, tpr);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)ceil_div(a.M, threads / tpr), 1, 1);
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    if (pdl) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 1;
    }
#define KEA_RN(VPT, VEC) cudaLaunchKernelEx(&cfg, kea::residual_norm_kernel<TX, TY, VPT, VEC>, a, tpr)
    if (vec) return vpt == 8 ? KEA_RN(8, true) : vpt == 16 ? KEA_RN(16, true) : KEA_RN(32, true);
    return vpt == 8 ? KEA_RN(8, false) : vpt == 16 ? KEA_RN(16, false) : KEA_RN(32, false);
#undef KEA_RN
}

template <typename TX>
cudaError_t launch_for(const kea::ResidualNormArgs &a, int y_type, bool vec, bool pdl, int sms, void *stream) {
    switch (y_type) {
        case KEA_TYPE_F32: return launch<TX, float>(a, vec, pdl, sms, stream);
        case KEA_TYPE_F16: return launch<TX, __half>(a, vec, pdl, sms, stream);
        default: return launch<TX, __nv_bfloat16>(a, vec, pdl, sms, stream);
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
    const bool vec = vectors(d), pdl = (d->flags & KEA_RNORM_PDL) != 0;
    const cudaError_t e = d->x_type == KEA_TYPE_F32   ? launch_for<float>(a, d->y_type, vec, pdl, dev.sms, stream)
                          : d->x_type == KEA_TYPE_F16 ? launch_for<__half>(a, d->y_type, vec, pdl, dev.sms, stream)
                                                      : launch_for<__nv_bfloat16>(a, d->y_type, vec, pdl, dev.sms, stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return KEA_ERR_CUDA;
    }
    return KEA_OK;
}
