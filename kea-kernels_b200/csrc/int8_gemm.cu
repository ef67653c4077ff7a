// int8_gemm.cu - host side of the 8-bit linear map (kea_lowbit_int8_gemm): argument checks, the choice of kernel and the
// launches.
#include <algorithm>

#include "host.h"
#include "int8_reg_kernel.cuh"
#include "kea_lowbit.h"

namespace {

using kea_host::aligned;
using kea_host::ceil_div;

constexpr int kMaxK = 131071;   // 128 * 128 * k < 2^31
constexpr int kRegMaxSmem = 64 * 1024;

int validate(const KeaInt8Desc *d) {
    if (!d || d->m < 0 || d->n < 1 || d->k < 1 || d->y_type < KEA_TYPE_F32 || d->y_type > KEA_TYPE_BF16 ||
        (d->flags & ~(KEA_INT8_SILU | KEA_INT8_PDL)) || d->kernel < 0 || d->kernel > KEA_INT8_KERNEL_REG)
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
template <typename T, int CG, int RG, int D>
cudaError_t launch_reg_as(const kea::Int8Args &a, int ks, bool pdl, void *stream) {
    const int cn = 16 * CG * (kea::kI8RegWarps / ks);
    const Launch l(dim3((unsigned)ceil_div(a.N, cn), (unsigned)ceil_div(a.M, 8 * RG), 1), kea::kI8RegThreads,
                   (size_t)kea::i8reg_smem_bytes(ks, 8 * RG, cn), stream, pdl);
    return cudaLaunchKernelEx(&l.cfg, kea::int8_gemm_reg_kernel<T, CG, RG, D>, a, ks);
}

template <typename T>
cudaError_t launch_reg(const kea::Int8Args &a, int sms, bool pdl, void *stream) {
    return launch_reg_as<T, 2, 4, 2>(a, a.K >= 512 ? 4 : 1, pdl, stream);
}

}  // namespace

int kea_host::setup_int8_gemm() { return KEA_OK; }

extern "C" int kea_lowbit_int8_gemm(const KeaInt8Desc *d, void *stream) {
    const int v = validate(d);
    if (v != KEA_OK || d->m == 0) return v;
    kea_host::Device dev;
    const int st = kea_host::device(&dev, stream);
    if (st != KEA_OK) return st;
    const kea::Int8Args a = arguments(d, dev);
    const bool pdl = (d->flags & KEA_INT8_PDL) != 0;
    if (ceil_div(a.M, 32) > 65535) return KEA_ERR_UNSUPPORTED;
    const cudaError_t e = a.y_type == KEA_TYPE_F32   ? launch_reg<float>(a, dev.sms, pdl, stream)
                          : a.y_type == KEA_TYPE_F16 ? launch_reg<__half>(a, dev.sms, pdl, stream)
                                                     : launch_reg<__nv_bfloat16>(a, dev.sms, pdl, stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return KEA_ERR_CUDA;
    }
    return KEA_OK;
}
