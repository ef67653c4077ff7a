// beam.cu - host side of the beam-search step: kea_lowbit_beam_select and kea_lowbit_beam_reorder.
#include <algorithm>
#include <atomic>

#include "beam_kernels.cuh"
#include "host.h"
#include "kea_lowbit.h"

namespace {

using kea_host::aligned;
using kea_host::ceil_div;

size_t type_size(int type) { return type == KEA_TYPE_F32 ? 4 : 2; }

// Indices of labels are 32 bits. A unit's end, a lane's next label and the label after the last vector are formed before they
// are compared with the row's end: at most 512 (units of a row) + 32 and 31 past it.
constexpr long long kMaxLabels = (1LL << 31) - 4096;

int validate(const KeaBeamDesc *d) {
    if (!d || d->clips < 0 || d->beams < 1 || d->vocab < 1 || d->width < 1 || d->end < -1 || d->end >= d->vocab ||
        d->logits_type < KEA_TYPE_F32 || d->logits_type > KEA_TYPE_BF16 || (d->flags & ~KEA_BEAM_PDL))
        return KEA_ERR_INVALID_VALUE;
    if (d->clips == 0) return KEA_OK;
    if (!d->logits || !d->scores || !d->out_scores || !d->parents || !d->labels || (d->ended && d->end < 0))
        return KEA_ERR_INVALID_VALUE;
    if (d->beams > kea::kBeamMax || d->width > kea::kBeamMax || (long long)d->beams * d->vocab > kMaxLabels ||
        d->width > (long long)d->beams * d->vocab || (long long)d->clips * kea::kBeamCluster >= (1LL << 31))
        return KEA_ERR_UNSUPPORTED;
    if (!aligned(d->logits, type_size(d->logits_type)) || !aligned(d->scores, 4) || !aligned(d->out_scores, 4) ||
        !aligned(d->parents, 4) || !aligned(d->labels, 4))
        return KEA_ERR_ALIGNMENT;
    return KEA_OK;
}

template <typename T, int WARPS>
cudaError_t launch_select_as(const kea::BeamArgs &a, int clips, int device, bool pdl, void *stream) {
    const auto kernel = kea::beam_select_kernel<T, WARPS>;
    static std::atomic<uint64_t> ready{0};   // devices on which clusters of 16 are allowed
    if (a.ctas > 8 && !(ready.load(std::memory_order_acquire) >> device & 1)) {
        const cudaError_t e = cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        ready.fetch_or(1ULL << device, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attrs[2];
    cfg.gridDim = dim3((unsigned)(a.ctas * clips), 1, 1);
    cfg.blockDim = dim3(32 * WARPS, 1, 1);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attrs;
    if (a.ctas > 1) {
        attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[cfg.numAttrs].val.clusterDim.x = (unsigned)a.ctas;
        attrs[cfg.numAttrs].val.clusterDim.y = 1;
        attrs[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    if (pdl) {
        attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T>
cudaError_t launch_select(const kea::BeamArgs &a, int clips, int warps, int device, bool pdl, void *stream) {
    return warps == 8 ? launch_select_as<T, 8>(a, clips, device, pdl, stream) : launch_select_as<T, 32>(a, clips, device, pdl, stream);
}

}  // namespace

extern "C" int kea_lowbit_beam_select(const KeaBeamDesc *d, void *stream) {
    const int v = validate(d);
    if (v != KEA_OK || d->clips == 0) return v;
    kea_host::Device dev;
    const int st = kea_host::device(&dev, stream);
    if (st != KEA_OK) return st;
    kea::BeamArgs a{};
    a.logits = d->logits;
    a.ld_clip = d->ld_clip;
    a.ld_beam = d->ld_beam;
    a.scores = d->scores;
    a.ended = d->ended;
    a.out_scores = d->out_scores;
    a.parents = d->parents;
    a.labels = d->labels;
    a.out_ended = d->out_ended;
    a.beams = d->beams;
    a.vocab = d->vocab;
    a.width = d->width;
    a.end = d->end;
    // Warps per clip: as many as the SMs hold at once (32 each), as long as each keeps some 512 logits; in CTAs of 8,
    // or of 32 where a cluster of 16 of those is not enough.
    const long long wanted = std::min((long long)d->beams * d->vocab / 512, 32LL * dev.sms / d->clips);
    const int warps = wanted <= 8 * kea::kBeamCluster ? 8 : 32;
    a.ctas = 1;
    while (a.ctas < kea::kBeamCluster && 2LL * a.ctas * warps <= wanted) a.ctas *= 2;
    const int all = a.ctas * warps;
    a.segs = std::max(1, all / d->beams);
    a.units = a.segs * d->beams;
    a.rounds = ceil_div(a.units, all);
    const bool pdl = (d->flags & KEA_BEAM_PDL) != 0;
    const cudaError_t e = d->logits_type == KEA_TYPE_F32   ? launch_select<float>(a, d->clips, warps, dev.index, pdl, stream)
                          : d->logits_type == KEA_TYPE_F16 ? launch_select<__half>(a, d->clips, warps, dev.index, pdl, stream)
                                                           : launch_select<__nv_bfloat16>(a, d->clips, warps, dev.index, pdl, stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return KEA_ERR_CUDA;
    }
    return KEA_OK;
}

extern "C" int kea_lowbit_beam_reorder(const KeaReorderDesc *d, const KeaReorderItem *items, void *stream) {
    if (!d || d->count < 0 || d->count > KEA_REORDER_MAX || d->clips < 0 || d->beams < 1 || d->width < 1 ||
        (d->flags & ~KEA_BEAM_PDL))
        return KEA_ERR_INVALID_VALUE;
    if (d->count == 0 || d->clips == 0) return KEA_OK;
    if (!d->parents || !items) return KEA_ERR_INVALID_VALUE;
    if (!aligned(d->parents, 4)) return KEA_ERR_ALIGNMENT;
    kea::ReorderArgs a;
    long long blocks = 0;
    a.count = 0;
    for (int i = 0; i < d->count; ++i) {
        const KeaReorderItem &s = items[i];
        if (s.groups < 1 || s.row_bytes < 0) return KEA_ERR_INVALID_VALUE;
        if (s.row_bytes == 0) continue;
        if (!s.src || !s.dst) return KEA_ERR_INVALID_VALUE;
        const long long rows = (long long)s.groups * d->clips * d->width;
        if (rows >= (1LL << 31) || s.row_bytes >= (1LL << 31)) return KEA_ERR_UNSUPPORTED;
        const uint64_t all = reinterpret_cast<uintptr_t>(s.src) | reinterpret_cast<uintptr_t>(s.dst) | (uint64_t)s.src_group |
                             (uint64_t)s.src_clip | (uint64_t)s.src_beam | (uint64_t)s.dst_group | (uint64_t)s.dst_clip |
                             (uint64_t)s.dst_beam | (uint64_t)s.row_bytes;
        kea::ReorderItem &t = a.item[a.count++];
        t.src = static_cast<const uint8_t *>(s.src);
        t.dst = static_cast<uint8_t *>(s.dst);
        t.src_group = s.src_group;
        t.src_clip = s.src_clip;
        t.src_beam = s.src_beam;
        t.dst_group = s.dst_group;
        t.dst_clip = s.dst_clip;
        t.dst_beam = s.dst_beam;
        t.unit = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
        t.row = (int)(s.row_bytes / t.unit);
        t.rows = (unsigned)rows;
        t.first_block = (unsigned)blocks;
        t.rows_per_block = t.row <= kea::kReorderUnits ? kea::kReorderUnits / t.row : 0;
        t.blocks_per_row = ceil_div(t.row, kea::kReorderUnits);
        blocks += t.rows_per_block ? ceil_div(rows, t.rows_per_block) : rows * t.blocks_per_row;
        if (blocks >= (1LL << 31)) return KEA_ERR_UNSUPPORTED;
    }
    if (a.count == 0) return KEA_OK;
    kea_host::Device dev;
    const int st = kea_host::device(&dev, stream);
    if (st != KEA_OK) return st;
    a.parents = d->parents;
    a.clips = d->clips;
    a.beams = d->beams;
    a.width = d->width;
    a.err = d->error_word ? d->error_word : dev.error_word;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)blocks, 1, 1);
    cfg.blockDim = dim3(kea::kReorderThreads, 1, 1);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    if (d->flags & KEA_BEAM_PDL) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 1;
    }
    if (cudaLaunchKernelEx(&cfg, kea::beam_reorder_kernel, a) != cudaSuccess) {
        cudaGetLastError();
        return KEA_ERR_CUDA;
    }
    return KEA_OK;
}
