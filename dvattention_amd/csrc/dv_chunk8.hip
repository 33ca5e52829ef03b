// gfx950 multi-query attention over 8-bit caches: instances of the kernel in
// dv_chunk_kernel.h whose 16-bit tiles are made from E4M3 rows in LDS, and their launches.
// Built like dv_chunk.hip.
#include "dv_chunk_kernel.h"

namespace dv {
namespace chunk {

static_assert(kTokBlk == kGroupTokens && kFewTok == kFewGroupTokens, "groups of a packed call's two launches");

template <int DT, int QM, bool P2, int RM>
hipError_t launch8(DecodeParams p, int device, int cus, long long cap, hipStream_t stream) {
    static std::atomic<unsigned long long> attr_done{0};
    hipError_t e = once_per_device(attr_done, device, [] {
        return hipFuncSetAttribute(reinterpret_cast<const void*>(&dv_chunk<DT, QM, kKvPaged, P2, RM, 1, true>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes<true>(kMaxRows));
    });
    if (e != hipSuccess) return e;
    const long long nwg = cus < cap ? cus : cap;  // one eight-wave workgroup per CU
    p.nwg = nwg < 1 ? 1 : (int)nwg;
    hipLaunchKernelGGL((dv_chunk<DT, QM, kKvPaged, P2, RM, 1, true>), dim3(p.nwg), dim3(kThreads),
                       lds_bytes<true>(p.nrows), stream, p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int ntb = max_group_tokens<RM>(p);
    hipLaunchKernelGGL((dv_merge_chunk<DT, RM, RM == kRowVarlen>), dim3(p.nrows * p.Hkv * ntb), dim3(256), 0, stream,
                       p, ntb);
    return hipGetLastError();
}

template <int DT, int QM, int RM>
hipError_t launch8(const DecodeParams& p, int device, int cus, long long cap, hipStream_t stream) {
    return p.bs_shift >= 0 ? launch8<DT, QM, true, RM>(p, device, cus, cap, stream)
                           : launch8<DT, QM, false, RM>(p, device, cus, cap, stream);
}

}  // namespace chunk

namespace {
struct Ws {
    size_t part, total;
};
Ws chunk8_ws(long long groups, int Hkv, int device) {
    const long long nseg = (groups < kMaxRows ? groups : kMaxRows) * Hkv;
    Ws w;
    w.part = ((size_t)((device_cu_count(device) + nseg) * (chunk::kTokBlk * kGqa * (kHeadDim + 1)) * 4) + 255) &
             ~(size_t)255;
    w.total = w.part + (size_t)nseg * 8;
    return w;
}
}  // namespace

size_t chunk8_workspace_bytes(long long groups, int Hkv, int device) { return chunk8_ws(groups, Hkv, device).total; }

hipError_t launch_chunk8(int dtype, bool varlen, const DecodeParams& base, long long groups,
                         long long max_keys_per_group, void* workspace, hipStream_t stream) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const int cus = device_cu_count(device);
    DecodeParams p = base;
    p.hpw = 1;
    p.slot_floats = chunk::kTokBlk * kGqa * (kHeadDim + 1);
    p.part = reinterpret_cast<float*>(workspace);
    p.dir = reinterpret_cast<int*>(reinterpret_cast<unsigned char*>(workspace) +
                                   chunk8_ws(groups, p.Hkv, device).part);
    p.piece_cost = chunk::kPieceCost;
    p.min_keys = 256;
    p.skew_pm = 30;  // as the 16-bit launches
    chunk::fold_scale(p);
    for (long long g0 = 0; g0 < groups; g0 += kMaxRows) {
        p.row_begin = (int)g0;
        p.nrows = (int)(groups - g0 < kMaxRows ? groups - g0 : kMaxRows);
        const long long cap =
            ((long long)p.nrows * p.Hkv * (max_keys_per_group + p.piece_cost) + p.min_keys - 1) / p.min_keys;
        if (dtype == kBF16)
            e = varlen ? chunk::launch8<kBF16, kQRotHalf, kRowVarlen>(p, device, cus, cap, stream)
                       : chunk::launch8<kBF16, kQRotFull, kRowWS>(p, device, cus, cap, stream);
        else if (dtype == kF16)
            e = varlen ? chunk::launch8<kF16, kQRotHalf, kRowVarlen>(p, device, cus, cap, stream)
                       : chunk::launch8<kF16, kQRotFull, kRowWS>(p, device, cus, cap, stream);
        else
            e = hipErrorInvalidValue;
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace dv
