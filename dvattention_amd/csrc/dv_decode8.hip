// Attention over 8-bit caches: rows and row groups of two tokens (kernels: dv_decode8.h),
// and which kernels a call takes.  Built with accumulators in VGPRs.
#include "dv_decode8.h"

namespace dv {

namespace {

template <int DT, int QM, int RM>
hipError_t launch8_row(const DecodeParams& p, int device, long long cap, int cus, hipStream_t stream) {
    const bool p2 = p.bs_shift >= 4;
    if (p.F == 1)
        return p2 ? launch8_one<DT, QM, RM, 1, false, true>(p, device, cap, cus, stream)
                  : launch8_one<DT, QM, RM, 1, false, false>(p, device, cap, cus, stream);
    return p2 ? launch8_one<DT, QM, RM, 1, true, true>(p, device, cap, cus, stream)
              : launch8_one<DT, QM, RM, 1, true, false>(p, device, cap, cus, stream);
}

template <int DT>
hipError_t launch8(bool varlen, int nt, const DecodeParams& p, int device, long long cap, int cus,
                   hipStream_t stream) {
    if (nt == 1)
        return varlen ? launch8_row<DT, kQRotHalf, kRowVarlen>(p, device, cap, cus, stream)
                      : launch8_row<DT, kQRotFull, kRowWS>(p, device, cap, cus, stream);
    if constexpr (DT != kF32)
        return varlen ? launch8_one<DT, kQRotHalf, kRowVarlen, 2, true, true>(p, device, cap, cus, stream)
                      : launch8_one<DT, kQRotFull, kRowWS, 2, true, true>(p, device, cap, cus, stream);
    return hipErrorInvalidValue;
}

// Workspace of a call: partial slots (of the workgroups, and one per segment), then the
// merge directory.  The same for both workgroup shapes of pick_hpw8, but for the
// directory, which is larger with fewer heads per workgroup.
struct Ws8 {
    size_t part, total;
};
Ws8 ws8(long long groups, int nt, int Hkv, int device) {
    const long long rows = groups < kMaxRows ? groups : kMaxRows;
    const long long heads = (long long)device_cu_count(device) * 8 + rows * Hkv;  // of all slots
    Ws8 w;
    w.part = ((size_t)(heads * nt * kGqa * (kHeadDim + 1) * 4) + 255) & ~(size_t)255;
    w.total = w.part + (size_t)rows * (Hkv / pick_hpw(Hkv)) * 8;
    return w;
}

// KV heads (waves) per workgroup: eight where there are as many, whose rows of a token
// then lie side by side in memory as a workgroup reads them (32 sequences of 1k - 8k
// tokens, 8 KV heads: 62.6 -> 60.6 us, 4 x 131072: 191 -> 184), unless the call is too
// small to fill the chip so (one sequence of 3001 tokens: 11.0 us with four, 13.3).
int pick_hpw8(long long groups, long long max_keys, int Hkv, int cus) {
    if (Hkv % 8 == 0 && groups <= 1024 && groups * max_keys >= 256ll * cus) return 8;
    return pick_hpw(Hkv);
}

}  // namespace

size_t decode8_workspace_bytes(long long groups, int nt, int Hkv, int device) {
    return ws8(groups, nt, Hkv, device).total;
}

hipError_t launch_decode8(int dtype, bool varlen, int nt, const DecodeParams& base, long long groups,
                          long long max_keys_per_row, void* workspace, hipStream_t stream) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const Ws8 l = ws8(groups, nt, base.Hkv, device);
    const int cus = device_cu_count(device);
    DecodeParams p = base;
    p.hpw = pick_hpw8(groups, max_keys_per_row, p.Hkv, cus);
    const int nhg = p.Hkv / p.hpw;
    p.slot_floats = p.hpw * nt * kGqa * (kHeadDim + 1);
    p.part = reinterpret_cast<float*>(workspace);
    p.dir = reinterpret_cast<int*>(reinterpret_cast<unsigned char*>(workspace) + l.part);
    p.piece_cost = kPieceCost;
    p.min_keys = kDecodeMinKeys;
    p.skew_pm = xcd_skew_pm();
    for (long long r0 = 0; r0 < groups; r0 += kMaxRows) {
        p.row_begin = (int)r0;
        p.nrows = (int)(groups - r0 < kMaxRows ? groups - r0 : kMaxRows);
        const long long cap =
            ((long long)p.nrows * nhg * (max_keys_per_row + p.piece_cost) + p.min_keys - 1) / p.min_keys;
        switch (dtype) {
            case kBF16: e = launch8<kBF16>(varlen, nt, p, device, cap, cus, stream); break;
            case kF16: e = launch8<kF16>(varlen, nt, p, device, cap, cus, stream); break;
            case kF32: e = launch8<kF32>(varlen, nt, p, device, cap, cus, stream); break;
            default: e = hipErrorInvalidValue;
        }
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// ---- which kernels a call takes --------------------------------------------------------
//
// A wave of the decode kernels holds a token or, in 16-bit types, up to two tokens of a
// sequence beside each other (K and V are read once for them).  16-bit calls of
// few tokens are cut into such pairs, which read the cache once each; those of more go
// through the multi-query kernel, 16 tokens to a workgroup.  24 sequences of 4096 keys, 4
// KV heads, us as pairs and in the multi-query kernel:
//   bf16: 4 tokens 72, 97;   6 tokens 91, 100;   8 tokens 110, 103
//   fp16: 4 tokens 81, 136;  6 tokens 102, 137;  8 tokens 126, 140;  10 tokens 146, 144
// (Four tokens to a wave, which has the SIMD to itself then: 93 us for 4 in bf16.)  Packed 16-bit
// calls of two or more tokens per sequence are cut into row groups on the device; those of up
// to four tokens and those of more are two launches.
namespace {

constexpr int few_tokens(int dtype) { return dtype == kBF16 ? 6 : 8; }  // the same of a [W, S] call's sequence

struct Plan8 {
    bool table;                // varlen row groups
    int nt;                    // decode kernels: tokens of a wave (0: none)
    int sub;                   // blocks of a table entry
    bool chunk;                // multi-query kernel
    long long groups;          // [W, S]: row groups; table: entries
    size_t ws, table_bytes;
};

Plan8 plan8(int dtype, bool varlen, int W, int S_or_T, int Hkv, int device) {
    Plan8 q = {};
    const int S = varlen ? 1 : S_or_T;
    q.sub = 1;
    if (dtype == kF32) {
        q.nt = 1;
        q.groups = varlen ? S_or_T : (long long)W * S;
    } else if (varlen && use_varlen_chunk(dtype, S_or_T, W)) {
        q.table = true;
        q.groups = (long long)S_or_T / kGroupTokens + W + 1;
        q.table_bytes = (size_t)q.groups * 16;
        q.nt = 2;
        q.sub = kFewGroupTokens / 2;
        q.chunk = true;
    } else if (varlen) {
        q.nt = 1;
        q.groups = S_or_T;
    } else if (S <= few_tokens(dtype)) {
        q.nt = S < 2 ? S : 2;
        q.groups = (long long)W * ((S + q.nt - 1) / q.nt);
    } else {
        q.chunk = true;
        q.groups = (long long)W * ((S + kGroupTokens - 1) / kGroupTokens);
    }
    // (one after the other, both kernels of a table use the same bytes)
    size_t a = q.nt ? decode8_workspace_bytes(q.groups * q.sub, q.nt, Hkv, device) : 0;
    const size_t b = q.chunk ? chunk8_workspace_bytes(q.groups, Hkv, device) : 0;
    q.ws = ((a > b ? a : b) + 255) & ~(size_t)255;
    return q;
}

}  // namespace

size_t sdpa8_workspace_bytes(int dtype, bool varlen, int W, int S_or_T, int Hkv, int device) {
    if (W <= 0 || S_or_T <= 0 || Hkv <= 0) return 0;
    const Plan8 q = plan8(dtype, varlen, W, S_or_T, Hkv, device);
    return q.ws + q.table_bytes;
}

hipError_t launch_sdpa8(int dtype, bool varlen, const DecodeParams& base, long long max_keys, void* workspace,
                        size_t ws_bytes, hipStream_t stream) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const Plan8 q = plan8(dtype, varlen, base.W, varlen ? base.T : base.S, base.Hkv, device);
    if (ws_bytes < q.ws + q.table_bytes) return hipErrorInvalidValue;
    DecodeParams p = base;
    p.sub = q.sub;
    if (q.table) {
        int* groups = reinterpret_cast<int*>(reinterpret_cast<unsigned char*>(workspace) + q.ws);
        p.vgroups = groups;
        e = launch_varlen_groups(p.cu_q, p.W, p.T, (int)q.groups, groups, stream);
        if (e != hipSuccess) return e;
    }
    if (q.chunk) {
        e = launch_chunk8(dtype, varlen, p, q.groups, max_keys, workspace, stream);
        if (e != hipSuccess) return e;
    }
    if (q.nt) e = launch_decode8(dtype, varlen, q.nt, p, q.groups * q.sub, max_keys, workspace, stream);
    return e;
}

}  // namespace dv
