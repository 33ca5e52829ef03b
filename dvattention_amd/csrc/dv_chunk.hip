// gfx950 multi-query attention over 16-bit caches: instances of the kernel in
// dv_chunk_kernel.h, the varlen row groups, and the launches of the multi-query path.
#include "dv_chunk_kernel.h"

namespace dv {
namespace chunk {

// ---- varlen row groups ----------------------------------------------------------
//
// Token t of a varlen call belongs to the first sequence i with
// t < cu_seqlens_q[i + 1], or to sequence 0 when there is none (the decode
// path's rule, varlen_paged_kernel_v21.cuh:40-47).  With M_i the running
// maximum of cu_seqlens_q[1 .. i + 1], sequence i's tokens are therefore
// [max(0, M_{i-1}), min(T, M_i)) (M_{-1} = 0), and the tokens from M_{W-1} on
// form one more run, of sequence 0 -- also for tables that are not
// non-decreasing.  Each run is cut into groups of kTokBlk tokens.  One
// workgroup writes entry g = {first token, tokens, sequence, 0} for every
// group, and {0, 0, 0, 0} for the entries from the group count up to gmax
// (the host's bound T / kTokBlk + W + 1: a run of n tokens makes at most
// n / kTokBlk + 1 groups).
constexpr int kVgThreads = 1024;

__device__ inline int block_scan_excl(int v, int* s_part, bool is_max) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int ident = is_max ? INT_MIN : 0;
    int incl = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int o = __shfl_up(incl, d, kWave);
        if (lane >= d) incl = is_max ? (o > incl ? o : incl) : incl + o;
    }
    if (lane == 63) s_part[wv] = incl;
    __syncthreads();
    int before = ident;
    for (int i = 0; i < wv; ++i) before = is_max ? (s_part[i] > before ? s_part[i] : before) : before + s_part[i];
    const int excl_lane = __shfl_up(incl, 1, kWave);
    const int mine = lane == 0 ? ident : excl_lane;
    __syncthreads();
    return is_max ? (mine > before ? mine : before) : before + mine;
}

__global__ __launch_bounds__(kVgThreads) void dv_varlen_groups(const int* cu, int W, int T, int gmax, int4* groups) {
    __shared__ int s_m[kVarlenChunkMaxW];       // M_i
    __shared__ int s_base[kVarlenChunkMaxW + 2];  // first group of run i (runs 0 .. W), then the total
    __shared__ int s_part[kVgThreads / kWave];
    const int tid = threadIdx.x;
    // running maximum of cu[1 .. W], each thread over a contiguous block of sequences
    const int per = (W + kVgThreads - 1) / kVgThreads;
    const int i0 = tid * per < W ? tid * per : W, i1 = i0 + per < W ? i0 + per : W;
    int mx = INT_MIN;
    for (int i = i0; i < i1; ++i) {
        const int c = cu[i + 1];
        mx = c > mx ? c : mx;
        s_m[i] = mx;
    }
    const int before = block_scan_excl(mx, s_part, true);
    for (int i = i0; i < i1; ++i) s_m[i] = s_m[i] > before ? s_m[i] : before;
    __syncthreads();
    // run i (i < W: sequence i; i == W: the tokens past M_{W-1}) = [a, b)
    auto run = [&](int i, int& a, int& b) {
        a = i == 0 ? 0 : (s_m[i - 1] > 0 ? s_m[i - 1] : 0);
        b = i == W ? T : (s_m[i] < T ? s_m[i] : T);
    };
    const int per1 = (W + 1 + kVgThreads - 1) / kVgThreads;
    const int j0 = tid * per1 < W + 1 ? tid * per1 : W + 1, j1 = j0 + per1 < W + 1 ? j0 + per1 : W + 1;
    int cnt = 0;
    for (int i = j0; i < j1; ++i) {
        int a, b;
        run(i, a, b);
        const int c = b > a ? (b - a + kTokBlk - 1) / kTokBlk : 0;
        s_base[i] = c;
        cnt += c;
    }
    int acc = block_scan_excl(cnt, s_part, false);
    for (int i = j0; i < j1; ++i) {
        const int c = s_base[i];
        s_base[i] = acc;
        acc += c;
    }
    if (tid == kVgThreads - 1) s_base[W + 1] = acc;
    __syncthreads();
    const int total = s_base[W + 1];
    for (int gi = tid; gi < gmax; gi += kVgThreads) {
        int4 e = {0, 0, 0, 0};
        if (gi < total) {
            // the last run whose first group is <= gi (it has groups: the next run's first is larger)
            int lo = 0, hi = W;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_base[mid] <= gi) lo = mid;
                else hi = mid - 1;
            }
            int a, b;
            run(lo, a, b);
            const int t0 = a + (gi - s_base[lo]) * kTokBlk;
            e.x = t0;
            e.y = b - t0 < kTokBlk ? b - t0 : kTokBlk;
            e.z = lo == W ? 0 : lo;
        }
        groups[gi] = e;
    }
}

template <int DT, int QM, int KVM, bool P2, int RM, int KS>
hipError_t launch1(DecodeParams p, int device, int cus, long long cap, hipStream_t stream) {
    static std::atomic<unsigned long long> attr_done{0};
    hipError_t ea = once_per_device(attr_done, device, [] {
        return hipFuncSetAttribute(reinterpret_cast<const void*>(&dv_chunk<DT, QM, KVM, P2, RM, KS>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes<>(kMaxRows));
    });
    if (ea != hipSuccess) return ea;
    const size_t lds = lds_bytes<>(p.nrows);
    long long nwg = cus;  // one eight-wave workgroup per CU (LDS ring 96 KiB)
    if (nwg > cap) nwg = cap;
    p.nwg = nwg < 1 ? 1 : (int)nwg;
    hipLaunchKernelGGL((dv_chunk<DT, QM, KVM, P2, RM, KS>), dim3(p.nwg), dim3(kThreads), lds, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int ntb = max_group_tokens<RM>(p);
    if (p.parents) return launch_merge_tree(DT, p, ntb, stream);
    hipLaunchKernelGGL((dv_merge_chunk<DT, RM>), dim3(p.nrows * p.Hkv * ntb), dim3(256), 0, stream, p, ntb);
    return hipGetLastError();
}

template <int DT, int QM, int KVM, int RM, bool P2>
hipError_t launch_split(const DecodeParams& p, int ks, int device, int cus, long long cap, hipStream_t stream) {
    if constexpr (RM == kRowVarlen) {
        return launch1<DT, QM, KVM, P2, RM, 0>(p, device, cus, cap, stream);
    } else {
        if (ks == 4) return launch1<DT, QM, KVM, P2, RM, 4>(p, device, cus, cap, stream);
        if (ks == 2) return launch1<DT, QM, KVM, P2, RM, 2>(p, device, cus, cap, stream);
        return launch1<DT, QM, KVM, P2, RM, 1>(p, device, cus, cap, stream);
    }
}

template <int DT, int QM, int KVM, int RM>
hipError_t launch(const DecodeParams& p, int ks, int device, int cus, long long cap, hipStream_t stream) {
    if constexpr (DT == kF32) {
        return launch_chunk32(QM, KVM, RM, p, device, cus, cap, stream);
    } else {
        if constexpr (KVM == kKvPaged)
            if (p.bs_shift >= 0) return launch_split<DT, QM, KVM, RM, true>(p, ks, device, cus, cap, stream);
        return launch_split<DT, QM, KVM, RM, false>(p, ks, device, cus, cap, stream);
    }
}

// Key split of a launch whose groups have at most ntok tokens: as many wave sets
// as hold two tokens per wave.  (Eight sets for two tokens would take a ring step
// of all eight stages, with nothing in flight beside it; two tokens run at 5.3
// TB/s with four.)  Faster than no split over the whole range: 2 / 4 / 8 tokens,
// bf16, one sequence of 3001 keys, 8 KV heads 29.7 / 30.8 / 32.7 -> 26.2 / 27.1 /
// 29.1 us; fp16, 32 x 4608 keys 224 / 223 / 234 -> 112 / 114 / 153; contiguous fp16,
// 16 x 4096 keys 119 / 120 / 122 -> 60 / 63 / 84; 64 x 60-100 keys, bf16 50.1 /
// 52.5 / 58.7 -> 45.1 / 47.0 / 51.6.  Short views
// gain nothing (each one's queries are staged for all sets, and a piece ends with the
// sets' combination), so a call is split from 48 keys per view on, as far as the host
// knows them (paged: what the block tables hold), and a contiguous one of 5 - 8
// tokens in several views from 128 on: without the split / with it, 8 KV heads, 6 x 30
// contiguous keys, 2 tokens 68 / 76 us, paged 96 / 99; 12 x 90 contiguous, 8 tokens 62
// / 67; 6 x 60 paged, 2 / 8 tokens 65 / 62, 70 / 62; 6 x 150 contiguous, 8 tokens 51 / 50.
int key_split(int ntok, long long keys, int F, bool contig) {
    if (ntok > 8) return 1;
    const int ks = ntok > kFewTok ? 2 : 4;
    const long long per_view = contig && ks == 2 && F > 1 ? kSplitContig2Keys : kSplitMinKeys;
    return keys < per_view * F ? 1 : ks;
}

}  // namespace chunk

namespace {
int chunk_cus(int device) { return device_cu_count(device); }

// Workspace of the chunk path for `groups` row groups: partial slots, merge
// directory, and (varlen) the group table.
struct ChunkWs {
    size_t part, dir, vgroups, total;
};

ChunkWs chunk_ws(long long groups, int Hkv, int device, bool varlen) {
    const long long rows = groups < kMaxRows ? groups : kMaxRows;
    const long long nseg = rows * Hkv;
    const long long slot_floats = (long long)chunk::kTokBlk * kGqa * (kHeadDim + 1);
    ChunkWs l;
    l.part = ((size_t)((chunk_cus(device) + nseg) * slot_floats * 4) + 255) & ~(size_t)255;
    l.dir = ((size_t)(nseg * 2 * 4) + 255) & ~(size_t)255;
    l.vgroups = varlen ? (size_t)groups * 16 : 0;
    l.total = l.part + l.dir + l.vgroups;
    return l;
}

long long varlen_gmax(int T, int W) { return (long long)T / chunk::kTokBlk + W + 1; }

// The chunk launches over `groups` row groups, kMaxRows at a time.
template <int RM>
hipError_t launch_groups(int dtype, int qmode, int kvmode, DecodeParams p, long long groups_total,
                         long long max_keys_per_group, int ks, const ChunkWs& l, void* workspace,
                         hipStream_t stream) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const int cus = chunk_cus(device);
    p.hpw = 1;
    p.slot_floats = chunk::kTokBlk * kGqa * (kHeadDim + 1);
    p.part = reinterpret_cast<float*>(workspace);
    p.dir = reinterpret_cast<int*>(reinterpret_cast<unsigned char*>(workspace) + l.part);
    // ks = 0: the schedule counts in cost units (dv_chunk)
    const int unit = ks == 0 ? chunk::kLongKeyCost : 1;
    p.piece_cost = unit * (ks <= 1 ? chunk::kPieceCost : chunk::kPieceCostSplit);
    const int min_keys = p.min_keys;
    p.min_keys *= unit;
    // odd workgroups (odd XCD of each pair) take shorter chunks, as in the decode
    // split; 30 per mille measured best on configuration 5
    static const int skew = env_per_mille("DVATTN_CHUNK_SKEW_PM", 30);
    p.skew_pm = skew;
    chunk::fold_scale(p);
    for (long long g0 = 0; g0 < groups_total; g0 += kMaxRows) {
        p.row_begin = (int)g0;
        p.nrows = (int)(groups_total - g0 < kMaxRows ? groups_total - g0 : kMaxRows);
        const long long cap = ((long long)p.nrows * p.Hkv * max_keys_per_group + min_keys - 1) / min_keys;
        if constexpr (RM == kRowVarlen) {
            if (dtype == kBF16 && qmode == kQRotHalf && kvmode == kKvPaged)
                e = chunk::launch<kBF16, kQRotHalf, kKvPaged, RM>(p, ks, device, cus, cap, stream);
            else if (dtype == kF16 && qmode == kQRotHalf && kvmode == kKvPaged)
                e = chunk::launch<kF16, kQRotHalf, kKvPaged, RM>(p, ks, device, cus, cap, stream);
            else if (dtype == kF32 && qmode == kQRotHalf && kvmode == kKvPaged)
                e = chunk::launch<kF32, kQRotHalf, kKvPaged, RM>(p, ks, device, cus, cap, stream);
            else
                e = hipErrorInvalidValue;
        } else {
            if (dtype == kBF16 && qmode == kQRotFull && kvmode == kKvPaged)
                e = chunk::launch<kBF16, kQRotFull, kKvPaged, RM>(p, ks, device, cus, cap, stream);
            else if (dtype == kF16 && qmode == kQRotFull && kvmode == kKvPaged)
                e = chunk::launch<kF16, kQRotFull, kKvPaged, RM>(p, ks, device, cus, cap, stream);
            else if (dtype == kBF16 && qmode == kQPre && kvmode == kKvContig)
                e = chunk::launch<kBF16, kQPre, kKvContig, RM>(p, ks, device, cus, cap, stream);
            else if (dtype == kF16 && qmode == kQPre && kvmode == kKvContig)
                e = chunk::launch<kF16, kQPre, kKvContig, RM>(p, ks, device, cus, cap, stream);
            else if (dtype == kF32 && qmode == kQRotFull && kvmode == kKvPaged)
                e = chunk::launch<kF32, kQRotFull, kKvPaged, RM>(p, ks, device, cus, cap, stream);
            else if (dtype == kF32 && qmode == kQPre && kvmode == kKvContig)
                e = chunk::launch<kF32, kQPre, kKvContig, RM>(p, ks, device, cus, cap, stream);
            else
                e = hipErrorInvalidValue;
        }
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
}  // namespace

size_t chunk_workspace_bytes(int W, int S, int Hkv, int device) {
    if (W <= 0 || S <= 0 || Hkv <= 0) return 0;
    const long long groups = (long long)W * ((S + chunk::kTokBlk - 1) / chunk::kTokBlk);
    return chunk_ws(groups, Hkv, device, false).total;
}

hipError_t launch_chunk(int dtype, int qmode, int kvmode, const DecodeParams& base, long long max_keys_per_group,
                        void* workspace, size_t ws_bytes, hipStream_t stream) {
    if (base.W <= 0 || base.S <= 0 || base.Hkv <= 0) return hipSuccess;
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const long long groups = (long long)base.W * ((base.S + chunk::kTokBlk - 1) / chunk::kTokBlk);
    const ChunkWs l = chunk_ws(groups, base.Hkv, device, false);
    if (ws_bytes < l.total) return hipErrorInvalidValue;
    const int ks = dtype == kF32 ? 1
                                 : chunk::key_split(base.S, max_keys_per_group, base.F, kvmode == kKvContig);
    return launch_groups<kRowWS>(dtype, qmode, kvmode, base, groups, max_keys_per_group, ks, l, workspace, stream);
}

hipError_t launch_varlen_groups(const int* cu, int W, int T, int gmax, int* groups, hipStream_t stream) {
    hipLaunchKernelGGL(chunk::dv_varlen_groups, dim3(1), dim3(chunk::kVgThreads), 0, stream, cu, W, T, gmax,
                       reinterpret_cast<int4*>(groups));
    return hipGetLastError();
}

size_t varlen_chunk_workspace_bytes(int T, int W, int Hkv, int device) {
    if (T <= 0 || W <= 0 || Hkv <= 0) return 0;
    return chunk_ws(varlen_gmax(T, W), Hkv, device, true).total;
}

hipError_t launch_varlen_chunk(int dtype, const DecodeParams& base, long long max_keys_per_group, void* workspace,
                               size_t ws_bytes, hipStream_t stream) {
    if (base.T <= 0 || base.W <= 0 || base.Hkv <= 0) return hipSuccess;
    if (base.W > kVarlenChunkMaxW) return hipErrorInvalidValue;
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const long long gmax = varlen_gmax(base.T, base.W);
    const ChunkWs l = chunk_ws(gmax, base.Hkv, device, true);
    if (ws_bytes < l.total) return hipErrorInvalidValue;
    DecodeParams p = base;
    int4* groups = reinterpret_cast<int4*>(reinterpret_cast<unsigned char*>(workspace) + l.part + l.dir);
    p.vgroups = reinterpret_cast<const int*>(groups);
    e = launch_varlen_groups(base.cu_q, base.W, base.T, (int)gmax, reinterpret_cast<int*>(groups), stream);
    if (e != hipSuccess) return e;
    const int ks = dtype == kF32 ? 1 : 0;
    return launch_groups<kRowVarlen>(dtype, kQRotHalf, kKvPaged, p, gmax, max_keys_per_group, ks, l, workspace,
                                     stream);
}

}  // namespace dv
