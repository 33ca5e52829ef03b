// Bounded caches: which rows to keep (dv_kv_select) and their move together
// (dv_kv_compact).
#include "dv_common.h"
#include "dv_device.h"

namespace dv {

namespace {

typedef __attribute__((address_space(1))) u32x4 gw_u32x4;

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kDigit = 11;  // bits of a weight resolved per pass: 11 + 11 + 10
constexpr int kBins = 1 << kDigit;

// Weights as integers in their order; a NaN is lighter than any number.
__device__ inline uint32_t order_of(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
    if ((u & 0x7fffffffu) == 0u) return 0x80000000u;  // -0 and +0 weigh the same
    return (u >> 31) ? ~u : u | 0x80000000u;
}

// Exclusive sum of v over the block's threads, and the total.
__device__ inline int block_excl(int v, int* s_wave, int& total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int o = __shfl_up(incl, d, kWave);
        if (lane >= d) incl += o;
    }
    if (lane == 63) s_wave[wv] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) {
        const int x = s_wave[i];
        before += i < wv ? x : 0;
        all += x;
    }
    __syncthreads();
    total = all;
    return before + incl - v;
}

}  // namespace

// Block = (sequence, KV head).  Of the n rows, the first keep_first and the last
// keep_last stay, and of those between the `need` heaviest: the weight T of the
// need-th is found digit by digit (a histogram of the digit over the rows that
// agree with T so far, most significant first), then the rows above T and the first
// of those equal to it (ties go to the lowest row) are written in ascending order,
// their places from a running count.  Bound by latency: the weights are read from
// memory once and then from L2 three more times, each pass a few barriers.
__global__ __launch_bounds__(kSelThreads) void dv_kv_select(const SelectParams p) {
    __shared__ int s_hist[kBins];
    __shared__ int s_wave[kSelWaves];
    __shared__ int s_digit, s_above;
    const int tid = threadIdx.x;
    const int w = blockIdx.x / p.Hkv;
    int* rows = p.rows + (long long)blockIdx.x * p.budget;
    const long long first = p.first[w];
    long long cap = first < 0 ? 0 : p.C - first;
    if (cap < 0) cap = 0;
    long long len = p.lengths[w];
    len = len < 0 ? 0 : len;
    const int n = (int)(len < cap ? len : cap);
    if (n <= p.budget) {
        for (int i = tid; i < p.budget; i += kSelThreads) rows[i] = i < n ? i : -1;
        return;
    }
    const int a = p.keep_first, b = n - p.keep_last;  // rows [a, b) compete
    const int need = p.budget - p.keep_first - p.keep_last;
    const float* mass = p.mass + (long long)blockIdx.x * p.C + first;
    for (int i = tid; i < a; i += kSelThreads) rows[i] = i;
    for (int i = tid; i < p.keep_last; i += kSelThreads) rows[a + need + i] = b + i;
    if (need == 0) return;

    uint32_t top = 0;   // T's digits so far
    int want = need;    // of the rows that agree with them, how many stay
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t known = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u;
        const uint32_t mask = pass == 2 ? 0x3ffu : 0x7ffu;
        for (int i = tid; i < kBins; i += kSelThreads) s_hist[i] = 0;
        __syncthreads();
        for (int i0 = a; i0 < b; i0 += kSelThreads) {
            const int i = i0 + tid;
            const bool in = i < b;
            const uint32_t u = order_of(in ? mass[i] : 0.0f);
            const bool match = in && (u & known) == top;
            const int dg = (int)((u >> shift) & mask);
            // lanes of one digit count together (weights of one power of two, or all zero)
            const uint64_t live = ballot(match);
            if (live) {
                const int lead = __builtin_amdgcn_readlane(dg, __builtin_ctzll(live));
                const uint64_t same = ballot(match && dg == lead);
                if ((tid & 63) == __builtin_ctzll(live)) atomicAdd(&s_hist[lead], __builtin_popcountll(same));
                if (match && dg != lead) atomicAdd(&s_hist[dg], 1);
            }
        }
        __syncthreads();
        // the digit whose rows hold the want-th heaviest: thread t owns bins 2t, 2t + 1
        // counted from the heaviest
        const int h0 = s_hist[kBins - 1 - 2 * tid], h1 = s_hist[kBins - 2 - 2 * tid];
        int total;
        const int before = block_excl(h0 + h1, s_wave, total);
        if (before < want && want <= before + h0) {
            s_digit = kBins - 1 - 2 * tid;
            s_above = before;
        } else if (before + h0 < want && want <= before + h0 + h1) {
            s_digit = kBins - 2 - 2 * tid;
            s_above = before + h0;
        }
        __syncthreads();
        top |= (uint32_t)s_digit << shift;
        want -= s_above;
    }

    // rows above T, and the first `want` of those equal to it
    int out = a, ties = 0;
    for (int i0 = a; i0 < b; i0 += kSelThreads) {
        const int i = i0 + tid;
        const uint32_t u = i < b ? order_of(mass[i]) : 0u;
        const bool gt = i < b && u > top, eq = i < b && u == top;
        // both counts in one scan: at most 1024 of each
        int total;
        const int e = block_excl((gt ? 1 : 0) | (eq ? 1 << 16 : 0), s_wave, total);
        const int eqs = ties + (e >> 16);              // equal rows before this one
        const int eq_kept = eqs < want ? eqs : want;   // of them, kept
        const int gts = e & 0xffff;
        const int ties_kept0 = ties < want ? ties : want;
        if (gt || (eq && eqs < want)) rows[out + gts + (eq_kept - ties_kept0)] = i;
        const int ties1 = ties + (total >> 16);
        out += (total & 0xffff) + ((ties1 < want ? ties1 : want) - ties_kept0);
        ties = ties1;
    }
}

hipError_t launch_kv_select(const SelectParams& p, hipStream_t stream) {
    hipLaunchKernelGGL(dv_kv_select, dim3((unsigned)(p.W * p.Hkv)), dim3(kSelThreads), 0, stream, p);
    return hipGetLastError();
}

// ---- compaction -----------------------------------------------------------------
//
// Row first + i of a sequence and KV head takes what row first + rows[i] held, for
// every i with rows[i] >= i (others stay as they are); mass entries move alike, and
// those of rows that nothing kept moves into become 0.  All in place: a block moves
// its rows in batches of ascending i, reading a whole batch before it writes one row
// of it.  A later batch reads rows[j] >= j, beyond every row that an earlier one
// wrote, so no copy of the cache is needed and nothing but a block barrier orders the
// reads and writes.
//
// Bound by memory: each moved row is read and written once.  The order within a
// sequence leaves one block per (sequence, KV head, keys or values), so a call of few
// of those also cuts the rows into column slices, which move independently.
namespace {
constexpr int kMoveThreads = 1024;
constexpr int kMoveRows = 8;  // rows per thread and batch
}  // namespace

template <typename VT>
__global__ __launch_bounds__(kMoveThreads) void dv_kv_compact(const CompactParams p, int k_vecs, int v_vecs,
                                                              int vec_elems, int es) {
    const int tid = threadIdx.x;
    const int parts = 2 * p.slices + (p.mass ? 1 : 0);
    const int part = blockIdx.x % parts;
    const int wh = blockIdx.x / parts;
    const int w = wh / p.Hkv, h = wh - w * p.Hkv;
    const long long first = p.first[w];
    if (first < 0) return;
    const int limit = p.lengths ? p.lengths[w] : 0x7fffffff;  // rows of the range
    const int* rows = p.rows + ((long long)w * p.heads + (p.heads > 1 ? h : 0)) * p.N;

    if (part == 2 * p.slices) {
        // mass: entries of [first, first + limit), those without a kept row cleared
        float* mass = p.mass + ((long long)w * p.Hkv + h) * p.C;
        const long long cap = p.C - first;
        const int end = (int)(limit < cap ? limit : cap);  // negative: nothing
        for (int i0 = 0; i0 < end; i0 += kMoveThreads * 4) {
            float x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + u * kMoveThreads + tid;
                x[u] = 0.0f;
                if (i < end && i < p.N) {
                    const int r = rows[i];
                    if (r >= i && r < end) x[u] = mass[first + r];
                }
            }
            wait_vmcnt<0>();
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + u * kMoveThreads + tid;
                if (i < end) mass[first + i] = x[u];
            }
        }
        return;
    }
    const bool is_v = part >= p.slices;
    const int slice = is_v ? part - p.slices : part;
    const int vecs = is_v ? v_vecs : k_vecs;  // vectors of a row
    if (vecs == 0) return;
    const long long* st = is_v ? p.vcs : p.kcs;
    unsigned char* cache = reinterpret_cast<unsigned char*>(is_v ? p.vc : p.kc) + (long long)h * st[2] * es;
    const int c0 = vecs * slice / p.slices, c1 = vecs * (slice + 1) / p.slices;
    const int lanes = c1 - c0;  // vectors of this slice; the launcher keeps it at most kMoveThreads
    if (lanes == 0) return;
    const int per = kMoveThreads / lanes;  // rows moved side by side
    const int lane = tid % lanes, sub = tid / lanes;
    const bool active = sub < per;
    const long long col = (long long)(c0 + lane) * vec_elems;
    const int* bt = p.bt + (long long)w * p.maxB;
    // address of a row's vector, null where it lies on no valid page
    auto at = [&](long long row) -> VT* {
        const long long lp = row / p.bs;
        if (lp >= p.maxB) return nullptr;
        const int page = bt[lp];
        if (page < 0 || page >= p.nblocks) return nullptr;
        return reinterpret_cast<VT*>(cache + (page * st[0] + (row - lp * p.bs) * st[1] + col) * es);
    };
    const int batch = per * kMoveRows;
    for (int i0 = 0; i0 < p.N; i0 += batch) {
        VT x[kMoveRows];
        VT* dst[kMoveRows];
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const int i = i0 + u * per + sub;
            dst[u] = nullptr;
            if (active && i < p.N) {
                const int r = rows[i];
                if (r > i && r < limit) {  // r == i: the row is there already
                    const VT* src = at(first + r);
                    if (src) {
                        dst[u] = at(first + i);
                        if (dst[u]) x[u] = *src;
                    }
                }
            }
        }
        wait_vmcnt<0>();  // this thread's rows are here before any thread writes one
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u)
            if (dst[u]) *dst[u] = x[u];
    }
}

hipError_t launch_kv_compact(int dtype, const CompactParams& base, hipStream_t stream) {
    CompactParams p = base;
    const int es = dtype == kF32 ? 4 : 2;
    auto al = [](const void* ptr) { return ((uintptr_t)ptr & 15) == 0; };
    bool vec = al(p.kc) && al(p.vc) && (p.E * es) % 16 == 0 && (p.Ev * es) % 16 == 0;
    for (int i = 0; i < 3; ++i) vec = vec && (p.kcs[i] * es) % 16 == 0 && (p.vcs[i] * es) % 16 == 0;
    const int elems = vec ? 16 / es : 1;
    const int kv = p.E / elems, vv = p.Ev / elems;
    const int widest = kv > vv ? kv : vv;
    // slices of at least 128 bytes until the call has 256 blocks, and as many as a
    // block's threads need
    int slices = 1;
    while (slices < widest && ((long long)p.W * p.Hkv * 2 * slices < 256 && widest * elems * es / (2 * slices) >= 128))
        slices *= 2;
    while ((widest + slices - 1) / slices > kMoveThreads) slices *= 2;
    p.slices = slices;
    const dim3 grid((unsigned)(p.W * p.Hkv * (2 * slices + (p.mass ? 1 : 0)))), block(kMoveThreads);
    if (vec) hipLaunchKernelGGL(dv_kv_compact<u32x4>, grid, block, 0, stream, p, kv, vv, elems, es);
    else if (es == 4) hipLaunchKernelGGL(dv_kv_compact<uint32_t>, grid, block, 0, stream, p, kv, vv, 1, es);
    else hipLaunchKernelGGL(dv_kv_compact<uint16_t>, grid, block, 0, stream, p, kv, vv, 1, es);
    return hipGetLastError();
}

}  // namespace dv
