// Bounded caches: which rows to keep (dv_kv_select) and their move together
// (dv_kv_compact).
#include "dv_common.h"
#include "dv_device.h"

namespace dv {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kBins = 1 << 13;
// Rows per thread held in registers: an instance for capacities of up to 4096 rows,
// whose code is short, and one for the others.
constexpr int kSelHeldFew = 4, kSelHeldMany = 32;
constexpr int kSelList = 4096;  // rows that share T's first digit, held in LDS

// Weights as integers in their order; a NaN is lighter than any number, and 0 is left
// for lanes without a row.
__device__ inline uint32_t order_of(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 1u;
    if ((u & 0x7fffffffu) == 0u) return 0x80000000u;  // -0 and +0 weigh the same
    return (u >> 31) ? ~u : u | 0x80000000u;
}

// Set bits of a wave's mask below this lane.
__device__ inline int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// Exclusive sum of v over the block's threads.
__device__ inline int block_excl(int v, int* s_wave) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int o = __shfl_up(incl, d, kWave);
        if (lane >= d) incl += o;
    }
    if (lane == 63) s_wave[wv] = incl;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) before += i < wv ? s_wave[i] : 0;
    return before + incl - v;
}

}  // namespace

// Block = (sequence, KV head).  Of the n rows, the first keep_first and the last
// keep_last stay, and of those between the `need` heaviest: the weight T of the
// need-th is found digit by digit (a histogram of the digit over the rows that
// agree with T so far, most significant first), then the rows above T and the first
// of those equal to it (ties go to the lowest row) are written in ascending order.
// A wave owns a contiguous stretch of rows, so its places follow from one count per
// wave and a running one inside it, and no pass has a barrier in its loop.  Up to
// kSelHeld * 1024 rows are read once and held in registers; more are read again
// (from L2) in each of the five passes.  Bound by the chain of passes, and a list has one
// block: 1000 rows 7.2 us; 128 lists of 32768 rows 25.4, with half of the CUs idle.
template <int kSelHeld>
__global__ __launch_bounds__(kSelThreads) void dv_kv_select(const SelectParams p) {
    __shared__ int s_hist[kBins];
    __shared__ uint32_t s_list[kSelList];
    __shared__ int s_wave[kSelWaves], s_gt[kSelWaves], s_eq[kSelWaves];
    __shared__ int s_digit, s_above, s_listed;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = uniform(tid >> 6);
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
    const int a = p.keep_first, m = n - p.keep_last - a;  // rows [a, a + m) compete
    const int need = p.budget - p.keep_first - p.keep_last;
    const float* mass = p.mass + (long long)blockIdx.x * p.C + first + a;
    for (int i = tid; i < a; i += kSelThreads) rows[i] = i;
    for (int i = tid; i < p.keep_last; i += kSelThreads) rows[a + need + i] = a + m + i;
    if (need == 0) return;

    const int steps = (m + kSelThreads - 1) / kSelThreads;  // of 64 rows per wave
    const int base = wv * steps * kWave + lane;
    const bool held = steps <= kSelHeld;
    uint32_t key[kSelHeld];
    if (held) {
        float x[kSelHeld];
#pragma unroll
        for (int j = 0; j < kSelHeld; ++j) {
            x[j] = 0.0f;
            if (j < steps && base + j * kWave < m) x[j] = mass[base + j * kWave];
        }
#pragma unroll
        for (int j = 0; j < kSelHeld; ++j) {
            key[j] = 0u;
            if (j < steps) key[j] = base + j * kWave < m ? order_of(x[j]) : 0u;
        }
    }
    // fn(weight, the row) for the wave's rows in order (weight 0: no row)
    auto visit = [&](auto&& fn) {
        if (held) {
#pragma unroll
            for (int j = 0; j < kSelHeld; ++j) {
                if (j >= steps) break;
                fn(key[j], base + j * kWave);
            }
        } else {
            for (int j0 = 0; j0 < steps; j0 += 8) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = base + (j0 + j) * kWave;
                    x[j] = 0.0f;
                    if (j0 + j < steps && i < m) x[j] = mass[i];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = base + (j0 + j) * kWave;
                    if (j0 + j < steps) fn(i < m ? order_of(x[j]) : 0u, i);
                }
            }
        }
    };

    // Bits of a weight resolved per pass.  A wide first digit (sign, exponent, four bits of
    // the fraction) spreads weights of a few octaves over a hundred bins and more,
    // where lanes of a wave rarely meet in one (an LDS atomic serialises those); clearing
    // and summing its bins costs a short call more than that saves.  Lanes without a
    // row count in the lowest bin, which no heavier weight's place depends on.
    const int bits0 = m <= 4096 ? 11 : 13, bits1 = m <= 4096 ? 11 : 10;
    uint32_t top = 0;   // T's digits so far
    int want = need;    // of the rows that agree with them, how many stay
    int shift = 32;
    bool listed = false;  // the rows that agree with them are in the list
    if (tid == 0) s_listed = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const uint32_t known = pass == 0 ? 0u : ~0u << shift;
        const int bits = pass == 0 ? bits0 : pass == 1 ? bits1 : shift;
        shift -= bits;
        const int bins = 1 << bits;
        for (int i = tid; i < bins; i += kSelThreads) s_hist[i] = 0;
        if (pass == 1 && steps > 8) {
            // the few rows that share T's first digit go to the list, as far as it holds
            // them: less to go through than all rows, if those are many
            visit([&](uint32_t u, int) {
                const uint64_t same = ballot((u & known) == top);
                if (same) {
                    int at = 0;
                    if (lane == 0) at = atomicAdd(&s_listed, __builtin_popcountll(same));
                    at = uniform(at) + lanes_below(same);
                    if ((u & known) == top && at < kSelList) s_list[at] = u;
                }
            });
        }
        __syncthreads();
        if (pass == 1 && steps > 8) listed = s_listed <= kSelList;
        auto count = [&](uint32_t u) {
            if ((u & known) == top) atomicAdd(&s_hist[(u >> shift) & (uint32_t)(bins - 1)], 1);
        };
        if (listed)
            for (int i = tid; i < s_listed; i += kSelThreads) count(s_list[i]);
        else
            visit([&](uint32_t u, int) { count(u); });
        __syncthreads();
        // the digit whose rows hold the want-th heaviest: a thread owns `per` bins,
        // counted from the heaviest
        const int per = bins > kSelThreads ? bins / kSelThreads : 1;
        const int b0 = bins - 1 - per * tid;  // negative: none
        int sum = 0;
        for (int i = 0; i < per; ++i) sum += b0 - i >= 0 ? s_hist[b0 - i] : 0;
        int before = block_excl(sum, s_wave);
        if (before < want && want <= before + sum) {
            int i = 0;
            while (before + s_hist[b0 - i] < want) before += s_hist[b0 - i++];
            s_digit = b0 - i;
            s_above = before;
        }
        __syncthreads();
        top |= (uint32_t)s_digit << shift;
        want -= s_above;
    }

    // rows above T and equal to it, per wave and then before each wave
    int gts = 0, eqs = 0;
    visit([&](uint32_t u, int) {
        gts += __builtin_popcountll(ballot(u > top));
        eqs += __builtin_popcountll(ballot(u == top));
    });
    if (lane == 0) {
        s_gt[wv] = gts;
        s_eq[wv] = eqs;
    }
    __syncthreads();
    gts = eqs = 0;
    for (int i = 0; i < wv; ++i) {
        gts += s_gt[i];
        eqs += s_eq[i];
    }
    // rows kept before the wave's next one; of the equal rows, the first `want` are
    int kept = gts + (eqs < want ? eqs : want);
    int* out = rows + a;
    visit([&](uint32_t u, int i) {
        uint64_t keep = ballot(u > top);
        const uint64_t eq = ballot(u == top);
        if (eq) {
            const int left = want - eqs;
            keep |= left > 0 ? ballot(u == top && lanes_below(eq) < left) : 0ull;
            eqs += __builtin_popcountll(eq);
        }
        if ((keep >> lane) & 1ull) out[kept + lanes_below(keep)] = a + i;
        kept += __builtin_popcountll(keep);
    });
}

hipError_t launch_kv_select(const SelectParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)(p.W * p.Hkv)), block(kSelThreads);
    if (p.C <= kSelHeldFew * kSelThreads) hipLaunchKernelGGL(dv_kv_select<kSelHeldFew>, grid, block, 0, stream, p);
    else hipLaunchKernelGGL(dv_kv_select<kSelHeldMany>, grid, block, 0, stream, p);
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
constexpr int kMoveThreads = 512;
constexpr int kMoveRows = 8;                                    // rows per thread and batch
constexpr int kMoveBatch = kMoveThreads;                        // rows per batch, at most
constexpr int kMoveSide = kMoveBatch / kMoveRows;               // rows side by side, at most
struct Move {
    long long src, dst;  // byte offsets of a row's head; src < 0: nothing to move
};
}  // namespace

// Where the rows of a batch lie is worked out by one thread per row (into LDS), for
// the next batch while this one's rows are on their way; the rows of the next batch
// are asked for before this one's are written.
template <typename VT>
__global__ __launch_bounds__(kMoveThreads) void dv_kv_compact(const CompactParams p, int k_vecs, int v_vecs,
                                                              int vec_bytes, int es) {
    __shared__ Move s_move[3][kMoveBatch];  // three: a batch's is read until its rows are written
    const int tid = threadIdx.x;
    const int parts = 2 * p.slices + (p.mass ? 1 : 0);
    const int part = blockIdx.x % parts;
    const int wh = blockIdx.x / parts;
    const int w = wh / p.Hkv, h = wh - w * p.Hkv;
    const int first = p.first[w];
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
    const int c0 = vecs * slice / p.slices, c1 = vecs * (slice + 1) / p.slices;
    const int lanes = c1 - c0;  // vectors of this slice; the launcher keeps it at most kMoveThreads
    if (lanes == 0) return;
    const long long s0 = is_v ? p.vcs[0] : p.kcs[0], s1 = is_v ? p.vcs[1] : p.kcs[1];
    unsigned char* cache = reinterpret_cast<unsigned char*>(is_v ? p.vc : p.kc) +
                           (long long)h * (is_v ? p.vcs[2] : p.kcs[2]) * es;
    const int fit = kMoveThreads / lanes;
    const int per = fit < kMoveSide ? fit : kMoveSide;  // rows moved side by side
    const int lane = tid % lanes, sub = tid / lanes;
    const bool active = sub < per;
    unsigned char* col = cache + (long long)(c0 + lane) * vec_bytes;
    const int* bt = p.bt + (long long)w * p.maxB;
    const int batch = per * kMoveRows;

    // byte offset of a stream row (below 2^32: two ints), negative on no valid page
    auto at = [&](uint32_t row) -> long long {
        uint32_t lp, in;
        if (p.bs_shift >= 0) {
            lp = row >> p.bs_shift;
            in = row & ((1u << p.bs_shift) - 1u);
        } else {
            lp = row / (uint32_t)p.bs;
            in = row - lp * (uint32_t)p.bs;
        }
        if (lp >= (uint32_t)p.maxB) return -1;
        const int page = bt[lp];
        if (page < 0 || page >= p.nblocks) return -1;
        return (page * s0 + (long long)in * s1) * es;
    };
    auto plan = [&](int i0, Move* to) {
        if (tid >= batch) return;
        const int i = i0 + tid;
        Move m{-1, -1};
        if (i < p.N) {
            const int r = rows[i];
            if (r > i && r < limit) {  // r == i: the row is there already
                m.dst = at((uint32_t)first + (uint32_t)i);
                if (m.dst >= 0) m.src = at((uint32_t)first + (uint32_t)r);
            }
        }
        to[tid] = m;
    };
    auto fetch = [&](const Move* from, VT (&x)[kMoveRows]) {
        if (!active) return;
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const long long src = from[u * per + sub].src;
            if (src >= 0) x[u] = *reinterpret_cast<const VT*>(col + src);
        }
    };
    VT x[2][kMoveRows];
    plan(0, s_move[0]);
    __syncthreads();
    fetch(s_move[0], x[0]);
    int t = 0;  // the batch's table
    auto step = [&](int i0, const int cur) {
        const bool more = i0 + batch < p.N;
        const Move* now = s_move[t];
        t = t == 2 ? 0 : t + 1;
        if (more) plan(i0 + batch, s_move[t]);
        wait_vmcnt<0>();  // this thread's rows are here before any thread writes one
        __syncthreads();
        if (more) fetch(s_move[t], x[cur ^ 1]);
        if (!active) return;
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const Move m = now[u * per + sub];
            if (m.src >= 0) *reinterpret_cast<VT*>(col + m.dst) = x[cur][u];
        }
    };
    for (int i0 = 0; i0 < p.N; i0 += 2 * batch) {
        step(i0, 0);
        if (i0 + batch < p.N) step(i0 + batch, 1);
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
    // slices of at least 128 bytes while the call has fewer than 512 blocks, two per CU (16
    // sequences, 8 KV heads, 4096 of 8100 rows kept: 112-118 us, with 256 blocks 132, of 1024
    // threads 132) -- a 16-bit row of 128 is two slices at most, so fewer than 128 (sequence,
    // KV head) pairs stay below that -- and as many as a block's threads need
    int slices = 1;
    while (slices < widest && ((long long)p.W * p.Hkv * 2 * slices < 512 && widest * elems * es / (2 * slices) >= 128))
        slices *= 2;
    while ((widest + slices - 1) / slices > kMoveThreads) slices *= 2;
    p.slices = slices;
    const dim3 grid((unsigned)(p.W * p.Hkv * (2 * slices + (p.mass ? 1 : 0)))), block(kMoveThreads);
    if (vec) hipLaunchKernelGGL(dv_kv_compact<u32x4>, grid, block, 0, stream, p, kv, vv, 16, es);
    else if (es == 4) hipLaunchKernelGGL(dv_kv_compact<uint32_t>, grid, block, 0, stream, p, kv, vv, es, es);
    else hipLaunchKernelGGL(dv_kv_compact<uint16_t>, grid, block, 0, stream, p, kv, vv, es, es);
    return hipGetLastError();
}

}  // namespace dv
