// Attention weight that every cached key receives (dvattn_paged_key_mass):
//   out[w, h, c] = decay * mass[w, h, c]
//                + sum over tokens s and the 16 query heads n of KV head h of
//                  2^(x_{s,n,c} - lse_{s,n}),
// x the base-2 scores of the key in stream row c (rotated query of c's view), lse the
// base-2 log-sum-exp of row (s, n) over its visible keys.  The weights need the sums
// over all keys first, so the keys are passed twice: a first kernel leaves every
// row's (max, sum) over each part of the keys, the second joins them and adds the
// weights up.
//
// K rows are the A operand of S^T = K Q^T (16x16x32 MFMA, 16x16x4 for fp32), held in
// registers while the tokens go by: with no second product there is nothing else to
// do with them.  Every K row is read once per pass however many tokens vote, and a
// key's weight is summed in a fixed order -- no atomics, the same bits from every run.
// Scores, maxima, sums and weights are fp32.
//
//  * S = 1 (a decode step; bound by memory): the queries are rotated in the kernel
//    and the scores stored (64 bytes per key and KV head, a quarter of a 16-bit K row, an
//    eighth of an fp32 one), so the second pass reads those and not K.
//  * S > 1 (a window of tokens; bound by waits and issue, see dv_mass_stats): a wave holds 64 keys (32
//    for fp32) and walks the tokens, whose queries one launch beforehand rotated into
//    the MFMA's operand order; the second pass computes the scores again (storing
//    them would cost more bytes than K from two tokens on).  Over few keys, where that
//    walk is all a call's time, the waves of a block share the tokens (dv_mass_small).
//    A launch takes at most kMassTokens tokens, which bounds the pairs (max, sum) in the
//    workspace; the rotated queries in it are those of all tokens and views.
#include <type_traits>

#include "dv_common.h"
#include "dv_device.h"

namespace dv {

namespace {

constexpr int kMassWaves = 4;
constexpr int kMassThreads = kMassWaves * kWave;
constexpr int kSmallWaves = 8;      // of a block that shares its tokens among them
constexpr int kSmallThreads = kSmallWaves * kWave;
constexpr int kMaxUnits = 4;        // S = 1: units of keys per wave
constexpr int kMassTokens = kWave;  // one lane per token holds what it sees

// 16-byte pieces of a K row per lane: lane (g, n) of a 16-key tile holds bytes
// cc * 64 + g * 16 of key n's row, for both operands alike (the order of the dims in a
// dot product does not matter as long as both agree).
template <int DT> constexpr int kPieces = kHeadDim * Tr<DT>::kBytes / 64;
template <int DT> constexpr int kOperandBytes = kPieces<DT> * kWave * 16;  // one token's 16 heads
// 16-key tiles per wave: 64 registers of K
template <int DT> constexpr int kTilesOf = DT == kF32 ? 2 : 4;

// Scores of NT tiles: piece by piece over all tiles, so that consecutive MFMAs do not
// wait for each other's result.
template <int DT, int NT>
__device__ inline void dot_tiles(const u32x4 (&k)[NT][kPieces<DT>], const u32x4 (&q)[kPieces<DT>], f32x4 (&x)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) x[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int cc = 0; cc < kPieces<DT>; ++cc) {
        if constexpr (DT == kF32) {
            const f32x4 qf = __builtin_bit_cast(f32x4, q[cc]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    x[t] = Tr<kF32>::mma1(__builtin_bit_cast(f32x4, k[t][cc])[j], qf[j], x[t]);
        } else {
#pragma unroll
            for (int t = 0; t < NT; ++t) x[t] = Tr<DT>::mma(k[t][cc], q[cc], x[t]);
        }
    }
}

__device__ inline int view_len(const MassParams& p, int f) { return p.fl[f] > 0 ? p.fl[f] : 0; }

// Keys of view f that token s of sequence w sees.
__device__ inline int seen_of(const MassParams& p, int f, int w, int s, int len) {
    const long long l = (long long)p.loc[((long long)f * p.W + w) * p.S + s] + 1;
    return l <= 0 ? 0 : l < len ? (int)l : len;
}

// What each of the launch's tokens sees of view f, token s0 + i in lane i (0 past the last).
__device__ inline int seen_lane(const MassParams& p, int f, int w, int len) {
    const int lane = threadIdx.x & 63;
    return lane < p.ns ? seen_of(p, f, w, p.s0 + lane, len) : 0;
}

__device__ inline int lanes_max(int v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const int o = __shfl_xor(v, d, kWave);
        v = o > v ? o : v;
    }
    return uniform(v);
}

__device__ inline int seen_most(const MassParams& p, int f, int w, int len) {
    return p.ns == 1 ? uniform(seen_of(p, f, w, p.s0, len)) : lanes_max(seen_lane(p, f, w, len));
}

// One past the last stream row that some token of the launch sees in sequence w.
__device__ inline long long visible_end(const MassParams& p, int w) {
    long long off = 0, end = 0;
    for (int f = 0; f < p.F; ++f) {
        const int len = view_len(p, f);
        const int v = seen_most(p, f, w, len);
        if (v > 0) end = off + v;
        off += len;
    }
    const long long rows = (long long)p.maxB * p.bs;
    return end < rows ? end : rows;
}

// Index of the cache row (token, KV head) of stream row c, or -1 (as 32 bits) if it
// lies on no valid page; want: the row is needed at all.
__device__ inline uint32_t cache_row(const MassParams& p, int w, int hkv, long long c, bool want) {
    uint32_t lp, in;
    const uint32_t u = (uint32_t)c;
    want = want && c <= (long long)UINT32_MAX;  // rows past the block table end at 2^32 at most
    if (p.bs_shift >= 0) {
        lp = u >> p.bs_shift;
        in = u & ((1u << p.bs_shift) - 1u);
    } else {
        lp = u / (uint32_t)p.bs;
        in = u - lp * (uint32_t)p.bs;
    }
    int page = -1;
    if (want && lp < (uint32_t)p.maxB) page = p.bt[(long long)w * p.maxB + lp];
    return page >= 0 && page < p.nblocks ? ((uint32_t)page * (uint32_t)p.bs + in) * (uint32_t)p.Hkv + (uint32_t)hkv
                                         : 0xffffffffu;
}

// K rows of NT tiles: lane i holds the cache row of key i (lanes past NT * 16: none).
// Rows without one are zeros and never read.
template <int DT, int NT>
__device__ inline void load_keys(const MassParams& p, uint32_t row, u32x4 (&k)[NT][kPieces<DT>]) {
    const int lane = threadIdx.x & 63;
    const unsigned char* base = reinterpret_cast<const unsigned char*>(p.kc) + (lane >> 4) * 16;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t r = (uint32_t)__shfl((int)row, t * 16 + (lane & 15), kWave);
#pragma unroll
        for (int cc = 0; cc < kPieces<DT>; ++cc) k[t][cc] = u32x4{0u, 0u, 0u, 0u};
        if (r != 0xffffffffu) {
            const unsigned char* src = base + (unsigned long long)r * (kHeadDim * Tr<DT>::kBytes);
#pragma unroll
            for (int cc = 0; cc < kPieces<DT>; ++cc) k[t][cc] = ld16(src + cc * 64);
        }
    }
}

// The first n of NT * 16 keys as bits.
template <int NT>
__device__ inline uint64_t first_keys(int n) {
    return n <= 0 ? 0ull : ~0ull >> (64 - n);
}
template <int NT> constexpr uint64_t kAllKeys = ~0ull >> (64 - NT * 16);

// Scheduling of a region of `mfmas` matrix instructions and the VALU work of one token:
// one of the former, six of the latter.
template <int mfmas>
__device__ inline void interleave() {
#pragma unroll
    for (int i = 0; i < (mfmas < 16 ? mfmas : 16); ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, mfmas < 16 ? 1 : mfmas / 16, 0);  // MFMA
        __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);                            // VALU
    }
}

// Bits 0-3: keys t * 16 + g * 4 + i of a mask, for this lane's g.
__device__ inline uint32_t lane_bits(uint64_t mask, int t) {
    return (uint32_t)(mask >> (t * 16 + ((threadIdx.x & 63) >> 4) * 4)) & 15u;
}

// Raw scores -> base-2, -inf outside the mask.
template <int NT>
__device__ inline void scale_masked(f32x4 (&x)[NT], uint64_t mask, float l2) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t b = lane_bits(mask, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[t][i] = ((b >> i) & 1u) ? x[t][i] * l2 : -DV_INF;
    }
}

// Piece `piece` (cc * 64 + lane) of the rotated query operand of (view, sequence, KV
// head, token).
template <int DT>
__device__ inline u32x4 rotated_piece(const MassParams& p, int f, int w, int hkv, int s, int piece) {
    using raw = typename Tr<DT>::raw;
    constexpr int N = 16 / Tr<DT>::kBytes;
    const int cc = piece >> 6, g = (piece >> 4) & 3, n = piece & 15;
    const raw* qrow = reinterpret_cast<const raw*>(p.q) + (((long long)w * p.Hq + hkv * kGqa + n) * p.S + s) * kHeadDim;
    const long long cs = (((long long)f * p.W + w) * p.S + s) * p.R;
    raw r[N];
    rotate_run<DT, N>(qrow, p.cosv + cs, p.sinv + cs, p.R, (cc * 64 + g * 16) / Tr<DT>::kBytes, r);
    u32x4 v;
    __builtin_memcpy(&v, r, 16);
    return v;
}

struct Item {
    int w, hkv;
    long long chunk, wh;
};

// Blocks: KV heads fastest (they share pages), then sequences, then chunks of keys.
__device__ inline Item item_of(const MassParams& p) {
    Item it;
    const uint32_t b = blockIdx.x;
    it.hkv = (int)(b % (uint32_t)p.Hkv);
    const uint32_t r = b / (uint32_t)p.Hkv;
    it.w = (int)(r % (uint32_t)p.W);
    it.chunk = r / (uint32_t)p.W;
    it.wh = (long long)it.w * p.Hkv + it.hkv;
    return it;
}

// (m, l) joined with (m2, l2).
__device__ inline void join(float& m, float& l, float m2, float l2) {
    const float mn = fmaxf(m, m2);
    const float mz = mn == -DV_INF ? 0.0f : mn;
    l = l * __builtin_amdgcn_exp2f(m - mz) + l2 * __builtin_amdgcn_exp2f(m2 - mz);
    m = mn;
}

// Minus the log-sum-exp; -inf where no key is seen, so that 2^(x + it) is 0.
__device__ inline float minus_lse(float m, float l) { return l == 0.0f ? -DV_INF : -(m + log2f(l)); }

// That of head tid % 16 over `count` pairs (pair u of head n at pairs[u * 16 + n]), in
// every thread of the block.
__device__ inline float joined_lse(const float2* pairs, long long count, float2 (&s_pair)[kMassThreads]) {
    const int tid = threadIdx.x;
    const int n = tid & 15;
    float m = -DV_INF, l = 0.0f;
    for (long long u = tid >> 4; u < count; u += kMassThreads / 16) {
        const float2 e = pairs[u * kGqa + n];
        join(m, l, e.x, e.y);
    }
    s_pair[tid] = make_float2(m, l);
    __syncthreads();
    m = -DV_INF;
    l = 0.0f;
#pragma unroll
    for (int u = 0; u < kMassThreads / 16; ++u) join(m, l, s_pair[u * 16 + n].x, s_pair[u * 16 + n].y);
    return minus_lse(m, l);
}

// A weight: invisible keys (-inf) get none, whatever the row's sum is.
__device__ inline float weight(float x, float nl) { return x == -DV_INF ? 0.0f : __builtin_amdgcn_exp2f(x + nl); }

// out = decay * mass + acc summed over the 16 heads, for a unit's rows below `end` and C.
template <int NT>
__device__ inline void store_mass(const MassParams& p, long long wh, long long c0, long long end,
                                  const f32x4 (&acc)[NT]) {
    end = end < p.C ? end : p.C;
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, n = lane & 15;
    float old[NT];
    const long long c = c0 + g * 4 + n;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        old[t] = 0.0f;
        if (n < 4 && c + t * 16 < end && p.decay != 0.0f) old[t] = p.mass[wh * p.C + c + t * 16] * p.decay;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float mine = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = row16_sum(acc[t][i]);
            mine = n == i ? a : mine;
        }
        if (n < 4 && c + t * 16 < end) p.out[wh * p.C + c + t * 16] = old[t] + mine;
    }
}

// The same for rows [c0, c0 + n) that no token sees.
__device__ inline void store_decayed(const MassParams& p, long long wh, long long c0, int n) {
    if (p.out == p.mass && p.decay == 1.0f) return;
    const int lane = threadIdx.x & 63;
    for (int r = lane; r < n; r += kWave) {
        const long long c = c0 + r;
        if (c < p.C) {
            const long long at = wh * p.C + c;
            p.out[at] = p.decay == 0.0f ? 0.0f : p.mass[at] * p.decay;
        }
    }
}

}  // namespace

// S = 1.  Block: p.units * 4 * NT * 16 rows of one (sequence, KV head), a contiguous
// quarter for each wave.  Leaves the scores (tile by tile, as the lanes hold them) and,
// per block and head, (max, sum).
//
// K rows come through LDS: a wave copies 8 KiB at a time into one half of a ring of its
// own (whole rows per instruction) while it computes the other half; rows are
// XOR-swizzled by 16-byte pieces so that an operand read of sixteen rows meets
// different banks.  Loads straight into the operands' registers touch a row in four
// instructions of 64 bytes and ran 84 us on 32 sequences of 1k - 8k keys, 8 KV heads.
constexpr int kScoreBytes = 8192;
constexpr int kScoreRing = kMassWaves * 2 * kScoreBytes;

static __device__ __align__(16) unsigned char zero_row[kHeadDim * 4];

template <int DT, int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_scores(const MassParams p) {
    constexpr int kRowBytes = kHeadDim * Tr<DT>::kBytes;
    constexpr int kKeys = kScoreBytes / kRowBytes;          // keys per ring half
    constexpr int kTiles = kKeys / 16;
    constexpr int kLanes = kRowBytes / 16;                  // lanes that copy one row
    constexpr int kIds = kMaxUnits * NT * 16 / kWave;       // registers of cache rows
    static_assert(kIds * kWave == kMaxUnits * NT * 16, "whole registers of cache rows");
    extern __shared__ __align__(256) unsigned char ring[];
    __shared__ u32x4 s_q[kPieces<DT> * kWave];
    __shared__ float2 s_pair[kMassWaves][kGqa];
    const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const Item it = item_of(p);
    const long long end = visible_end(p, it.w);
    const int mine_rows = NT * 16 * p.units;  // of a wave
    const long long rows = (long long)kMassWaves * mine_rows;
    const long long b0 = it.chunk * rows;
    if (b0 >= end) return;
    const long long w0 = b0 + wv * mine_rows;
    // the wave's visible part
    const int keys = uniform((int)(end - w0 < mine_rows ? (end - w0 > 0 ? end - w0 : 0) : mine_rows));
    // whole units of NT tiles, as dv_mass_apply_scores reads them
    const int steps = (keys + NT * 16 - 1) / (NT * 16) * (NT * 16 / kKeys);
    unsigned char* mine = ring + wv * 2 * kScoreBytes;
    const uint32_t mine_at = lds_addr(mine);
    float m = -DV_INF, l = 0.0f;  // this lane's keys
    long long off = 0;
    bool first = true;            // no view's scores are stored yet
    for (int f = 0; f < p.F && off < b0 + rows && off < end; ++f) {
        const int len = view_len(p, f);
        const long long lo = off;
        off += len;
        if (off <= b0) continue;
        const long long hi = lo + uniform(seen_of(p, f, it.w, p.s0, len));
        uint32_t ids[kIds];
#pragma unroll
        for (int r = 0; r < kIds; ++r) {
            const long long c = w0 + r * kWave + lane;
            ids[r] = 0xffffffffu;
            if (r * kWave < keys) ids[r] = cache_row(p, it.w, it.hkv, c, r * kWave + lane < keys && c >= lo && c < hi);
        }
        if (!first) __syncthreads();  // the previous view's query is read
        for (int i = threadIdx.x; i < kPieces<DT> * kWave; i += kMassThreads)
            s_q[i] = rotated_piece<DT>(p, f, it.w, it.hkv, p.s0, i);
        // the page ids are here: no wait for them (for all loads, that is) among the copies
#pragma unroll
        for (int r = 0; r < kIds; ++r) asm volatile("" : "+v"(ids[r]));
        // ids of a step, from lane `at` on
        auto ids_of = [&](int step, int& at) {
            uint32_t v = ids[0];
#pragma unroll
            for (int r = 1; r < kIds; ++r) v = step * kKeys >= r * kWave ? ids[r] : v;
            at = step * kKeys & (kWave - 1);
            return v;
        };
        auto copy = [&](int step) {
            int at;
            const uint32_t v = ids_of(step, at);
#pragma unroll
            for (int i = 0; i < kScoreBytes / 1024; ++i) {
                const int row = i * (kWave / kLanes) + lane / kLanes;
                const uint32_t id = (uint32_t)__shfl((int)v, at + row, kWave);
                const unsigned char* src = id != 0xffffffffu ? reinterpret_cast<const unsigned char*>(p.kc) +
                                                                   (unsigned long long)id * kRowBytes
                                                             : zero_row;
                dma16(src + ((lane % kLanes) ^ (row & 15)) * 16,
                      __builtin_amdgcn_readfirstlane(mine_at + (uint32_t)((step & 1) * kScoreBytes + i * 1024)));
            }
        };
        if (steps > 0) copy(0);
        if (steps > 1) copy(1);
        __syncthreads();
        u32x4 q[kPieces<DT>];
#pragma unroll
        for (int cc = 0; cc < kPieces<DT>; ++cc) q[cc] = s_q[cc * kWave + lane];
        float* out = p.scores + (it.wh * p.nchunks * rows + w0) / 16 * (kWave * 4) + lane * 4;
        for (int step = 0; step < steps; ++step) {
            if (step + 1 < steps) wait_vmcnt<kScoreBytes / 1024>();  // all but the next step's copies
            else wait_vmcnt<0>();
            compiler_fence();
            u32x4 k[kTiles][kPieces<DT>];
            const unsigned char* half = mine + (step & 1) * kScoreBytes + n * kRowBytes;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int cc = 0; cc < kPieces<DT>; ++cc)
                    k[t][cc] = *reinterpret_cast<const u32x4*>(half + t * 16 * kRowBytes + ((cc * 4 + g) ^ n) * 16);
            f32x4 x[kTiles];
            dot_tiles<DT, kTiles>(k, q, x);
            int at;
            const uint32_t v = ids_of(step, at);
            const uint64_t mask = (ballot(v != 0xffffffffu) >> at) & kAllKeys<kTiles>;
            scale_masked<kTiles>(x, mask, p.l2scale);
            if (first) {
#pragma unroll
                for (int t = 0; t < kTiles; ++t) *reinterpret_cast<f32x4*>(out + t * kWave * 4) = x[t];
            } else {
                // rows of earlier views keep theirs
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    const uint32_t b = lane_bits(mask, t);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if ((b >> i) & 1u) out[t * kWave * 4 + i] = x[t][i];
                }
            }
            out += kTiles * kWave * 4;
            lds_wait();  // the half is read
            if (step + 2 < steps) copy(step + 2);
            float mx = -DV_INF;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) mx = fmaxf(mx, fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
            const float mn = fmaxf(m, mx);
            const float mz = mn == -DV_INF ? 0.0f : mn;
            l *= __builtin_amdgcn_exp2f(m - mz);
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(x[t][i] - mz);
            m = mn;
        }
        first = false;
    }
    // the lanes of a head, the waves
    const float mw = rows4_max(m);
    const float lw = rows4_sum(l * __builtin_amdgcn_exp2f(m - (mw == -DV_INF ? 0.0f : mw)));
    if (lane < kGqa) s_pair[wv][lane] = make_float2(mw, lw);
    __syncthreads();
    if (threadIdx.x < kGqa) {
        m = -DV_INF;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < kMassWaves; ++i) join(m, l, s_pair[i][threadIdx.x].x, s_pair[i][threadIdx.x].y);
        reinterpret_cast<float2*>(p.part)[(it.wh * p.nchunks + it.chunk) * kGqa + threadIdx.x] = make_float2(m, l);
    }
}

// Block: the same rows as above.
template <int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_apply_scores(const MassParams p) {
    __shared__ float2 s_pair[kMassThreads];
    constexpr int kRows = NT * 16;
    const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
    const Item it = item_of(p);
    const long long end = visible_end(p, it.w);
    const long long rows = (long long)kMassWaves * kRows * p.units;
    long long c0 = it.chunk * rows + wv * kRows;
    const float* src = p.scores + ((it.wh * p.nchunks * rows + c0) / 16 * kWave + lane) * 4;
    f32x4 x[NT];
    auto fetch = [&](long long c, const float* from) {
        if (c < end)
#pragma unroll
            for (int t = 0; t < NT; ++t) x[t] = ld16f_nt(from + t * kWave * 4);
    };
    fetch(c0, src);  // on its way while the block's heads' sums are joined
    float nl = 0.0f;
    if (it.chunk * rows < end)
        nl = joined_lse(reinterpret_cast<const float2*>(p.part) + it.wh * p.nchunks * kGqa, (end + rows - 1) / rows,
                        s_pair);
    for (int u = 0; u < p.units; ++u) {
        const long long c = c0;
        c0 += kMassWaves * kRows;
        src += kMassWaves * NT * kWave * 4;
        if (c >= end) {
            store_decayed(p, it.wh, c, kRows);
            continue;
        }
        f32x4 acc[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = weight(x[t][i], nl);
        if (u + 1 < p.units) fetch(c0, src);
        store_mass<NT>(p, it.wh, c, p.C, acc);
    }
}

// S > 1 and few keys in all (a short cache, a single sequence): no launch fills the card,
// so a call costs the longest chain of one of its waves and not its work.  Here the chain
// is short: a block of eight waves takes up to NT * 16 stream rows of one view (parts cut
// across views' borders went through them one after the other: 33 tokens on two views of
// 100 keys 32 us), every wave holds all of their K rows and takes every eighth token.  The
// first launch leaves (max, sum) per block, token and head; the second joins them (each
// wave for its own tokens, eight blocks' pairs loaded together: one after the other took
// up to 20 us of a call's 49), adds the weights over its tokens, and the waves' shares in
// order.  The K rows come through LDS: eight waves that each load them into registers
// cost 0.5 us per wave.
template <int DT, int NT, bool APPLY>
__global__ __launch_bounds__(kSmallThreads) void dv_mass_small(const MassParams p) {
    constexpr int kRows = NT * 16;
    constexpr int kRowBytes = kHeadDim * Tr<DT>::kBytes;
    constexpr int kLanes = kRowBytes / 16;                       // lanes that copy one row
    __shared__ __align__(256) unsigned char s_keys[kRows * kRowBytes];
    __shared__ float s_nl[APPLY ? kMassTokens : 1][kGqa];        // minus a token's log-sum-exp: its wave's own
    __shared__ float s_part[APPLY ? kSmallWaves : 1][kRows];
    const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
    const int n = lane & 15, S = p.ns;
    const Item it = item_of(p);
    // this block's rows: [c0, c0 + here) of view f, which starts at row off (the rows behind
    // the last view and below the capacity count as one more view)
    const long long rows = (long long)p.maxB * p.bs;             // keys lie below
    const long long limit = rows > p.C ? rows : p.C;             // and outputs
    int f = -1, len = 0, here = 0, count = 0;                    // count: of the views' blocks
    long long c0 = 0, off = 0, end = 0;
    for (int g = 0; g <= p.F && end < limit; ++g) {
        const long long lo = end;
        const long long all = g < p.F ? view_len(p, g) : limit - end;
        end += all;
        const long long left = all < limit - lo ? all : limit - lo;
        const int blocks = (int)((left + kRows - 1) / kRows);
        if (it.chunk >= count && it.chunk < count + blocks) {
            f = g;
            off = lo;
            len = (int)all;
            c0 = lo + (it.chunk - count) * kRows;
            here = lo + left - c0 < kRows ? (int)(lo + left - c0) : kRows;
        }
        if (g < p.F) count += blocks;
    }
    if (f < 0) return;
    float2* part = reinterpret_cast<float2*>(p.part) + it.wh * p.nchunks * S * kGqa;
    // keys of the block that each token sees, token i in lane i
    int ends = 0;
    if (f < p.F) {
        const long long below = seen_lane(p, f, it.w, len) - (c0 - off);
        ends = below < 0 ? 0 : below < here ? (int)below : here;
    }
    const int most = lanes_max(ends);
    const uint32_t row = cache_row(p, it.w, it.hkv, c0 + lane, lane < most);
    const uint64_t valid = ballot(row != 0xffffffffu);
    if (!valid) {
        if constexpr (APPLY) {
            if (wv == 0) store_decayed(p, it.wh, c0, here);
        } else {
            for (int i = threadIdx.x; i < S * kGqa && f < p.F; i += kSmallThreads)
                part[it.chunk * S * kGqa + i] = make_float2(-DV_INF, 0.0f);
        }
        return;
    }
#pragma unroll
    for (int i = wv; i < kRows * kLanes / kWave; i += kSmallWaves) {
        const int r = i * (kWave / kLanes) + lane / kLanes;
        const uint32_t id = (uint32_t)__shfl((int)row, r, kWave);
        const unsigned char* src = id != 0xffffffffu ? reinterpret_cast<const unsigned char*>(p.kc) +
                                                           (unsigned long long)id * kRowBytes
                                                     : zero_row;
        dma16(src + ((lane % kLanes) ^ (r & 15)) * 16,
              __builtin_amdgcn_readfirstlane(lds_addr(s_keys) + (uint32_t)(i * 1024)));
    }
    u32x4 q[kPieces<DT>];
    const u32x4* ops = reinterpret_cast<const u32x4*>(p.rq) +
                       (((long long)f * p.W + it.w) * p.Hkv + it.hkv) * S * (kPieces<DT> * kWave) + lane;
    auto query = [&](int s) {
#pragma unroll
        for (int cc = 0; cc < kPieces<DT>; ++cc) q[cc] = ld16(ops + (s * kPieces<DT> + cc) * kWave);
    };
    if (wv < S) query(wv);
    if constexpr (APPLY) {
        constexpr int kBatch = 8;
        for (int s = wv; s < S; s += kSmallWaves) {
            float m = -DV_INF, l = 0.0f;
            for (int u0 = lane >> 4; u0 < count; u0 += 4 * kBatch) {
                float2 e[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int u = u0 + 4 * j;
                    e[j] = u < count ? part[((long long)u * S + s) * kGqa + n] : make_float2(-DV_INF, 0.0f);
                }
#pragma unroll
                for (int j = 0; j < kBatch; ++j) join(m, l, e[j].x, e[j].y);
            }
            const float mw = rows4_max(m);
            const float lw = rows4_sum(l * __builtin_amdgcn_exp2f(m - (mw == -DV_INF ? 0.0f : mw)));
            if (lane < kGqa) s_nl[s][n] = minus_lse(mw, lw);
        }
    }
    wait_vmcnt<0>();
    __syncthreads();
    u32x4 k[NT][kPieces<DT>];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int cc = 0; cc < kPieces<DT>; ++cc)
            k[t][cc] = *reinterpret_cast<const u32x4*>(s_keys + (t * 16 + n) * kRowBytes +
                                                       ((cc * 4 + (lane >> 4)) ^ n) * 16);
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s = wv; s < S; s += kSmallWaves) {
        const uint64_t mask = valid & first_keys<NT>(__builtin_amdgcn_readlane(ends, s));
        f32x4 x[NT];
        dot_tiles<DT, NT>(k, q, x);
        if (s + kSmallWaves < S) query(s + kSmallWaves);
        scale_masked<NT>(x, mask, p.l2scale);
        if constexpr (APPLY) {
            const float nl = s_nl[s][n];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] += weight(x[t][i], nl);
        } else {
            float mx = -DV_INF;
#pragma unroll
            for (int t = 0; t < NT; ++t) mx = fmaxf(mx, fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
            const float m = rows4_max(mx);
            const float mz = m == -DV_INF ? 0.0f : m;
            float l = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(x[t][i] - mz);
            l = rows4_sum(l);
            if (lane < kGqa) part[(it.chunk * S + s) * kGqa + n] = make_float2(m, l);
        }
    }
    if constexpr (APPLY) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = row16_sum(acc[t][i]);
                if (n == i) s_part[wv][t * 16 + (lane >> 4) * 4 + i] = a;
            }
        __syncthreads();
        const long long c = c0 + threadIdx.x;
        if (threadIdx.x < (unsigned)here && c < p.C) {
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < kSmallWaves; ++v) sum += s_part[v][threadIdx.x];
            const long long at = it.wh * p.C + c;
            p.out[at] = (p.decay == 0.0f ? 0.0f : p.mass[at] * p.decay) + sum;
        }
    }
}

// S > 1: the query operands, [F, W, Hkv, S] of kOperandBytes each, a thread per 16
// bytes; and, in the first `plans` blocks (W, or none), the plan.  A part is what one
// block of the kernels below takes: up to part_rows rows of one view (the rows behind the
// last view and below the capacity count as one more view, F).  The list of a sequence's parts
// has those that some token sees in front, and they get the first blocks of the
// launches that follow.  Both matter where a launch is about one block per CU: parts
// cut across the views' border took twice as long as the others (four sequences of
// two views, 4000 keys, 32 tokens, 4 KV heads: 52 us, one view 26), and blocks with
// nothing to do, strewn among the others, drew the blocks after them to the CUs that
// had them.
template <int DT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_prepare(const MassParams p, long long n, int plans,
                                                                int part_rows) {
    if (blockIdx.x >= (unsigned)plans) {
        const long long i = (long long)(blockIdx.x - plans) * kMassThreads + threadIdx.x;
        if (i >= n) return;
        constexpr int kPer = kPieces<DT> * kWave;
        const long long op = i / kPer;
        const int piece = (int)(i - op * kPer);
        const int s = (int)(op % p.S);
        const long long r = op / p.S;
        const int hkv = (int)(r % p.Hkv);
        const long long fw = r / p.Hkv;
        reinterpret_cast<u32x4*>(p.rq)[i] = rotated_piece<DT>(p, (int)(fw / p.W), (int)(fw % p.W), hkv, s, piece);
        return;
    }
    const int w = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6);
    int* seen = p.plan_seen + (long long)w * p.F;
    for (int f = wv; f < p.F; f += kMassWaves) {
        const int len = view_len(p, f);
        int best = 0;
        for (int s = lane; s < p.S; s += kWave) {
            const int v = seen_of(p, f, w, s, len);
            best = v > best ? v : best;
        }
        best = lanes_max(best);
        if (lane == 0) seen[f] = best;
    }
    __syncthreads();
    const long long rows = (long long)p.maxB * p.bs;       // keys lie below
    const long long limit = rows > p.C ? rows : p.C;       // and outputs
    int4* list = p.plan_list + (long long)w * p.nparts;
    // seen parts of the views before f, and other parts; the others go behind all seen ones
    auto seen_parts = [&](int f, long long off) {
        const long long left = rows - off;
        const long long keys = seen[f] < left ? seen[f] : left;
        return keys > 0 ? (int)((keys + part_rows - 1) / part_rows) : 0;
    };
    int count = 0;
    long long off = 0;
    for (int f = 0; f < p.F; ++f) {
        count += seen_parts(f, off);
        off += view_len(p, f);
    }
    int on = 0, idle = count;
    off = 0;
    for (int f = 0; f <= p.F && off < limit; ++f) {
        const long long len = f < p.F ? view_len(p, f) : limit - off;
        const long long here = len < limit - off ? len : limit - off;
        const int all = (int)((here + part_rows - 1) / part_rows);
        const int a = f < p.F ? seen_parts(f, off) : 0;
        for (int k = tid; k < all; k += kMassThreads)
            list[k < a ? on + k : idle + k - a] =
                make_int4(f, (int)(uint32_t)(off + (long long)k * part_rows), (int)(uint32_t)off, (int)len);
        on += a;
        idle += all - a;
        off += len;
    }
    if (tid == 0) {
        p.plan_count[w] = count;
        p.plan_count[p.W + w] = idle;
    }
}

namespace {

// The part of block blockIdx.x: parts that some token sees first (seen), in sequence
// order, KV heads fastest; index: its place in its sequence's list.
struct Part {
    int w, hkv, index;
    int f, len;          // view and its keys
    long long c0, off;   // first stream row of the part, and of the view
    long long wh;
    bool seen, any;
};

__device__ inline Part part_of(const MassParams& p) {
    const int lane = threadIdx.x & 63;
    Part it;
    it.hkv = (int)(blockIdx.x % (uint32_t)p.Hkv);
    long long r = blockIdx.x / (uint32_t)p.Hkv;
    it.any = false;
    for (int pass = 0; pass < 2 && !it.any; ++pass)
        for (int w0 = 0; w0 < p.W && !it.any; w0 += kWave) {
            const int w = w0 + lane;
            int base = 0, n = 0;
            if (w < p.W) {
                const int c = p.plan_count[w], all = p.plan_count[p.W + w];
                base = pass == 0 ? 0 : c;
                n = pass == 0 ? c : all - c;
            }
            int incl = n;
#pragma unroll
            for (int d = 1; d < kWave; d <<= 1) {
                const int o = __shfl_up(incl, d, kWave);
                if (lane >= d) incl += o;
            }
            const int total = __builtin_amdgcn_readlane(incl, 63);
            if (r < total) {
                const int l = __builtin_ctzll(ballot(incl > (int)r));
                it.w = w0 + l;
                it.seen = pass == 0;
                it.index = (int)r - __builtin_amdgcn_readlane(incl - n - base, l);
                it.any = true;
            }
            r -= total;
        }
    if (!it.any) return it;
    const int4 e = p.plan_list[(long long)it.w * p.nparts + it.index];
    it.f = uniform(e.x);
    it.c0 = (uint32_t)uniform(e.y);
    it.off = (uint32_t)uniform(e.z);
    it.len = uniform(e.w);
    it.wh = (long long)it.w * p.Hkv + it.hkv;
    return it;
}

// Tokens whose operands one ring half holds, staged together: a ring of 32 KiB lets as many
// blocks share a CU as their registers do (three).  One of 64 KiB, for two of them, took
// 20 % longer for fp32 at every size and up to 20 % for 16 bits where the parts did not
// fill the card evenly (but 5 % less where they did).
template <int DT> constexpr int kGroup = DT == kF32 ? 2 : 4;
template <int DT> constexpr int kRingBytes = 2 * kGroup<DT> * kOperandBytes<DT>;

// A seen part's keys (a unit per wave) against every token of the launch, kGroup tokens
// at a time: the operands of a group are copied to LDS, in turns by the waves (they
// lie in the order the waves read them), while the group before it is computed.
// prepare(s0) runs in every wave before the group of tokens s0 is waited for; body(s, x,
// all) gets token s's scores x: raw ones if it sees all of the unit (all, as a type),
// else base-2 ones with -inf for keys that it does not see (not called where it sees
// none); done(s0, n) runs in every wave after a group and may use block barriers.
//
// A group of tokens that see all of the unit (most of them) runs without masks, the
// MFMAs of the next token beside the exponentials of this one.
template <int DT, int NT, class Prepare, class Body, class Done>
__device__ inline void walk_tokens(const MassParams& p, const Part& it, unsigned char* ring, Prepare&& prepare,
                                   Body&& body, Done&& done) {
    constexpr int kRows = NT * 16;
    constexpr int kG = kGroup<DT>;
    const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
    const uint32_t ring_at = lds_addr(ring);
    const int groups = (p.ns + kG - 1) / kG;
    const unsigned char* ops = reinterpret_cast<const unsigned char*>(p.rq) +
                               ((((long long)it.f * p.W + it.w) * p.Hkv + it.hkv) * p.S + p.s0) * kOperandBytes<DT>;
    auto stage = [&](int gi) {
        const int n = p.ns - gi * kG < kG ? p.ns - gi * kG : kG;
        const uint32_t half = ring_at + (uint32_t)((gi & 1) * kG * kOperandBytes<DT>);
        for (int i = wv; i < n * kPieces<DT>; i += kMassWaves)
            dma16(ops + ((long long)gi * kG * kPieces<DT> + i) * 1024 + lane * 16,
                  __builtin_amdgcn_readfirstlane(half + (uint32_t)(i * 1024)));
    };
    stage(0);
    // keys of the unit before the end of what token s sees, in lane s
    const long long c0 = it.c0 + wv * kRows;
    const int before = (int)(c0 - it.off);  // the view's keys before the unit
    const int left = seen_lane(p, it.f, it.w, it.len) - before;
    const int ends = left < 0 ? 0 : left < kRows ? left : kRows;
    const int most = lanes_max(ends);
    const uint32_t row = cache_row(p, it.w, it.hkv, c0 + lane, lane < most);
    const uint64_t valid = ballot(row != 0xffffffffu);
    u32x4 k[NT][kPieces<DT>];
    load_keys<DT, NT>(p, row, k);
    // the keys are here before the token loop: a wait for them inside it would wait for the
    // next group's operands too (one counter for all loads)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int cc = 0; cc < kPieces<DT>; ++cc) asm volatile("" : "+v"(k[t][cc]));
    // tokens that see the whole unit
    const uint64_t whole = valid == kAllKeys<NT> ? ballot(ends == kRows) : 0ull;
    for (int gi = 0; gi < groups; ++gi) {
        const int t0 = gi * kG;
        const int n = p.ns - t0 < kG ? p.ns - t0 : kG;
        prepare(t0);
        wait_vmcnt<0>();
        __syncthreads();  // the group is here; every wave is done with the other half
        if (gi + 1 < groups) stage(gi + 1);
        const u32x4* half = reinterpret_cast<const u32x4*>(ring + (gi & 1) * kG * kOperandBytes<DT>) + lane;
        auto query = [&](int s, u32x4(&q)[kPieces<DT>]) {
#pragma unroll
            for (int cc = 0; cc < kPieces<DT>; ++cc) q[cc] = half[(s * kPieces<DT> + cc) * kWave];
        };
        if (n == kG && (uint32_t)((whole >> t0) & ((1u << kG) - 1u)) == (1u << kG) - 1u) {
            u32x4 q[kPieces<DT>];
            f32x4 x[NT], y[NT];
            query(0, q);
            dot_tiles<DT, NT>(k, q, x);
            query(1, q);
#pragma unroll 1
            for (int s = 0; s < kG; s += 2) {
                dot_tiles<DT, NT>(k, q, y);
                query(s + 2 < kG ? s + 2 : s, q);
                body(t0 + s, x, std::true_type{});
                interleave<NT * kPieces<DT>>();
                dot_tiles<DT, NT>(k, q, x);  // of the next pair; after the last one, not used
                query(s + 3 < kG ? s + 3 : s, q);
                body(t0 + s + 1, y, std::true_type{});
                interleave<NT * kPieces<DT>>();
            }
        } else if (valid) {
#pragma unroll 1
            for (int s = 0; s < n; ++s) {
                const uint64_t mask = valid & first_keys<NT>(__builtin_amdgcn_readlane(ends, t0 + s));
                if (!mask) continue;
                u32x4 q[kPieces<DT>];
                query(s, q);
                f32x4 x[NT];
                dot_tiles<DT, NT>(k, q, x);
                scale_masked<NT>(x, mask, p.l2scale);
                body(t0 + s, x, std::false_type{});
            }
        }
        done(t0, n);
    }
}

}  // namespace

// Per seen part, token of the launch and head, (max, sum): about 110 VALU instructions
// (maximum, 16 exponentials, sums) beside 16 MFMAs per token and wave.  Four sequences of
// 9000 keys in two views, 4 KV heads, 32 tokens in fp16: 46 us (0.4 PFLOP/s), dv_mass_apply
// 43.  By its counters a SIMD issues VALU instructions for 15 us of that and its matrix unit
// runs for 8.5; the waves wait for 41 % of their time (apply: 45 %), at the end of every
// group of four tokens and its barriers, and the 587 parts are two or three per CU.
template <int DT, int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_stats(const MassParams p) {
    __shared__ __align__(16) unsigned char ring[kRingBytes<DT>];
    __shared__ float2 s_pair[kMassWaves][kGroup<DT>][kGqa];
    const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6);
    const Part it = part_of(p);
    if (!it.any || !it.seen) return;
    float2* part = reinterpret_cast<float2*>(p.part) + (it.wh * p.ns * p.nchunks + it.index) * kGqa;
    const float l2 = p.l2scale;
    const float2 none = make_float2(-DV_INF, 0.0f);
    walk_tokens<DT, NT>(
        p, it, ring,
        [&](int) {
            // tokens that see none of the wave's keys (the wave's own entries, read before
            // the last group's end)
            for (int i = lane; i < kGroup<DT> * kGqa; i += kWave) s_pair[wv][i >> 4][i & 15] = none;
        },
        [&](int s, f32x4(&x)[NT], auto all) {
            constexpr bool kRaw = decltype(all)::value;
            // the largest base-2 score: of the largest raw one, or the smallest for a negative scale
            const bool flip = kRaw && l2 < 0.0f;
            float mx = -DV_INF;
            if (flip) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    mx = fmaxf(mx, fmaxf(fmaxf(-x[t][0], -x[t][1]), fmaxf(-x[t][2], -x[t][3])));
            } else {
#pragma unroll
                for (int t = 0; t < NT; ++t) mx = fmaxf(mx, fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
            }
            const float f = kRaw ? l2 : 1.0f;
            const float m = rows4_max(mx) * (flip ? -f : f);
            const float mz = m == -DV_INF ? 0.0f : m;
            float l = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][i], f, -mz));
            l = rows4_sum(l);
            if (lane < kGqa) s_pair[wv][s & (kGroup<DT> - 1)][lane] = make_float2(m, l);
        },
        [&](int t0, int n) {
            __syncthreads();
            for (int i = tid; i < n * kGqa; i += kMassThreads) {
                const int s = i >> 4, h = i & 15;
                float2 e = none;
#pragma unroll
                for (int v = 0; v < kMassWaves; ++v) join(e.x, e.y, s_pair[v][s][h].x, s_pair[v][s][h].y);
                part[(long long)(t0 + s) * p.nchunks * kGqa + h] = e;
            }
            __syncthreads();
        });
}

// Block (sequence, KV head, token): minus the log-sum-exp of its heads.
__global__ __launch_bounds__(kMassThreads) void dv_mass_lse(const MassParams p) {
    __shared__ float2 s_pair[kMassThreads];
    const long long row = blockIdx.x;  // (w * Hkv + hkv) * ns + s
    const int w = (int)(row / ((long long)p.ns * p.Hkv));
    const float nl =
        joined_lse(reinterpret_cast<const float2*>(p.part) + row * p.nchunks * kGqa, p.plan_count[w], s_pair);
    if (threadIdx.x < kGqa) p.lse[row * kGqa + threadIdx.x] = nl;
}

template <int DT, int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_apply(const MassParams p) {
    __shared__ __align__(16) unsigned char ring[kRingBytes<DT>];
    __shared__ float s_nl[2][kGroup<DT> * kGqa];
    constexpr int kRows = NT * 16;
    const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
    const Part it = part_of(p);
    if (!it.any) return;
    const long long c0 = it.c0 + wv * kRows, end = it.off + it.len;
    if (!it.seen) {
        store_decayed(p, it.wh, c0, end - c0 < kRows ? (int)(end - c0) : kRows);
        return;
    }
    const float* lse = p.lse + it.wh * p.ns * kGqa;
    const float l2 = p.l2scale;
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    walk_tokens<DT, NT>(
        p, it, ring,
        [&](int t0) {
            // the half that the group before this one does not read
            for (int i = threadIdx.x; i < kGroup<DT> * kGqa; i += kMassThreads)
                s_nl[(t0 / kGroup<DT>)&1][i] = t0 * kGqa + i < p.ns * kGqa ? lse[t0 * kGqa + i] : 0.0f;
        },
        [&](int s, f32x4(&x)[NT], auto all) {
            const float nl = s_nl[(s / kGroup<DT>)&1][(s & (kGroup<DT> - 1)) * kGqa + (lane & 15)];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (decltype(all)::value)
                        acc[t][i] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][i], l2, nl));
                    else
                        acc[t][i] += weight(x[t][i], nl);
                }
        },
        [](int, int) {});
    store_mass<NT>(p, it.wh, c0, end, acc);
}

// ---- launches --------------------------------------------------------------------

namespace {

int tiles_of(int dtype) { return dtype == kF32 ? kTilesOf<kF32> : kTilesOf<kBF16>; }

// Stored scores of a decode step take a quarter of a 16-bit K cache's bytes; block tables
// far wider than the sequences would make that a lot of workspace for nothing, so
// from here on the second pass computes the scores again.
constexpr long long kMaxScoreBytes = 1ll << 30;

// dv_mass_small up to so many blocks of it: two per CU, and four where a sequence has few
// (each block goes through the pairs of all blocks of its sequence: 33 parts are about as fast either
// way at 1056 blocks, 64 parts slower at 1024).  Beside the kernels of
// the plan, bf16, 4 KV heads, 5 / 33 tokens: 20 blocks 13 / 21 us instead of 24 / 55; 252
// of one sequence 14 / 27 instead of 24 / 55; 400 of 20 sequences 19 / 40 instead of 25 /
// 62; 576 of 16 21 / 42 instead of 27 / 64; 760 of two 30 / 67 instead of 25 / 60; 1024 of
// four 35 / 76 instead of 25 / 60.  fp32 (32 rows per block): 640 of 20 31 / 95 instead of
// 35 / 115; 1056 of 8 34 / 122 instead of 34 / 111.
constexpr long long kSmallBlocks = 512, kManySmallBlocks = 1024, kFewParts = 34;

struct MassWs {
    bool stored;
    bool small;  // dv_mass_small
    int units;   // per wave (stored)
    int tokens;  // per launch
    long long rows, chunks, parts;  // stream rows of a block; blocks of a (sequence, KV head)'s keys; those of all its rows
    size_t rq, part, lse, scores, plan, total;
};

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

MassWs mass_ws(int dtype, int F, int W, int S, int Hkv, long long max_rows, long long capacity) {
    MassWs l{};
    const long long wh = (long long)W * Hkv;
    const int unit = tiles_of(dtype) * 16;
    long long rows = (long long)kMassWaves * unit;  // of a block
    l.units = 1;
    if (S == 1) {
        // as many units per wave, up to four, as leave 2048 blocks
        while (l.units < kMaxUnits && wh * (max_rows / (rows * 2 * l.units)) >= 2048) l.units *= 2;
        rows *= l.units;
    }
    l.chunks = (max_rows + rows - 1) / rows;
    const long long score_bytes = wh * l.chunks * rows * kGqa * 4;
    l.stored = S == 1 && score_bytes <= kMaxScoreBytes;
    const long long all = capacity > max_rows ? capacity : max_rows;
    // dv_mass_small's blocks per sequence and KV head (at least one: the capacity is not 0)
    const long long few = (all + unit - 1) / unit + F;
    l.small = S > 1 && S <= kMassTokens && wh * few <= (few <= kFewParts ? kManySmallBlocks : kSmallBlocks);
    if (l.small) {
        l.units = 1;
        l.rows = unit;
        l.tokens = S;
        l.chunks = few;
        l.rq = up256((size_t)F * wh * kGqa * S * kHeadDim * (dtype == kF32 ? 4 : 2));
        l.part = up256((size_t)(wh * l.chunks * S * kGqa * 8));
        l.total = l.rq + l.part;
        return l;
    }
    if (!l.stored) {
        rows = (long long)kMassWaves * unit;
        l.units = 1;
        // parts end with their view
        l.chunks = (max_rows + rows - 1) / rows + F;
    }
    l.rows = rows;
    l.parts = (all + rows - 1) / rows + F + 1;
    l.tokens = S < kMassTokens ? S : kMassTokens;
    if (l.stored) {
        l.part = up256((size_t)(wh * l.chunks * kGqa * 8));
        l.scores = (size_t)score_bytes;
    } else {
        l.rq = up256((size_t)F * wh * kGqa * S * kHeadDim * (dtype == kF32 ? 4 : 2));
        l.part = up256((size_t)(wh * l.tokens * l.chunks * kGqa * 8));
        l.lse = up256((size_t)(wh * l.tokens * kGqa * 4));
        l.plan = up256((size_t)W * (F + 2) * 4) + (size_t)W * l.parts * 16;
    }
    l.total = l.rq + l.part + l.lse + l.scores + l.plan;
    return l;
}

template <int DT>
hipError_t mass_go(MassParams p, const MassWs& l, int device, hipStream_t stream) {
    constexpr int NT = kTilesOf<DT>;
    const long long rows = l.rows;
    const unsigned wh = (unsigned)(p.W * p.Hkv);
    const dim3 block(kMassThreads);
    const dim3 keys((unsigned)(wh * l.chunks)), outs((unsigned)(wh * ((p.C + rows - 1) / rows)));
    hipError_t e;
    p.nchunks = (int)l.chunks;
    p.units = l.units;
    if (p.S == 0 || l.stored) {
        p.s0 = 0;
        p.ns = p.S;
        if (keys.x && p.S) {
            static std::atomic<unsigned long long> ring_done{0};
            e = once_per_device(ring_done, device, [] {
                return hipFuncSetAttribute(reinterpret_cast<const void*>(&dv_mass_scores<DT, NT>),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, kScoreRing);
            });
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL((dv_mass_scores<DT, NT>), keys, block, kScoreRing, stream, p);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        // without a token every row only decays
        if (outs.x) hipLaunchKernelGGL(dv_mass_apply_scores<NT>, outs, block, 0, stream, p);
        return hipGetLastError();
    }
    const long long pieces = (long long)p.F * wh * p.S * (kPieces<DT> * kWave);
    const int plans = l.small ? 0 : p.W;
    const dim3 prep((unsigned)plans + (unsigned)((pieces + kMassThreads - 1) / kMassThreads));
    p.nparts = (int)l.parts;
    if (prep.x) hipLaunchKernelGGL(dv_mass_prepare<DT>, prep, block, 0, stream, p, pieces, plans, (int)rows);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (l.small) {
        p.s0 = 0;
        p.ns = p.S;
        hipLaunchKernelGGL((dv_mass_small<DT, NT, false>), keys, dim3(kSmallThreads), 0, stream, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        hipLaunchKernelGGL((dv_mass_small<DT, NT, true>), keys, dim3(kSmallThreads), 0, stream, p);
        return hipGetLastError();
    }
    const dim3 parts((unsigned)(wh * l.parts));
    for (int s0 = 0; s0 < p.S; s0 += l.tokens) {
        p.s0 = s0;
        p.ns = p.S - s0 < l.tokens ? p.S - s0 : l.tokens;
        if (keys.x) {
            hipLaunchKernelGGL((dv_mass_stats<DT, NT>), keys, block, 0, stream, p);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        hipLaunchKernelGGL(dv_mass_lse, dim3(wh * (unsigned)p.ns), block, 0, stream, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        hipLaunchKernelGGL((dv_mass_apply<DT, NT>), parts, block, 0, stream, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        p.mass = p.out;  // the launches after the first add to the first's result
        p.decay = 1.0f;
    }
    return hipSuccess;
}

}  // namespace

size_t mass_workspace_bytes(int dtype, int F, int W, int S, int Hkv, long long max_rows, long long capacity) {
    if (F < 0 || W <= 0 || S <= 0 || Hkv <= 0 || max_rows < 0 || capacity < 0) return 0;
    return mass_ws(dtype, F, W, S, Hkv, max_rows, capacity).total;
}

hipError_t launch_key_mass(int dtype, const MassParams& base, void* workspace, hipStream_t stream) {
    MassParams p = base;
    const MassWs l = mass_ws(dtype, p.F, p.W, p.S, p.Hkv, (long long)p.maxB * p.bs, p.C);
    unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
    p.rq = ws;
    p.part = reinterpret_cast<float*>(ws + l.rq);
    p.lse = reinterpret_cast<float*>(ws + l.rq + l.part);
    p.scores = reinterpret_cast<float*>(ws + l.rq + l.part + l.lse);
    p.plan_seen = reinterpret_cast<int*>(ws + l.rq + l.part + l.lse + l.scores);
    p.plan_count = p.plan_seen + (size_t)p.W * p.F;
    p.plan_list = reinterpret_cast<int4*>(ws + l.rq + l.part + l.lse + l.scores + up256((size_t)p.W * (p.F + 2) * 4));
    int device = 0;
    const hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    switch (dtype) {
        case kBF16: return mass_go<kBF16>(p, l, device, stream);
        case kF16: return mass_go<kF16>(p, l, device, stream);
        case kF32: return mass_go<kF32>(p, l, device, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace dv
