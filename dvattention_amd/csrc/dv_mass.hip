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
// K rows are the A operand of S^T = K Q^T (16x16x32 MFMA, 16x16x4 for fp32), loaded
// into registers by the wave that owns the keys: with no second product there is
// nothing to share between waves.  Every K row is read once per pass however many
// tokens vote, and a key's weight is summed by one wave in a fixed order -- no
// atomics, the same bits from every run.  Scores, maxima, sums and weights are fp32.
//
//  * S = 1 (a decode step; bound by memory): the queries are rotated in the kernel
//    and the scores stored (64 bytes per key and KV head, a quarter of a 16-bit K row, an
//    eighth of an fp32 one), so the second pass reads those and not K.
//  * S > 1 (a window of tokens; bound by the exponentials): a wave holds 64 keys (32
//    for fp32) and walks the tokens, whose queries one launch beforehand rotated into
//    the MFMA's operand order; the second pass computes the scores again (storing
//    them would cost more bytes than K from two tokens on).  At most kMassTokens
//    tokens per launch bound the workspace.
#include "dv_common.h"
#include "dv_device.h"

namespace dv {

namespace {

constexpr int kMassWaves = 4;
constexpr int kMassThreads = kMassWaves * kWave;
constexpr int kMassTokens = kWave;  // one lane per token holds what it sees

// 16-byte pieces of a K row per lane: lane (g, n) of a 16-key tile holds bytes
// cc * 64 + g * 16 of key n's row, for both operands alike (the order of the dims in a
// dot product does not matter as long as both agree).
template <int DT> constexpr int kPieces = kHeadDim * Tr<DT>::kBytes / 64;
template <int DT> constexpr int kOperandBytes = kPieces<DT> * kWave * 16;  // one token's 16 heads
// 16-key tiles per wave: 64 registers of K
template <int DT> constexpr int kTilesOf = DT == kF32 ? 2 : 4;

template <int DT>
__device__ inline f32x4 dot_tile(const u32x4 (&k)[kPieces<DT>], const u32x4 (&q)[kPieces<DT>]) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int cc = 0; cc < kPieces<DT>; ++cc) {
        if constexpr (DT == kF32) {
            const f32x4 kf = __builtin_bit_cast(f32x4, k[cc]), qf = __builtin_bit_cast(f32x4, q[cc]);
#pragma unroll
            for (int j = 0; j < 4; ++j) s = Tr<kF32>::mma1(kf[j], qf[j], s);
        } else {
            s = Tr<DT>::mma(k[cc], q[cc], s);
        }
    }
    return s;
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

// Keys [lo, hi) of NT * 16 as bits.
template <int NT>
__device__ inline uint64_t range_bits(long long lo, long long hi) {
    lo = lo < 0 ? 0 : lo;
    hi = hi > NT * 16 ? NT * 16 : hi;
    if (lo >= hi) return 0;
    return (~0ull >> (64 - (hi - lo))) << lo;
}
template <int NT> constexpr uint64_t kAllKeys = ~0ull >> (64 - NT * 16);

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

// Minus the log-sum-exp of head tid % 16 over `count` pairs (pair u of head n at
// pairs[u * 16 + n]), in every thread of the block; -inf where no key is seen, so that
// 2^(x + it) is 0.
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
    return l == 0.0f ? -DV_INF : -(m + log2f(l));
}

__device__ inline float row16_sum(float v) {
    v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x128, 0xf, 0xf, false));  // ror 8
    v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x124, 0xf, 0xf, false));  // ror 4
    v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x122, 0xf, 0xf, false));  // ror 2
    v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x121, 0xf, 0xf, false));  // ror 1
    return v;
}

// A weight: invisible keys (-inf) get none, whatever the row's sum is.
__device__ inline float weight(float x, float nl) { return x == -DV_INF ? 0.0f : __builtin_amdgcn_exp2f(x + nl); }

// out = decay * mass + acc summed over the 16 heads, for a unit's rows below C.
template <int NT>
__device__ inline void store_mass(const MassParams& p, long long wh, long long c0, const f32x4 (&acc)[NT]) {
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, n = lane & 15;
    float old[NT];
    const long long c = c0 + g * 4 + n;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        old[t] = 0.0f;
        if (n < 4 && c + t * 16 < p.C && p.decay != 0.0f) old[t] = p.mass[wh * p.C + c + t * 16] * p.decay;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float mine = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = row16_sum(acc[t][i]);
            mine = n == i ? a : mine;
        }
        if (n < 4 && c + t * 16 < p.C) p.out[wh * p.C + c + t * 16] = old[t] + mine;
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

// S = 1.  Block: 4 waves times p.units units of NT tiles of one (sequence, KV head),
// unit u of wave v at rows (u * 4 + v) * NT * 16 of the block's.  Leaves the scores (tile
// by tile, as the lanes hold them) and, per block and head, (max, sum).  A unit's
// page ids are loaded while the unit before it is computed.
template <int DT, int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_scores(const MassParams p) {
    __shared__ u32x4 s_q[kPieces<DT> * kWave];
    __shared__ float2 s_pair[kMassWaves][kGqa];
    constexpr int kRows = NT * 16;
    const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
    const Item it = item_of(p);
    const long long end = visible_end(p, it.w);
    const long long rows = (long long)kMassWaves * kRows * p.units;
    const long long b0 = it.chunk * rows;
    if (b0 >= end) return;
    const long long b1 = b0 + rows < end ? b0 + rows : end;  // the block's visible part
    float m = -DV_INF, l = 0.0f;  // this lane's keys
    long long off = 0;
    bool first = true;            // no view's scores are stored yet
    for (int f = 0; f < p.F && off < b1; ++f) {
        const int len = view_len(p, f);
        const long long lo = off;
        off += len;
        if (off <= b0) continue;
        const long long hi = lo + uniform(seen_of(p, f, it.w, p.s0, len));
        if (!first) __syncthreads();  // the previous view's query is read
        for (int i = threadIdx.x; i < kPieces<DT> * kWave; i += kMassThreads)
            s_q[i] = rotated_piece<DT>(p, f, it.w, it.hkv, p.s0, i);
        __syncthreads();
        u32x4 q[kPieces<DT>];
#pragma unroll
        for (int cc = 0; cc < kPieces<DT>; ++cc) q[cc] = s_q[cc * kWave + lane];

        auto row_of = [&](long long c0) {
            const long long c = c0 + lane;
            return cache_row(p, it.w, it.hkv, c, lane < kRows && c >= lo && c < hi);
        };
        long long c0 = b0 + wv * kRows;
        uint32_t row = row_of(c0);
        for (int u = 0; u < p.units && c0 < b1; ++u, c0 += kMassWaves * kRows) {
            u32x4 k[NT][kPieces<DT>];
            load_keys<DT, NT>(p, row, k);
            const uint64_t mask = ballot(row != 0xffffffffu);
            row = row_of(c0 + kMassWaves * kRows);
            f32x4 x[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) x[t] = dot_tile<DT>(k[t], q);
            scale_masked<NT>(x, mask, p.l2scale);
            float* dst = p.scores + ((it.wh * p.nchunks * rows + c0) / 16 * kWave + lane) * 4;
            if (first) {
#pragma unroll
                for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(dst + t * kWave * 4) = x[t];
            } else {
                // rows of earlier views keep theirs
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint32_t b = lane_bits(mask, t);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if ((b >> i) & 1u) dst[t * kWave * 4 + i] = x[t][i];
                }
            }
            float mx = -DV_INF;
#pragma unroll
            for (int t = 0; t < NT; ++t) mx = fmaxf(mx, fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
            const float mn = fmaxf(m, mx);
            const float mz = mn == -DV_INF ? 0.0f : mn;
            l *= __builtin_amdgcn_exp2f(m - mz);
#pragma unroll
            for (int t = 0; t < NT; ++t)
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
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const Item it = item_of(p);
    const long long end = visible_end(p, it.w);
    const long long rows = (long long)kMassWaves * kRows * p.units;
    long long c0 = it.chunk * rows + wv * kRows;
    float nl = 0.0f;
    if (it.chunk * rows < end)
        nl = joined_lse(reinterpret_cast<const float2*>(p.part) + it.wh * p.nchunks * kGqa, (end + rows - 1) / rows,
                        s_pair);
    for (int u = 0; u < p.units; ++u, c0 += kMassWaves * kRows) {
        if (c0 >= end) {
            store_decayed(p, it.wh, c0, kRows);
            continue;
        }
        const float* src = p.scores + ((it.wh * p.nchunks * rows + c0) / 16 * kWave + lane) * 4;
        f32x4 x[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) x[t] = ld16f(src + t * kWave * 4);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[t][i] = weight(x[t][i], nl);
        store_mass<NT>(p, it.wh, c0, x);
    }
}

// S > 1: the query operands, [F, W, Hkv, S] of kOperandBytes each; a thread per 16 bytes.
template <int DT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_rotate(const MassParams p, long long n) {
    const long long i = (long long)blockIdx.x * kMassThreads + threadIdx.x;
    if (i >= n) return;
    constexpr int kPer = kPieces<DT> * kWave;
    const long long op = i / kPer;
    const int piece = (int)(i - op * kPer);
    const int s = (int)(op % p.S);
    const long long r = op / p.S;
    const int hkv = (int)(r % p.Hkv);
    const long long fw = r / p.Hkv;
    reinterpret_cast<u32x4*>(p.rq)[i] =
        rotated_piece<DT>(p, (int)(fw / p.W), (int)(fw % p.W), hkv, s, piece);
}

namespace {

// Tokens whose operands one ring half holds, staged together.
template <int DT> constexpr int kGroup = DT == kF32 ? 4 : 8;
template <int DT> constexpr int kRingBytes = 2 * kGroup<DT> * kOperandBytes<DT>;

// A block's keys (4 waves, one unit each) against every token of the launch, view by
// view and kGroup tokens at a time: the operands of a group are copied to LDS, a
// quarter by each wave (they lie in the order the waves read them), while the group
// before it is computed.  prepare(s0) runs in every wave before the group of tokens s0 is
// waited for; body(s, x, mask, all) gets token s's raw scores x and the keys of this
// view it sees (all: every key of the unit; not called where it sees none);
// done(s0, n, first) runs in every wave after a group (first: of the first view the
// block meets) and may use block barriers of its own.
template <int DT, int NT, class Prepare, class Body, class Done>
__device__ inline void walk_tokens(const MassParams& p, const Item& it, long long c0, unsigned char* ring,
                                   Prepare&& prepare, Body&& body, Done&& done) {
    constexpr int kRows = NT * 16;
    const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
    const long long b0 = it.chunk * (kMassWaves * kRows), b1 = b0 + kMassWaves * kRows;
    const uint32_t ring_at = lds_addr(ring);
    const int groups = (p.ns + kGroup<DT> - 1) / kGroup<DT>;
    long long off = 0;
    bool first = true;  // view of the block: a block below visible_end meets one
    for (int f = 0; f < p.F && off < b1; ++f) {
        const int len = view_len(p, f);
        const long long lo = off;
        off += len;
        if (off <= b0 || len == 0) continue;  // the same for all waves
        const int seen = seen_lane(p, f, it.w, len);
        const long long c = c0 + lane, hi = lo + lanes_max(seen);
        const uint32_t row = cache_row(p, it.w, it.hkv, c, lane < kRows && c >= lo && c < hi);
        const unsigned char* ops = reinterpret_cast<const unsigned char*>(p.rq) +
                                   ((((long long)f * p.W + it.w) * p.Hkv + it.hkv) * p.S + p.s0) * kOperandBytes<DT>;
        auto stage = [&](int gi) {
            const int n = p.ns - gi * kGroup<DT> < kGroup<DT> ? p.ns - gi * kGroup<DT> : kGroup<DT>;
            for (int i = wv; i < n * kPieces<DT>; i += kMassWaves)
                dma16(ops + ((long long)gi * kGroup<DT> * kPieces<DT> + i) * 1024 + lane * 16,
                      __builtin_amdgcn_readfirstlane(ring_at + (uint32_t)((gi & 1) * kGroup<DT> * kOperandBytes<DT> + i * 1024)));
        };
        stage(0);
        const uint64_t valid = ballot(row != 0xffffffffu);
        u32x4 k[NT][kPieces<DT>];
        load_keys<DT, NT>(p, row, k);
        // keys of the unit before the end of what token s sees, in lane s
        const long long upto = lo - c0 + seen;
        const int ends = (int)(upto < 0 ? 0 : upto < kRows ? upto : kRows);
        const uint64_t from = range_bits<NT>(lo - c0, kRows);
        for (int gi = 0; gi < groups; ++gi) {
            const int t0 = gi * kGroup<DT>;
            const int n = p.ns - t0 < kGroup<DT> ? p.ns - t0 : kGroup<DT>;
            prepare(t0);
            wait_vmcnt<0>();
            __syncthreads();  // the group is here; every wave is done with the other half
            if (gi + 1 < groups) stage(gi + 1);
            const u32x4* half = reinterpret_cast<const u32x4*>(ring + (gi & 1) * kGroup<DT> * kOperandBytes<DT>) + lane;
            if (valid) {
#pragma unroll 1
                for (int s = 0; s < n; ++s) {
                    const uint64_t mask = valid & from & range_bits<NT>(0, __builtin_amdgcn_readlane(ends, t0 + s));
                    if (!mask) continue;
                    u32x4 q[kPieces<DT>];
#pragma unroll
                    for (int cc = 0; cc < kPieces<DT>; ++cc) q[cc] = half[(s * kPieces<DT> + cc) * kWave];
                    f32x4 x[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) x[t] = dot_tile<DT>(k[t], q);
                    body(t0 + s, x, mask, mask == kAllKeys<NT>);
                }
            }
            done(t0, n, first);
        }
        first = false;
        __syncthreads();  // the ring is read before the next view fills it
    }
}

}  // namespace

// Per block of keys, token of the launch and head, (max, sum).
template <int DT, int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_stats(const MassParams p) {
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ float2 s_pair[kMassWaves][kGroup<DT>][kGqa];
    constexpr int kRows = NT * 16;
    const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6);
    const Item it = item_of(p);
    if (it.chunk * (kMassWaves * kRows) >= visible_end(p, it.w)) return;
    float2* part = reinterpret_cast<float2*>(p.part) + (it.wh * p.ns * p.nchunks + it.chunk) * kGqa;
    const float l2 = p.l2scale;
    const float2 none = make_float2(-DV_INF, 0.0f);
    walk_tokens<DT, NT>(
        p, it, (it.chunk * kMassWaves + wv) * kRows, ring,
        [&](int) {
            // tokens that see none of the wave's keys (the wave's own entries, read before
            // the last group's end)
            for (int i = lane; i < kGroup<DT> * kGqa; i += kWave) s_pair[wv][i >> 4][i & 15] = none;
        },
        [&](int s, f32x4(&x)[NT], uint64_t mask, bool all) {
            if (!all) scale_masked<NT>(x, mask, l2);
            float mx = -DV_INF;
            if (all && l2 < 0.0f) {
                float mn = DV_INF;
#pragma unroll
                for (int t = 0; t < NT; ++t) mn = fminf(mn, fminf(fminf(x[t][0], x[t][1]), fminf(x[t][2], x[t][3])));
                mx = mn * l2;
            } else {
#pragma unroll
                for (int t = 0; t < NT; ++t) mx = fmaxf(mx, fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
                if (all) mx *= l2;
            }
            const float m = rows4_max(mx);
            const float mz = m == -DV_INF ? 0.0f : m;
            const float f = all ? l2 : 1.0f;
            float l = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][i], f, -mz));
            l = rows4_sum(l);
            if (lane < kGqa) s_pair[wv][s & (kGroup<DT> - 1)][lane] = make_float2(m, l);
        },
        [&](int t0, int n, bool first) {
            // the block's waves, and the keys of an earlier view
            __syncthreads();
            const int s = tid >> 4, h = tid & 15;
            if (s < n) {
                float2* to = part + (long long)(t0 + s) * p.nchunks * kGqa + h;
                float2 e = first ? none : *to;
#pragma unroll
                for (int v = 0; v < kMassWaves; ++v) join(e.x, e.y, s_pair[v][s][h].x, s_pair[v][s][h].y);
                *to = e;
            }
            __syncthreads();
        });
}

// Block (sequence, KV head, token): minus the log-sum-exp of its heads.
__global__ __launch_bounds__(kMassThreads) void dv_mass_lse(const MassParams p, int block_rows) {
    __shared__ float2 s_pair[kMassThreads];
    const long long row = blockIdx.x;  // (w * Hkv + hkv) * ns + s
    const int w = (int)(row / ((long long)p.ns * p.Hkv));
    const long long live = (visible_end(p, w) + block_rows - 1) / block_rows;
    const float nl = joined_lse(reinterpret_cast<const float2*>(p.part) + row * p.nchunks * kGqa, live, s_pair);
    if (threadIdx.x < kGqa) p.lse[row * kGqa + threadIdx.x] = nl;
}

template <int DT, int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_apply(const MassParams p) {
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ float s_nl[2][kGroup<DT> * kGqa];
    constexpr int kRows = NT * 16;
    const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
    const Item it = item_of(p);
    const long long c0 = (it.chunk * kMassWaves + wv) * kRows;
    if (it.chunk * (kMassWaves * kRows) >= visible_end(p, it.w)) {
        store_decayed(p, it.wh, c0, kRows);
        return;
    }
    const float* lse = p.lse + it.wh * p.ns * kGqa;
    const float l2 = p.l2scale;
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    walk_tokens<DT, NT>(
        p, it, c0, ring,
        [&](int t0) {
            // the half that the group before this one does not read
            const int at = t0 * kGqa + (int)threadIdx.x;
            if (threadIdx.x < kGroup<DT> * kGqa)
                s_nl[(t0 / kGroup<DT>)&1][threadIdx.x] = at < p.ns * kGqa ? lse[at] : 0.0f;
        },
        [&](int s, f32x4(&x)[NT], uint64_t mask, bool all) {
            const float nl = s_nl[(s / kGroup<DT>)&1][(s & (kGroup<DT> - 1)) * kGqa + (lane & 15)];
            if (all) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t][i] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][i], l2, nl));
            } else {
                scale_masked<NT>(x, mask, l2);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t][i] += weight(x[t][i], nl);
            }
        },
        [](int, int, bool) {});
    store_mass<NT>(p, it.wh, c0, acc);
}

// ---- launches --------------------------------------------------------------------

namespace {

int tiles_of(int dtype) { return dtype == kF32 ? kTilesOf<kF32> : kTilesOf<kBF16>; }

// Stored scores of a decode step take a quarter of a 16-bit K cache's bytes; block tables
// far wider than the sequences would make that a lot of workspace for nothing, so
// from here on the second pass computes the scores again.
constexpr long long kMaxScoreBytes = 1ll << 30;

struct MassWs {
    bool stored;
    int units;   // per wave (stored)
    int tokens;  // per launch
    long long chunks;
    size_t rq, part, lse, scores, total;
};

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

MassWs mass_ws(int dtype, int F, int W, int S, int Hkv, long long max_rows) {
    MassWs l{};
    const long long wh = (long long)W * Hkv;
    long long rows = (long long)kMassWaves * tiles_of(dtype) * 16;  // of a block
    l.units = 1;
    if (S == 1) {
        // as many units per wave, up to four, as leave 2048 blocks
        while (l.units < 4 && wh * (max_rows / (rows * 2 * l.units)) >= 2048) l.units *= 2;
        rows *= l.units;
    }
    l.chunks = (max_rows + rows - 1) / rows;
    const long long score_bytes = wh * l.chunks * rows * kGqa * 4;
    l.stored = S == 1 && score_bytes <= kMaxScoreBytes;
    if (!l.stored && l.units > 1) {
        rows /= l.units;
        l.units = 1;
        l.chunks = (max_rows + rows - 1) / rows;
    }
    l.tokens = S < kMassTokens ? S : kMassTokens;
    if (l.stored) {
        l.part = up256((size_t)(wh * l.chunks * kGqa * 8));
        l.scores = (size_t)score_bytes;
    } else {
        l.rq = up256((size_t)F * wh * kGqa * S * kHeadDim * (dtype == kF32 ? 4 : 2));
        l.part = up256((size_t)(wh * l.tokens * l.chunks * kGqa * 8));
        l.lse = up256((size_t)(wh * l.tokens * kGqa * 4));
    }
    l.total = l.rq + l.part + l.lse + l.scores;
    return l;
}

template <int DT>
hipError_t mass_go(MassParams p, const MassWs& l, int device, hipStream_t stream) {
    constexpr int NT = kTilesOf<DT>;
    const long long rows = (long long)kMassWaves * NT * 16 * l.units;  // stream rows of a block
    const unsigned wh = (unsigned)(p.W * p.Hkv);
    const dim3 block(kMassThreads);
    const dim3 keys((unsigned)(wh * l.chunks)), outs((unsigned)(wh * ((p.C + rows - 1) / rows)));
    hipError_t e;
    p.nchunks = (int)l.chunks;
    p.units = l.units;
    if (!l.stored) {
        static std::atomic<unsigned long long> attr_done{0};
        e = once_per_device(attr_done, device, [] {
            const hipError_t es = hipFuncSetAttribute(reinterpret_cast<const void*>(&dv_mass_stats<DT, NT>),
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, kRingBytes<DT>);
            return es != hipSuccess ? es
                                    : hipFuncSetAttribute(reinterpret_cast<const void*>(&dv_mass_apply<DT, NT>),
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, kRingBytes<DT>);
        });
        if (e != hipSuccess) return e;
    }
    if (p.S == 0) {  // no token votes: every row only decays
        if (outs.x) hipLaunchKernelGGL((dv_mass_apply<DT, NT>), outs, block, kRingBytes<DT>, stream, p);
        return hipGetLastError();
    }
    if (l.stored) {
        p.s0 = 0;
        p.ns = 1;
        if (keys.x) {
            hipLaunchKernelGGL((dv_mass_scores<DT, NT>), keys, block, 0, stream, p);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        if (outs.x) hipLaunchKernelGGL(dv_mass_apply_scores<NT>, outs, block, 0, stream, p);
        return hipGetLastError();
    }
    const long long pieces = (long long)p.F * wh * p.S * (kPieces<DT> * kWave);
    if (pieces) {
        hipLaunchKernelGGL(dv_mass_rotate<DT>, dim3((unsigned)((pieces + kMassThreads - 1) / kMassThreads)), block, 0,
                           stream, p, pieces);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    for (int s0 = 0; s0 < p.S; s0 += l.tokens) {
        p.s0 = s0;
        p.ns = p.S - s0 < l.tokens ? p.S - s0 : l.tokens;
        if (keys.x) {
            hipLaunchKernelGGL((dv_mass_stats<DT, NT>), keys, block, kRingBytes<DT>, stream, p);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        hipLaunchKernelGGL(dv_mass_lse, dim3(wh * (unsigned)p.ns), block, 0, stream, p, (int)rows);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        if (outs.x) hipLaunchKernelGGL((dv_mass_apply<DT, NT>), outs, block, kRingBytes<DT>, stream, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        p.mass = p.out;  // the launches after the first add to the first's result
        p.decay = 1.0f;
    }
    return hipSuccess;
}

}  // namespace

size_t mass_workspace_bytes(int dtype, int F, int W, int S, int Hkv, long long max_rows, int) {
    if (F < 0 || W <= 0 || S <= 0 || Hkv <= 0 || max_rows < 0) return 0;
    return mass_ws(dtype, F, W, S, Hkv, max_rows).total;
}

hipError_t launch_key_mass(int dtype, const MassParams& base, void* workspace, hipStream_t stream) {
    MassParams p = base;
    const MassWs l = mass_ws(dtype, p.F, p.W, p.S, p.Hkv, (long long)p.maxB * p.bs);
    unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
    p.rq = ws;
    p.part = reinterpret_cast<float*>(ws + l.rq);
    p.lse = reinterpret_cast<float*>(ws + l.rq + l.part);
    p.scores = reinterpret_cast<float*>(ws + l.rq + l.part + l.lse);
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
