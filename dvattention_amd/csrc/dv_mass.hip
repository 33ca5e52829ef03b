// Attention weight that every cached key receives (dvattn_paged_key_mass):
//   out[w, h, c] = decay * mass[w, h, c]
//                + sum over tokens s and the 16 query heads n of KV head h of
//                  2^(x_{s,n,c} - lse_{s,n}),
// x the base-2 scores of the key in stream row c (rotated query of c's view), lse the
// base-2 log-sum-exp of row (s, n) over its visible keys.  The weights need the sums
// over all keys first, so the keys are passed twice: dv_mass_stats leaves every
// row's (max, sum) over each workgroup's or wave's keys, dv_mass_apply reads the
// joined lse and adds the weights up.
//
// A wave owns NT tiles of 16 keys, their K rows in registers (the A operand of
// S^T = K Q^T, 16x16x32 MFMA; 16x16x4 for fp32), and walks the tokens: every K row is
// read once per pass however many tokens vote, and a key's weight is summed by one
// wave in a fixed order -- no atomics, the same bits from every run.  Scores, maxima,
// sums and weights are fp32 throughout.
//
//  * S = 1 (a decode step; bound by memory): the queries are rotated in the kernel
//    and the scores stored (64 bytes per key and KV head, a quarter of a 16-bit K row, an
//    eighth of an fp32 one), so the second pass reads those and not K.
//  * S > 1 (a window of tokens; bound by the exponentials): queries rotated once
//    beforehand, scores computed again in the second pass (storing them would cost
//    more bytes than K from two tokens on); up to kMassTokens tokens per launch bound
//    the workspace.
#include "dv_common.h"
#include "dv_device.h"

namespace dv {

namespace {

constexpr int kMassWaves = 4;
constexpr int kMassThreads = kMassWaves * kWave;
constexpr int kMassTokens = 64;

// 16-byte pieces of a K row per lane (lane (g, n) of a tile holds bytes
// cc * 64 + g * 16 of key n's row), for both operands alike.
template <int DT> constexpr int kPieces = kHeadDim * Tr<DT>::kBytes / 64;

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

// Most keys of view f that any of the launch's tokens sees.
__device__ inline int seen_most(const MassParams& p, int f, int w, int len) {
    const int lane = threadIdx.x & 63;
    if (p.ns == 1) return uniform(seen_of(p, f, w, p.s0, len));
    int best = 0;
    for (int s = lane; s < p.ns; s += kWave) {
        const int v = seen_of(p, f, w, p.s0 + s, len);
        best = v > best ? v : best;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const int o = __shfl_xor(best, d, kWave);
        best = o > best ? o : best;
    }
    return uniform(best);
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

// A unit of stream rows [c0, c0 + NT * 16) of one (sequence, KV head): the views it
// meets (f0 .. f1, f0's key 0 in stream row off0) and its K rows.  ok[j], bit i: row
// c0 + 64 j + i is seen by some token of the launch and lies on a valid page; other
// rows are zeros and are never read.
template <int DT, int NT>
struct Unit {
    static constexpr int kRows = NT * 16;
    static constexpr int kRounds = (kRows + kWave - 1) / kWave;
    long long c0, off0;
    int f0, f1;
    uint64_t ok[kRounds];
    u32x4 k[NT][kPieces<DT>];

    __device__ inline bool all_ok() const {
        bool r = true;
#pragma unroll
        for (int j = 0; j < kRounds; ++j)
            r = r && ok[j] == (kRows - j * kWave >= kWave ? ~0ull : (1ull << (kRows - j * kWave)) - 1ull);
        return r;
    }
    // bits 0-3: rows t * 16 + g * 4 + i
    __device__ inline uint32_t ok4(int t, int g) const { return (uint32_t)(ok[t / 4] >> ((t % 4) * 16 + g * 4)) & 15u; }

    __device__ inline void load(const MassParams& p, int w, int hkv, long long first) {
        const int lane = threadIdx.x & 63;
        const int g = lane >> 4, n = lane & 15;
        c0 = first;
        off0 = 0;
        f0 = 0;
        f1 = -1;
        bool in[kRounds];
#pragma unroll
        for (int j = 0; j < kRounds; ++j) in[j] = false;
        long long off = 0;
        for (int f = 0; f < p.F && off < c0 + kRows; ++f) {
            const int len = view_len(p, f);
            if (len > 0 && off + len > c0) {
                if (f1 < 0) {
                    f0 = f;
                    off0 = off;
                }
                f1 = f;
                const long long lo = off, hi = off + seen_most(p, f, w, len);
#pragma unroll
                for (int j = 0; j < kRounds; ++j) {
                    const long long c = c0 + j * kWave + lane;
                    in[j] = in[j] || (c >= lo && c < hi);
                }
            }
            off += len;
        }
        uint32_t at[kRounds];
#pragma unroll
        for (int j = 0; j < kRounds; ++j) {
            const long long c = c0 + j * kWave + lane;
            const bool mine = j * kWave + lane < kRows;
            const long long lp = p.bs_shift >= 0 ? c >> p.bs_shift : c / p.bs;
            int page = -1;
            if (in[j] && mine && lp < p.maxB) page = p.bt[(long long)w * p.maxB + lp];
            const bool valid = page >= 0 && page < p.nblocks;
            at[j] = valid ? ((uint32_t)page * (uint32_t)p.bs + (uint32_t)(c - lp * p.bs)) * (uint32_t)p.Hkv +
                                (uint32_t)hkv
                          : 0u;
            ok[j] = ballot(valid);
        }
        const unsigned char* base = reinterpret_cast<const unsigned char*>(p.kc) + g * 16;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t row = (uint32_t)__shfl((int)at[t / 4], (t % 4) * 16 + n, kWave);
            const bool valid = (ok[t / 4] >> ((t % 4) * 16 + n)) & 1ull;
#pragma unroll
            for (int cc = 0; cc < kPieces<DT>; ++cc) k[t][cc] = u32x4{0u, 0u, 0u, 0u};
            if (valid) {
                const unsigned char* src = base + (unsigned long long)row * (kHeadDim * Tr<DT>::kBytes);
#pragma unroll
                for (int cc = 0; cc < kPieces<DT>; ++cc) k[t][cc] = ld16(src + cc * 64);
            }
        }
    }

    // Base-2 scores of token s (lane (g, n): rows t * 16 + g * 4 + i of head n), -inf where
    // it does not see the row.  query(f, q): the token's rotated query of view f.
    template <class Query>
    __device__ inline void scores(const MassParams& p, int w, int s, Query&& query, f32x4 (&x)[NT]) const {
        const int g = (threadIdx.x & 63) >> 4;
        long long off = off0;
        if (f0 != f1) {
#pragma unroll
            for (int t = 0; t < NT; ++t) x[t] = f32x4{-DV_INF, -DV_INF, -DV_INF, -DV_INF};
        }
        for (int f = f0; f <= f1; ++f) {
            const int len = view_len(p, f);
            const long long lo = off - c0, hi = lo + uniform(seen_of(p, f, w, s, len));
            off += len;
            u32x4 q[kPieces<DT>];
            query(f, q);
            const bool full = f0 == f1 && lo <= 0 && hi >= kRows && all_ok();
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const f32x4 d = dot_tile<DT>(k[t], q);
                if (full) {
                    x[t] = d * p.l2scale;
                } else {
                    const uint32_t bits = ok4(t, g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = t * 16 + g * 4 + i;
                        const bool see = r >= lo && r < hi && ((bits >> i) & 1u);
                        x[t][i] = see ? d[i] * p.l2scale : (f0 == f1 ? -DV_INF : x[t][i]);
                    }
                }
            }
        }
    }
};

// The rotated query of (view, sequence, token): lane (g, n) holds pieces g of head n.
template <int DT>
__device__ inline void rotated_query(const MassParams& p, int f, int w, int s, int hkv, u32x4 (&q)[kPieces<DT>]) {
    using raw = typename Tr<DT>::raw;
    constexpr int N = 16 / Tr<DT>::kBytes;
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, n = lane & 15;
    const raw* qrow = reinterpret_cast<const raw*>(p.q) + (((long long)w * p.Hq + hkv * kGqa + n) * p.S + s) * kHeadDim;
    const long long cs = (((long long)f * p.W + w) * p.S + s) * p.R;
#pragma unroll
    for (int cc = 0; cc < kPieces<DT>; ++cc) {
        raw r[N];
        rotate_run<DT, N>(qrow, p.cosv + cs, p.sinv + cs, p.R, (cc * 64 + g * 16) / Tr<DT>::kBytes, r);
        __builtin_memcpy(&q[cc], r, 16);
    }
}

template <int DT>
__device__ inline void stored_query(const MassParams& p, int f, int w, int s, int hkv, u32x4 (&q)[kPieces<DT>]) {
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, n = lane & 15;
    const long long row = (((long long)f * p.W + w) * p.Hq + hkv * kGqa + n) * p.S + s;
    const unsigned char* src =
        reinterpret_cast<const unsigned char*>(p.rq) + row * (kHeadDim * Tr<DT>::kBytes) + g * 16;
#pragma unroll
    for (int cc = 0; cc < kPieces<DT>; ++cc) q[cc] = ld16(src + cc * 64);
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

// A row's maximum and sum over its scores x, in every lane of the head.
template <int NT>
__device__ inline void row_stats(const f32x4 (&x)[NT], float& m, float& l) {
    float mx = -DV_INF;
#pragma unroll
    for (int t = 0; t < NT; ++t) mx = fmaxf(mx, fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
    m = rows4_max(mx);
    const float mz = m == -DV_INF ? 0.0f : m;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f(x[t][i] - mz);
    l = rows4_sum(sum);
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
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float mine = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = row16_sum(acc[t][i]);
            mine = n == i ? a : mine;
        }
        const long long c = c0 + t * 16 + g * 4 + n;
        if (n < 4 && c < p.C) {
            const long long at = wh * p.C + c;
            p.out[at] = (p.decay == 0.0f ? 0.0f : p.mass[at] * p.decay) + mine;
        }
    }
}

// The same for rows that no token sees.
template <int NT>
__device__ inline void store_decayed(const MassParams& p, long long wh, long long c0) {
    if (p.out == p.mass && p.decay == 1.0f) return;
    const int lane = threadIdx.x & 63;
    for (int r = lane; r < NT * 16; r += kWave) {
        const long long c = c0 + r;
        if (c < p.C) {
            const long long at = wh * p.C + c;
            p.out[at] = p.decay == 0.0f ? 0.0f : p.mass[at] * p.decay;
        }
    }
}

}  // namespace

// S = 1.  Block: 4 units of one (sequence, KV head).  Leaves the scores and, per block
// and head, (max, sum).
template <int DT, int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_scores(const MassParams p) {
    __shared__ float2 s_pair[kMassWaves][kGqa];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const Item it = item_of(p);
    constexpr int kRows = Unit<DT, NT>::kRows;
    if (it.chunk * (kMassWaves * kRows) >= visible_end(p, it.w)) return;
    const long long unit = it.chunk * kMassWaves + wv;
    Unit<DT, NT> u;
    u.load(p, it.w, it.hkv, unit * kRows);
    f32x4 x[NT];
    if (u.f1 < 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t) x[t] = f32x4{-DV_INF, -DV_INF, -DV_INF, -DV_INF};
    } else {
        u.scores(p, it.w, p.s0, [&](int f, u32x4(&q)[kPieces<DT>]) { rotated_query<DT>(p, f, it.w, p.s0, it.hkv, q); },
                 x);
    }
    float* dst = p.scores + ((it.wh * p.nchunks * kMassWaves + unit) * NT * kWave + lane) * 4;
#pragma unroll
    for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(dst + t * kWave * 4) = x[t];
    float m, l;
    row_stats<NT>(x, m, l);
    if (lane < kGqa) s_pair[wv][lane] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x < kGqa) {
        m = -DV_INF;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < kMassWaves; ++i) join(m, l, s_pair[i][threadIdx.x].x, s_pair[i][threadIdx.x].y);
        reinterpret_cast<float2*>(p.part)[(it.wh * p.nchunks + it.chunk) * kGqa + threadIdx.x] = make_float2(m, l);
    }
}

template <int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_apply_scores(const MassParams p) {
    __shared__ float2 s_pair[kMassThreads];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const Item it = item_of(p);
    constexpr int kRows = NT * 16;
    const long long end = visible_end(p, it.w);
    const long long unit = it.chunk * kMassWaves + wv;
    if (it.chunk * (kMassWaves * kRows) >= end) {
        store_decayed<NT>(p, it.wh, unit * kRows);
        return;
    }
    const float* src = p.scores + ((it.wh * p.nchunks * kMassWaves + unit) * NT * kWave + lane) * 4;
    f32x4 x[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) x[t] = ld16f(src + t * kWave * 4);
    const long long live = (end + kMassWaves * kRows - 1) / (kMassWaves * kRows);
    const float nl = joined_lse(reinterpret_cast<const float2*>(p.part) + it.wh * p.nchunks * kGqa, live, s_pair);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[t][i] = weight(x[t][i], nl);
    store_mass<NT>(p, it.wh, unit * kRows, x);
}

// S > 1.  Per unit, token of the launch and head, (max, sum).
template <int DT, int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_stats(const MassParams p) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const Item it = item_of(p);
    constexpr int kRows = Unit<DT, NT>::kRows;
    const long long unit = it.chunk * kMassWaves + wv;
    if (unit * kRows >= visible_end(p, it.w)) return;
    Unit<DT, NT> u;
    u.load(p, it.w, it.hkv, unit * kRows);
    const long long units = (long long)p.nchunks * kMassWaves;
    float2* part = reinterpret_cast<float2*>(p.part) + (it.wh * p.ns * units + unit) * kGqa;
    for (int s = 0; s < p.ns; ++s) {
        float m = -DV_INF, l = 0.0f;
        if (u.f1 >= 0) {
            f32x4 x[NT];
            u.scores(p, it.w, p.s0 + s,
                     [&](int f, u32x4(&q)[kPieces<DT>]) { stored_query<DT>(p, f, it.w, p.s0 + s, it.hkv, q); }, x);
            row_stats<NT>(x, m, l);
        }
        if (lane < kGqa) part[s * units * kGqa + lane] = make_float2(m, l);
    }
}

// Block (sequence, KV head, token): the log-sum-exp of its heads.
__global__ __launch_bounds__(kMassThreads) void dv_mass_lse(const MassParams p, int unit_rows) {
    __shared__ float2 s_pair[kMassThreads];
    const long long row = blockIdx.x;  // (w * Hkv + hkv) * ns + s
    const int w = (int)(row / ((long long)p.ns * p.Hkv));
    const long long units = (long long)p.nchunks * kMassWaves;
    const long long live = (visible_end(p, w) + unit_rows - 1) / unit_rows;
    const float nl = joined_lse(reinterpret_cast<const float2*>(p.part) + row * units * kGqa, live, s_pair);
    if (threadIdx.x < kGqa) p.lse[row * kGqa + threadIdx.x] = nl;
}

template <int DT, int NT>
__global__ __launch_bounds__(kMassThreads) void dv_mass_apply(const MassParams p) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const Item it = item_of(p);
    constexpr int kRows = Unit<DT, NT>::kRows;
    const long long unit = it.chunk * kMassWaves + wv;
    if (unit * kRows >= visible_end(p, it.w)) {
        store_decayed<NT>(p, it.wh, unit * kRows);
        return;
    }
    Unit<DT, NT> u;
    u.load(p, it.w, it.hkv, unit * kRows);
    const float* lse = p.lse + it.wh * p.ns * kGqa + (lane & 15);
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (u.f1 >= 0) {
        for (int s = 0; s < p.ns; ++s) {
            f32x4 x[NT];
            u.scores(p, it.w, p.s0 + s,
                     [&](int f, u32x4(&q)[kPieces<DT>]) { stored_query<DT>(p, f, it.w, p.s0 + s, it.hkv, q); }, x);
            const float nl = lse[s * kGqa];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] += weight(x[t][i], nl);
        }
    }
    store_mass<NT>(p, it.wh, unit * kRows, acc);
}

// ---- launches --------------------------------------------------------------------

namespace {

// Tiles per wave.
template <int DT> constexpr int kTilesOf = DT == kF32 ? 2 : 4;
int tiles_of(int dtype) { return dtype == kF32 ? kTilesOf<kF32> : kTilesOf<kBF16>; }

// Stored scores of a decode step take a quarter of a 16-bit K cache's bytes; block tables
// far wider than the sequences would make that a lot of workspace for nothing, so
// from here on the second pass computes the scores again.
constexpr long long kMaxScoreBytes = 1ll << 30;

struct MassWs {
    bool stored;
    int tokens;  // per launch
    long long chunks;
    size_t rq, part, lse, scores, total;
};

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

MassWs mass_ws(int dtype, int F, int W, int S, int Hkv, long long max_rows) {
    MassWs l{};
    const long long rows = (long long)kMassWaves * tiles_of(dtype) * 16;
    const long long wh = (long long)W * Hkv;
    l.chunks = (max_rows + rows - 1) / rows;
    const long long score_bytes = wh * l.chunks * rows * kGqa * 4;
    l.stored = S == 1 && score_bytes <= kMaxScoreBytes;
    l.tokens = S < kMassTokens ? S : kMassTokens;
    if (l.stored) {
        l.part = up256((size_t)(wh * l.chunks * kGqa * 8));
        l.scores = (size_t)score_bytes;
    } else {
        l.rq = up256((size_t)F * wh * kGqa * S * kHeadDim * (dtype == kF32 ? 4 : 2));
        l.part = up256((size_t)(wh * l.tokens * l.chunks * kMassWaves * kGqa * 8));
        l.lse = up256((size_t)(wh * l.tokens * kGqa * 4));
    }
    l.total = l.rq + l.part + l.lse + l.scores;
    return l;
}

template <int DT>
hipError_t mass_go(MassParams p, const MassWs& l, hipStream_t stream) {
    constexpr int NT = kTilesOf<DT>;
    constexpr int kRows = kMassWaves * NT * 16;  // stream rows of a block
    const unsigned wh = (unsigned)(p.W * p.Hkv);
    const dim3 block(kMassThreads);
    const dim3 keys((unsigned)(wh * l.chunks)), outs((unsigned)(wh * ((p.C + kRows - 1) / kRows)));
    hipError_t e;
    p.nchunks = (int)l.chunks;
    if (p.S == 0) {  // no token votes: every row only decays
        if (outs.x) hipLaunchKernelGGL((dv_mass_apply<DT, NT>), outs, block, 0, stream, p);
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
    RopeParams rp{};
    rp.out = p.rq;
    rp.q = p.q;
    rp.cosv = p.cosv;
    rp.sinv = p.sinv;
    rp.F = p.F;
    rp.W = p.W;
    rp.Hq = p.Hq;
    rp.S = p.S;
    rp.E = kHeadDim;
    rp.R = p.R;
    if ((e = launch_rope(DT, rp, stream)) != hipSuccess) return e;
    for (int s0 = 0; s0 < p.S; s0 += l.tokens) {
        p.s0 = s0;
        p.ns = p.S - s0 < l.tokens ? p.S - s0 : l.tokens;
        if (keys.x) {
            hipLaunchKernelGGL((dv_mass_stats<DT, NT>), keys, block, 0, stream, p);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        hipLaunchKernelGGL(dv_mass_lse, dim3(wh * (unsigned)p.ns), block, 0, stream, p, NT * 16);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        if (outs.x) hipLaunchKernelGGL((dv_mass_apply<DT, NT>), outs, block, 0, stream, p);
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
    switch (dtype) {
        case kBF16: return mass_go<kBF16>(p, l, stream);
        case kF16: return mass_go<kF16>(p, l, stream);
        case kF32: return mass_go<kF32>(p, l, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace dv
