// Serving-side kernels of paged caches:
//  * dv_block_tables -- where a step's tokens go: block tables, positions and cache slots
//    from the sequences' lengths and a stack of free pages.
//  * dv_kv_append8   -- new keys (rotated) and values rounded to E4M3 in their slots, one
//    power-of-two scale per page and KV head.
#include "dv_common.h"
#include "dv_device.h"

namespace dv {

namespace {

// ---- block tables ------------------------------------------------------------------
//
// Everything follows from two prefix sums over the sequences: the pages that ended
// sequences give back (which come first, so that this step can hand them out again), and
// the pages that the others need.  One workgroup of sixteen waves: a step of some
// hundred sequences is bound by the latency of its few dependent reads (lengths, table
// entries, stack entries), not by bytes.
constexpr int kTabThreads = 1024;
constexpr int kTabWaves = kTabThreads / kWave;
// Tokens that the table workgroup still places itself; with more, a second launch places
// them (the workgroup writes about 12 bytes per token at one CU's rate).
constexpr int kTabTokens = 4096;

// Exclusive prefix sum of v over the workgroup's threads; total: the sum.
__device__ inline long long block_sum_excl(long long v, long long* s_part, long long& total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    long long incl = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const long long o = __shfl_up(incl, d, kWave);
        if (lane >= d) incl += o;
    }
    __syncthreads();  // s_part is free
    if (lane == kWave - 1) s_part[wv] = incl;
    __syncthreads();
    long long before = 0;
    total = 0;
    for (int i = 0; i < kTabWaves; ++i) {
        if (i < wv) before += s_part[i];
        total += s_part[i];
    }
    return before + incl - v;
}

__device__ inline int pages_of(long long n, int bs) { return (int)((n + bs - 1) / bs); }

// Position and slot of packed token t: its sequence is the last one that starts at or
// before it among those with tokens (cu ascending, cu[0] = 0).
__device__ inline void place_token(const TablesParams& p, const int* cu, const int* starts, int t) {
    int pos = -1;
    long long slot = -1;
    if (t < cu[p.W]) {
        int lo = 0, hi = p.W - 1;  // the first w with t < cu[w + 1]
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (t < cu[mid + 1]) hi = mid;
            else lo = mid + 1;
        }
        if (starts[lo] >= 0) {
            pos = starts[lo] + (t - cu[lo]);
            const int lp = pos / p.bs;
            const int page = p.bt[(long long)lo * p.maxB + lp];
            if (page >= 0 && page < p.nblocks) slot = (long long)page * p.bs + (pos - lp * p.bs);
        }
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
}

__global__ __launch_bounds__(kTabThreads) void dv_block_tables(const TablesParams p) {
    extern __shared__ __align__(16) int s_tab[];
    __shared__ long long s_part[kTabWaves];
    int* s_cu = s_tab;                 // [W + 1]
    int* s_start = s_cu + p.W + 1;     // [W] length before the step (0: ended), then the start
    int* s_off = s_start + p.W;        // [W] first stack entry given back, then pages needed before w
    int* s_got = s_off + p.W;          // [W] pages given back, then pages taken
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int W = p.W;
    long long room = (long long)p.maxB * p.bs;
    room = room < 0x7fffffffll ? room : 0x7fffffffll;  // positions are 32-bit
    // each thread takes a run of sequences
    const int per = (W + kTabThreads - 1) / kTabThreads;
    const int w0 = tid * per < W ? tid * per : W, w1 = w0 + per < W ? w0 + per : W;
    const int cnt0 = *p.count;
    const long long count = cnt0 < 0 ? 0 : cnt0 < p.nblocks ? cnt0 : p.nblocks;

    // 1. lengths, packed token counts and pages given back
    long long gone = 0, toks = 0;
    for (int w = w0; w < w1; ++w) {
        long long len = p.lengths[w];
        len = len < 0 ? 0 : len < room ? len : room;
        const int nw = p.new_tokens[w];
        const int g = nw < 0 ? pages_of(len, p.bs) : 0;
        s_start[w] = nw < 0 ? -1 : (int)len;
        s_cu[w + 1] = nw > 0 ? nw : 0;
        s_got[w] = g;
        gone += g;
        toks += nw > 0 ? nw : 0;
    }
    long long gone_all, toks_all, need_all;
    long long g_at = block_sum_excl(gone, s_part, gone_all);
    long long t_at = block_sum_excl(toks, s_part, toks_all);
    for (int w = w0; w < w1; ++w) {
        const long long at = count + g_at;
        s_off[w] = (int)(at < p.nblocks ? at : p.nblocks);
        g_at += s_got[w];
    }
    __syncthreads();
    // 2. ended sequences' pages go on the stack, a wave per sequence
    if (gone_all > 0) {
        for (int w = wv; w < W; w += kTabWaves) {
            const int g = s_got[w], at = s_off[w];
            for (int b = lane; b < g; b += kWave)
                if (at + b < p.nblocks) p.stack[at + b] = p.bt[(long long)w * p.maxB + b];
        }
    }
    const long long have = count + gone_all < p.nblocks ? count + gone_all : p.nblocks;
    __syncthreads();
    // 3. packed starts, and the pages the others need
    long long need = 0;
    for (int w = w0; w < w1; ++w) {
        const int nw = s_cu[w + 1];
        const int len = s_start[w];
        const long long end = t_at + nw;
        // a sequence that has not the room in its table row, or whose tokens run past the
        // output, asks for nothing (-1: refused)
        const bool fits = len >= 0 && (long long)len + nw <= room && end <= p.T;
        const int nd = fits ? pages_of((long long)len + nw, p.bs) - pages_of(len, p.bs) : len < 0 ? 0 : -1;
        s_got[w] = nd;
        need += nd > 0 ? nd : 0;
        t_at = end;
        s_cu[w + 1] = (int)(end < 0x7fffffff ? end : 0x7fffffff);
    }
    long long n_at = block_sum_excl(need, s_part, need_all);
    long long taken = 0;
    for (int w = w0; w < w1; ++w) {
        const int nd = s_got[w];
        const bool ok = nd == 0 || (nd > 0 && n_at + nd <= have);
        s_off[w] = (int)(n_at < have ? n_at : have);
        if (nd > 0) n_at += nd;
        s_got[w] = ok ? nd : -1;
        taken += ok ? nd : 0;
    }
    long long taken_all;
    block_sum_excl(taken, s_part, taken_all);
    if (tid == 0) {
        s_cu[0] = 0;
        p.cu[0] = 0;
        *p.count_out = (int)(have - taken_all);
    }
    __syncthreads();
    for (int w = w0; w < w1; ++w) {
        const int len = s_start[w];
        const bool ok = s_got[w] >= 0;
        const int nw = s_cu[w + 1] - s_cu[w];
        p.cu[w + 1] = s_cu[w + 1];
        p.starts[w] = ok ? len : -1;
        p.lengths_out[w] = len < 0 ? 0 : ok ? len + nw : len;
    }
    // 4. the pages themselves, from the top of the stack down
    for (int w = wv; w < W; w += kTabWaves) {
        const int got = s_got[w];
        if (got <= 0) continue;
        const int held = pages_of(s_start[w], p.bs);
        for (int j = lane; j < got; j += kWave)
            p.bt[(long long)w * p.maxB + held + j] = p.stack[have - 1 - s_off[w] - j];
    }
    if (p.T > kTabTokens) return;
    __syncthreads();
    for (int w = w0; w < w1; ++w)
        if (s_got[w] < 0) s_start[w] = -1;
    __syncthreads();
    for (int t = tid; t < p.T; t += kTabThreads) place_token(p, s_cu, s_start, t);
}

__global__ __launch_bounds__(256) void dv_place_tokens(const TablesParams p) {
    extern __shared__ __align__(16) int s_tab[];
    int* s_cu = s_tab;
    int* s_start = s_cu + p.W + 1;
    for (int w = threadIdx.x; w <= p.W; w += 256) {
        s_cu[w] = p.cu[w];
        if (w < p.W) s_start[w] = p.starts[w];
    }
    __syncthreads();
    const int stride = (int)gridDim.x * 256;
    for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < p.T; t += stride)
        place_token(p, s_cu, s_start, (int)t);
}

// ---- quantising append ---------------------------------------------------------------

// E4M3 bytes of eight floats of magnitude at most 448 (or NaN), ties to even.
__device__ inline u32x2 to_fp8(const float (&x)[8]) {
    u32x2 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
        r[i] = (uint32_t)w;
    }
    return r;
}

__device__ inline void from_fp8(u32x2 b, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)b[i], false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)b[i], true);
        x[4 * i] = lo[0];
        x[4 * i + 1] = lo[1];
        x[4 * i + 2] = hi[0];
        x[4 * i + 3] = hi[1];
    }
}

// The smallest exponent byte b >= 1 with amax <= 448 * 2^(b - 127) (448 = 1.75 * 2^8).
__device__ inline int exponent_of(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int b = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b < 1 ? 1 : b;
}

template <int DT>
__device__ inline float round_to(float f) {
    return Tr<DT>::tof(Tr<DT>::fromf(f));
}

// Eight elements of X as floats, 16 bytes at a time where `vec` says they are aligned.
template <int DT>
__device__ inline void load8(const typename Tr<DT>::raw* x, bool vec, float (&f)[8]) {
    using raw = typename Tr<DT>::raw;
    raw r[8];
    if (vec) {
        constexpr int V = (int)sizeof(r) / 16;
        u32x4 t[V];
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = ld16(reinterpret_cast<const unsigned char*>(x) + 16 * i);
        __builtin_memcpy(r, t, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = x[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Tr<DT>::tof(r[i]);
}

// Dims [d0, d0 + 8) of token t's key (rotated as dv_kv_append does, PyTorch's rounding) or
// value for head h, as the storage type holds them.
template <int DT, int CDT, bool K>
__device__ inline void load_row8(const Append8Params& p, int t, int h, int d0, float (&x)[8]) {
#pragma clang fp contract(off)
    using raw = typename Tr<DT>::raw;
    using craw = typename Tr<CDT>::raw;
    const int w = t / p.S, s = t - w * p.S;
    const long long* st = K ? p.kst : p.vst;
    const raw* row = reinterpret_cast<const raw*>(K ? p.k : p.v) + w * st[0] + h * st[1] + s * st[2];
    load8<DT>(row + d0, p.vec, x);
    if constexpr (K) {
        if (d0 < p.R) {
            constexpr bool kF32Math = DT == kF32 || CDT == kF32;
            const int half = p.R >> 1;
            const long long co = w * p.cs[0] + s * p.cs[1];
            const craw* cr = reinterpret_cast<const craw*>(p.cosv) + co;
            const craw* sr = reinterpret_cast<const craw*>(p.sinv) + co;
            auto turn = [&](float v, float o, float c, float sn, bool first) {
                float a = v * c, b = o * sn;
                if constexpr (!kF32Math) {
                    a = round_to<DT>(a);
                    b = round_to<DT>(b);
                }
                return round_to<DT>(first ? a - b : a + b);
            };
            if ((half & 7) == 0) {  // the run lies in one half
                const bool first = d0 < half;
                float o[8], c[8], sn[8];
                load8<DT>(row + (first ? d0 + half : d0 - half), p.vec, o);
                load8<CDT>(cr + d0, p.vec, c);
                load8<CDT>(sr + d0, p.vec, sn);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = turn(x[i], o[i], c[i], sn[i], first);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int d = d0 + i;
                    if (d >= p.R) continue;
                    const bool first = d < half;
                    const float o = Tr<DT>::tof(row[first ? d + half : d - half]);
                    x[i] = turn(x[i], o, Tr<CDT>::tof(cr[d]), Tr<CDT>::tof(sr[d]), first);
                }
            }
        }
    }
    // fp16: magnitudes above 61440 are held as 61440 (the next E4M3 number, 65536, is
    // none of fp16); infinities are no E4M3 numbers and become NaN
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = __builtin_fabsf(x[i]);
        if constexpr (DT == kF16) {
            if (a > 61440.0f && a < DV_INF) x[i] = __builtin_copysignf(61440.0f, x[i]);
        }
        if (!(a < DV_INF)) x[i] = __builtin_nanf("");
    }
}

constexpr int kAppWaves = 16;     // most waves of a workgroup
constexpr int kAppRows = 16;      // rows of a page that a wave holds in registers: 4 passes of 4

}  // namespace

// A run: tokens of the call in consecutive rows of one page.  A workgroup finds the runs
// that start among its `tile` tokens, then its waves take (run, KV head, K or V) units:
// the largest magnitude of the written rows gives the page's exponent, rows that were
// held under a smaller one are rounded again, and the new rows are written.  That needs
// the page to itself: all slots of the call are compared with the run's page (they are
// few bytes beside the rows), and where other tokens of the page exist -- a page in
// several runs, a slot named twice -- the first token's workgroup writes them all, the
// last token of a slot winning.
template <int DT, int CDT>
__global__ __launch_bounds__(kAppWaves * kWave) void dv_kv_append8(const Append8Params p, int T) {
    __shared__ int s_run[64];      // first tokens of the runs
    __shared__ int s_nrun;
    __shared__ int s_other[64];    // 1: the run's page has tokens outside it; 2: earlier ones
    const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6), nthreads = blockDim.x;
    const long long nslots = (long long)p.nblocks * p.bs;
    const int t0 = blockIdx.x * p.tile;
    auto slot_at = [&](int t) {
        const long long s = p.slots[t];
        return s >= 0 && s < nslots ? s : -1;
    };
    // 1. runs of the tile (at most 64 tokens: one wave)
    if (wv == 0) {
        const int t = t0 + lane;
        bool start = false;
        if (lane < p.tile && t < T) {
            const long long s = slot_at(t);
            const long long before = t > 0 ? slot_at(t - 1) : -1;
            start = s >= 0 && (before < 0 || s != before + 1 || s % p.bs == 0);
        }
        const uint64_t m = ballot(start);
        if (start) s_run[__builtin_popcountll(m & ((1ull << lane) - 1ull))] = t;
        if (lane == 0) s_nrun = __builtin_popcountll(m);
        s_other[lane] = 0;
    }
    __syncthreads();
    const int nrun = s_nrun;
    if (nrun == 0) return;
    auto run_of = [&](int i, int& t, long long& base, int& row0, int& n) {
        t = s_run[i];
        const long long s = p.slots[t];
        row0 = (int)(s % p.bs);
        base = s - row0;
        n = 0;
        const int most = p.bs - row0 < T - t ? p.bs - row0 : T - t;
        while (n < most) {  // consecutive slots, 64 at a time
            const int k = n + lane;
            const uint64_t b = ballot(k < most && p.slots[t + (k < most ? k : 0)] == s + k);
            const int good = b == ~0ull ? 64 : __builtin_ctzll(~b);
            n += good;
            if (good < 64) break;
        }
    };
    // 2. tokens of the runs' pages elsewhere in the call
    for (int i = 0; i < nrun; ++i) {
        int t, row0, n;
        long long base;
        run_of(i, t, base, row0, n);
        int found = 0;
        for (int u = tid; u < T; u += nthreads)
            if ((unsigned long long)(p.slots[u] - base) < (unsigned long long)p.bs && (u < t || u >= t + n))
                found |= u < t ? 2 : 1;
        if (found) atomicOr(&s_other[i], found);
    }
    __syncthreads();
    // 3. units
    const int g = lane >> 4, d0 = (lane & 15) * 8;
    const int nwaves = nthreads >> 6;
    const int units = nrun * p.Hkv * 2;
    for (int u = blockIdx.y * nwaves + wv; u < units; u += gridDim.y * nwaves) {
        const int i = u / (2 * p.Hkv), hk = u - i * 2 * p.Hkv;
        const int h = hk >> 1;
        const bool isk = (hk & 1) == 0;
        const int other = s_other[i];
        if (other & 2) continue;  // the page's first token lies in an earlier run
        int t, row0, n;
        long long base;
        run_of(i, t, base, row0, n);
        const int page = (int)(base / p.bs);
        unsigned char* cache = (isk ? p.kc : p.vc) + ((base * p.Hkv + h) << 7);
        const long long rstride = (long long)p.Hkv << 7;
        unsigned char* sc = (isk ? p.ks : p.vs) + (long long)page * p.Hkv + h;
        const int old = *sc;
        // rows [r0, r1) of the page may have a token; tok(r): the one written there (-1: none)
        const int r0 = other ? 0 : row0, r1 = other ? p.bs : row0 + n;
        auto tok = [&](int r) {
            if (!other) return r >= row0 && r < row0 + n ? t + r - row0 : -1;
            int last = -1;
            for (int k = t; k < T; ++k)
                if (p.slots[k] == base + r) last = k;
            return last;
        };
        float x[kAppRows / 4][8];
        int rt[kAppRows / 4];
        auto load_block = [&](int rb) {
#pragma unroll
            for (int q = 0; q < kAppRows / 4; ++q) {
                const int r = rb + q * 4 + g;
                rt[q] = r < r1 ? tok(r) : -1;
                const int tt = rt[q] >= 0 ? rt[q] : t;
                if (isk) load_row8<DT, CDT, true>(p, tt, h, d0, x[q]);
                else load_row8<DT, CDT, false>(p, tt, h, d0, x[q]);
            }
        };
        float amax = 0.0f;
        bool first_row = false;
        for (int rb = r0; rb < r1; rb += kAppRows) {
            load_block(rb);
#pragma unroll
            for (int q = 0; q < kAppRows / 4; ++q) {
                first_row |= rt[q] >= 0 && rb + q * 4 + g == 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float a = __builtin_fabsf(x[q][e]);
                    amax = rt[q] >= 0 && a > amax ? a : amax;  // (NaN compares false)
                }
            }
        }
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d, kWave));
        const bool fresh = ballot(first_row) != 0 || old == 255;
        const int want = exponent_of(amax);
        const int b = fresh || want > old ? want : old;
        if (!fresh && b > old) {
            // rows held under the smaller exponent
            for (int rb = 0; rb < p.bs; rb += 4) {
                const int r = rb + g;
                if (r < p.bs && tok(r) < 0) {
                    u32x2* row = reinterpret_cast<u32x2*>(cache + r * rstride + d0);
                    float y[8];
                    from_fp8(*row, y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_ldexpf(y[e], old - b);
                    *row = to_fp8(y);
                }
            }
        }
        for (int rb = r0; rb < r1; rb += kAppRows) {
            if (r1 - r0 > kAppRows) load_block(rb);
#pragma unroll
            for (int q = 0; q < kAppRows / 4; ++q) {
                const int r = rb + q * 4 + g;
                if (rt[q] < 0) continue;
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_ldexpf(x[q][e], 127 - b);
                *reinterpret_cast<u32x2*>(cache + r * rstride + d0) = to_fp8(y);
            }
        }
        if (lane == 0 && b != old) *sc = (unsigned char)b;
    }
}

namespace {

template <int DT, int CDT>
hipError_t append8_go(Append8Params p, hipStream_t stream) {
    const long long T = (long long)p.W * p.S;
    // a token per workgroup while there are few (their pages are found and written side by
    // side), then about a page of tokens
    p.tile = T <= 512 ? 1 : p.bs < 16 ? 16 : p.bs < 64 ? p.bs : 64;
    const int units = 2 * p.Hkv;
    const int waves = units < kAppWaves ? units : kAppWaves;
    const dim3 grid((unsigned)((T + p.tile - 1) / p.tile), (unsigned)((units + waves - 1) / waves));
    hipLaunchKernelGGL((dv_kv_append8<DT, CDT>), grid, dim3(waves * kWave), 0, stream, p, (int)T);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_append8(int dtype, int rope_dtype, const Append8Params& base, hipStream_t stream) {
    Append8Params p = base;
    const int es = dtype == kF32 ? 4 : 2, cs = rope_dtype == kF32 ? 4 : 2;
    auto al = [](const void* q) { return ((uintptr_t)q & 15) == 0; };
    bool vec = al(p.k) && al(p.v) && al(p.cosv) && al(p.sinv);
    for (int i = 0; i < 3; ++i) vec = vec && p.kst[i] * es % 16 == 0 && p.vst[i] * es % 16 == 0;
    for (int i = 0; i < 2; ++i) vec = vec && p.cs[i] * cs % 16 == 0;
    p.vec = vec;
    const bool f32rope = rope_dtype == kF32;
    switch (dtype) {
        case kBF16: return f32rope ? append8_go<kBF16, kF32>(p, stream) : append8_go<kBF16, kBF16>(p, stream);
        case kF16: return f32rope ? append8_go<kF16, kF32>(p, stream) : append8_go<kF16, kF16>(p, stream);
        case kF32: return append8_go<kF32, kF32>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_block_tables(const TablesParams& p, hipStream_t stream) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    static std::atomic<unsigned long long> attr_done{0};
    e = once_per_device(attr_done, device, [] {
        return hipFuncSetAttribute(reinterpret_cast<const void*>(&dv_block_tables),
                                   hipFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)((4 * kMaxTableSeqs + 1) * sizeof(int)));
    });
    if (e != hipSuccess) return e;
    static std::atomic<unsigned long long> place_done{0};
    e = once_per_device(place_done, device, [] {
        return hipFuncSetAttribute(reinterpret_cast<const void*>(&dv_place_tokens),
                                   hipFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)((2 * kMaxTableSeqs + 1) * sizeof(int)));
    });
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(dv_block_tables, dim3(1), dim3(kTabThreads), (size_t)(4 * p.W + 1) * sizeof(int), stream, p);
    e = hipGetLastError();
    if (e != hipSuccess || p.T <= kTabTokens) return e;
    const long long blocks = ((long long)p.T + 255) / 256;
    hipLaunchKernelGGL(dv_place_tokens, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256),
                       (size_t)(2 * p.W + 1) * sizeof(int), stream, p);
    return hipGetLastError();
}

}  // namespace dv
