// Serving-side kernels of paged caches:
//  * dv_block_tables -- where a step's tokens go: block tables, positions and cache slots
//    from the sequences' lengths and a stack of free pages.
//  * dv_kv_append8   -- new keys (rotated) and values rounded to E4M3 in their slots, one
//    power-of-two scale per page and KV head.
#include <type_traits>

#include "dv_common.h"
#include "dv_device.h"

namespace dv {

namespace {

typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
typedef __attribute__((ext_vector_type(2))) short i16x2;

// ---- block tables ------------------------------------------------------------------
//
// Everything follows from two prefix sums over the sequences: the pages that ended
// sequences give back (which come first, so that this step can hand them out again), and
// the pages that the others need.  One workgroup of sixteen waves: a step of some
// hundred sequences is bound by the latency of its few dependent reads (lengths, table
// entries, stack entries) and its scans, not by bytes.  64 sequences, one token each: 7.5
// us; 512 of up to 32000 tokens, 24 of which end and 32 of which add up to 512 tokens:
// 16.6 us (22 with a wave per sequence for the pages), and 3.9 for the places of its 8000
// tokens.
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
    __shared__ int s_gone[kTabThreads];  // ended sequences with pages
    __shared__ int s_ngone;
    int* s_cu = s_tab;                 // [W + 1]
    int* s_start = s_cu + p.W + 1;     // [W] length before the step (-1: ended), then the start
    int* s_off = s_start + p.W;        // [W] first stack entry given back, then pages needed before w
    int* s_got = s_off + p.W;          // [W] pages given back, then pages taken
    const int tid = threadIdx.x;
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
    // 2. ended sequences' pages go on the stack: eight sequences at a time by all threads
    if (gone_all > 0) {
        for (int k = 0; k < per; ++k) {
            if (tid == 0) s_ngone = 0;
            __syncthreads();
            const int w = w0 + k;
            if (w < w1 && s_got[w] > 0) s_gone[atomicAdd(&s_ngone, 1)] = w;  // (in any order)
            __syncthreads();
            const int ngone = s_ngone;
            for (int i = 0; i < ngone; i += 8) {
                int most = 0;
                for (int j = 0; j < 8; ++j) {
                    const int g = i + j < ngone ? s_got[s_gone[i + j]] : 0;
                    most = g > most ? g : most;
                }
                for (int b = tid; b < most; b += kTabThreads) {
                    int page[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int v = s_gone[i + j < ngone ? i + j : i];
                        page[j] = b < s_got[v] ? p.bt[(long long)v * p.maxB + b] : 0;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int v = s_gone[i + j < ngone ? i + j : i];
                        const int at = s_off[v];
                        if (i + j < ngone && b < s_got[v] && at < p.nblocks - b) p.stack[at + b] = page[j];
                    }
                }
            }
            __syncthreads();
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
    // 4. the pages themselves, from the top of the stack down, a thread each: the page
    // before which e others are needed goes to the last sequence that starts at or before e
    const int pages = (int)(need_all < have ? need_all : have);
    for (int e = tid; e < pages; e += kTabThreads) {
        int lo = 0, hi = W - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s_off[mid] <= e) lo = mid;
            else hi = mid - 1;
        }
        const int j = e - s_off[lo];
        if (j < s_got[lo])
            p.bt[(long long)lo * p.maxB + pages_of(s_start[lo], p.bs) + j] = p.stack[have - 1 - e];
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

// fp16: magnitudes above 61440 are held as 61440 (the next E4M3 number, 65536, is none of
// fp16); infinities are no E4M3 numbers and become NaN.
template <int DT>
__device__ inline float storable(float x) {
    const float a = __builtin_fabsf(x);
    if constexpr (DT == kF16) {
        if (a > 61440.0f && a < DV_INF) x = __builtin_copysignf(61440.0f, x);
    }
    return a < DV_INF ? x : __builtin_nanf("");
}

// Eight elements that are held under the exponent byte `old`, which is too small, rounded
// again under b (0: an empty page, which holds zeros whatever its bytes are).
__device__ inline void raise_row(unsigned char* at, int old, int b) {
    u32x2* row = reinterpret_cast<u32x2*>(at);
    float y[8];
    from_fp8(*row, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = old ? __builtin_amdgcn_ldexpf(y[e], old - b) : 0.0f;
    *row = to_fp8(y);
}

// One element of a rotated key, evaluated as PyTorch does in the rows' type.
template <int DT, int CDT>
__device__ inline float turn(float v, float o, float c, float sn, bool first) {
#pragma clang fp contract(off)
    float a = v * c, b = o * (first ? -sn : sn);
    if constexpr (DT != kF32 && CDT != kF32) {
        a = round_to<DT>(a);
        b = round_to<DT>(b);
    }
    return round_to<DT>(a + b);
}

// Dims d0 and d0 + 1 of token t's key (rotated) or value for head h.
template <int DT, int CDT>
__device__ inline void load_pair(const Append8Params& p, bool isk, int t, int h, int d0, float (&x)[2]) {
    using raw = typename Tr<DT>::raw;
    using craw = typename Tr<CDT>::raw;
    const int w = t / p.S, s = t - w * p.S;
    const long long* st = isk ? p.kst : p.vst;
    const raw* row = reinterpret_cast<const raw*>(isk ? p.k : p.v) + w * st[0] + h * st[1] + s * st[2];
    const long long co = w * p.cs[0] + s * p.cs[1];
    const int half = p.R >> 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = d0 + i;
        x[i] = Tr<DT>::tof(row[d]);
        if (isk && d < p.R) {
            const bool first = d < half;
            x[i] = turn<DT, CDT>(x[i], Tr<DT>::tof(row[first ? d + half : d - half]),
                                 Tr<CDT>::tof(reinterpret_cast<const craw*>(p.cosv)[co + d]),
                                 Tr<CDT>::tof(reinterpret_cast<const craw*>(p.sinv)[co + d]), first);
        }
        x[i] = storable<DT>(x[i]);
    }
}

// Eight elements of a row as its type has them, in whole 16-byte words.
template <int DT>
struct Row8 {
    static constexpr int kWords = (int)sizeof(typename Tr<DT>::raw) * 2;
    uint32_t w[kWords];
    __device__ inline void load(const unsigned char* base, uint32_t off) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
            const u32x4 v = ld16(base + off + 16 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
        }
    }
    __device__ inline float at(int i) const {
        if constexpr (DT == kF32) return __uint_as_float(w[i]);
        else return Tr<DT>::tof((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
    }
    // magnitudes, as integers of the type's width (which order like them), folded into m
    __device__ inline void fold(uint32_t& m) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (DT == kF32) {
                const uint32_t u = w[i] & 0x7fffffffu;
                m = u > m ? u : m;
            } else {
                const u16x2 u = __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu);
                m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), u));
            }
        }
    }
    // the same over finite ones; fp16: magnitudes above 61440 become that
    __device__ inline void fold_finite(uint32_t& m) {
        constexpr uint32_t kInf = DT == kF32 ? 0x7f800000u : DT == kF16 ? 0x7c00u : 0x7f80u;
        constexpr int kPer = DT == kF32 ? 1 : 2, kBits = 32 / kPer;
#pragma unroll
        for (int i = 0; i < kWords; ++i)
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                uint32_t u = (w[i] >> (kBits * j)) & (DT == kF32 ? 0x7fffffffu : 0x7fffu);
                if constexpr (DT == kF16) {
                    if (u > 0x7b80u && u < kInf) {
                        w[i] = (w[i] & ~(0x7fffu << (kBits * j))) | (0x7b80u << (kBits * j));
                        u = 0x7b80u;
                    }
                }
                m = u < kInf && u > m ? u : m;
            }
    }
    // E4M3 bytes of the elements times 2^(127 - b), ties to even: magnitudes are at most
    // 448 then, infinities and NaN become NaN
    __device__ inline u32x2 bytes(int b) const {
        if constexpr (DT == kF32) {
            const float f = __uint_as_float(b < 254 ? (uint32_t)(254 - b) << 23 : 0x400000u);  // (2^-127 is subnormal)
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(w[e]) * f;
            return to_fp8(y);
        } else {
            const float f = __uint_as_float((uint32_t)b << 23);  // (these divide)
            u32x2 r;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                i16x2 o = {0, 0};
                if constexpr (DT == kBF16) {
                    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(bf16x2, w[2 * i]), f, false);
                    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(bf16x2, w[2 * i + 1]), f, true);
                } else {
                    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, __builtin_bit_cast(f16x2, w[2 * i]), f, false);
                    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, __builtin_bit_cast(f16x2, w[2 * i + 1]), f, true);
                }
                r[i] = __builtin_bit_cast(uint32_t, o);
            }
            return r;
        }
    }
};

// The largest magnitude that fold() may find without a look at single elements, and a
// folded magnitude as a float.
template <int DT>
__device__ inline bool beyond(uint32_t m) {
    if constexpr (DT == kF32) return m > 0x7f7fffffu;
    const uint32_t k = DT == kF16 ? 0x7b80u : 0x7f7fu;
    return (m & 0xffffu) > k || (m >> 16) > k;
}

// x rotated where `rot`: o holds the elements half a rotation away, c and sn the angles.
template <int DT, int CDT>
__device__ inline void rotate8(Row8<DT>& x, const Row8<DT>& o, const Row8<CDT>& c, const Row8<CDT>& sn, bool first,
                               bool rot) {
#pragma clang fp contract(off)
    if constexpr (DT == kF32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t y = __float_as_uint(turn<DT, CDT>(x.at(i), o.at(i), c.at(i), sn.at(i), first));
            x.w[i] = rot ? y : x.w[i];
        }
    } else if constexpr (DT == kF16 && CDT == kF16) {
        // products and sum in their own type: what rounding the exact products, and the
        // sum in 24 bits, to 11 bits gives as well
        const uint32_t flip = first ? 0x80008000u : 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x2 a = __builtin_bit_cast(f16x2, x.w[i]) * __builtin_bit_cast(f16x2, c.w[i]);
            const f16x2 b = __builtin_bit_cast(f16x2, o.w[i]) * __builtin_bit_cast(f16x2, sn.w[i] ^ flip);
            const uint32_t y = __builtin_bit_cast(uint32_t, a + b);
            x.w[i] = rot ? y : x.w[i];
        }
    } else {
        using T2 = std::conditional_t<DT == kBF16, bf16x2, f16x2>;
        using T1 = std::conditional_t<DT == kBF16, __bf16, _Float16>;
        const uint32_t flip = first ? 0x80000000u : 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a[2], b[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                a[j] = x.at(2 * i + j) * c.at(2 * i + j);
                b[j] = o.at(2 * i + j) * __uint_as_float(__float_as_uint(sn.at(2 * i + j)) ^ flip);
            }
            if constexpr (CDT != kF32) {
                const T2 ra = {(T1)a[0], (T1)a[1]}, rb = {(T1)b[0], (T1)b[1]};
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    a[j] = (float)ra[j];
                    b[j] = (float)rb[j];
                }
            }
            const T2 y = {(T1)(a[0] + b[0]), (T1)(a[1] + b[1])};
            x.w[i] = rot ? __builtin_bit_cast(uint32_t, y) : x.w[i];
        }
    }
}

// The exponent byte of a page with the byte `old` after rows of magnitude m (see fold) were
// written, row 0 among them where `first_row`.
template <int DT>
__device__ inline int exponent_after(uint32_t m, bool first_row, int old) {
    if constexpr (DT != kF32) m = (m & 0xffffu) > (m >> 16) ? m & 0xffffu : m >> 16;
    const float amax = DT == kF32 ? __uint_as_float(m) : Tr<DT>::tof((typename Tr<DT>::raw)m);
    const int want = exponent_of(amax);
    return first_row || old == 255 || want > old ? want : old;
}

constexpr int kAppRows = 16;      // most rows of a page that a wave holds in registers: 4 times 4

// Tokens that have their pages to themselves, rows and angles in whole 16-byte words, 16
// lanes a row.  kPass > 0: the run's rows [row0, row0 + n) of one KV head, kPass * 4 at
// once, without a branch (those behind the run's end repeat its last row).  kPass = 0: one
// row of four KV heads from h on.  cache, sc: the page's bytes and exponents of head h.
// `team` waves share a run, the caller being the rank-th of them: s_max has their largest
// magnitudes, and all waves of the workgroup come here (store: false where only for that).
template <int DT, int CDT, bool kTurn, int kPass>
__device__ inline void write_run(const Append8Params& p, bool isk, int t, int row0, int n, int h, int lane,
                                 unsigned char* cache, unsigned char* sc, int team = 1, int rank = 0,
                                 uint32_t* s_max = nullptr, bool store = true) {
    constexpr bool kHeads = kPass == 0;
    constexpr int kQ = kHeads ? 1 : kPass, kRows = 4 * kQ;
    constexpr uint32_t kEs = sizeof(typename Tr<DT>::raw), kCs = sizeof(typename Tr<CDT>::raw);
    asm("" : "+v"(lane));  // (else lane offsets are held in registers over all units)
    const int g = lane >> 4, d0 = (lane & 15) * 8;
    const long long rstride = (long long)p.Hkv << 7;
    // (a head behind the last one repeats the last)
    const int hg = kHeads ? (h + g < p.Hkv ? g : p.Hkv - 1 - h) : 0;
    const int old = sc[hg];
    const int w = t / p.S, sq = t - w * p.S;
    const long long* st = isk ? p.kst : p.vst;
    const unsigned char* src = reinterpret_cast<const unsigned char*>(isk ? p.k : p.v) +
                               (w * st[0] + h * st[1] + sq * st[2]) * (long long)kEs;
    const unsigned char* ac = reinterpret_cast<const unsigned char*>(p.cosv);
    const unsigned char* as = reinterpret_cast<const unsigned char*>(p.sinv);
    const long long ao = (w * p.cs[0] + sq * p.cs[1]) * (long long)kCs;
    const int half = p.R >> 1;
    const bool rot = kTurn && d0 < p.R, first = d0 < half;
    // byte offsets of a lane's row and of its angles; rows are less than 2^27 bytes apart
    const uint32_t rs = (uint32_t)((kHeads ? st[1] : st[2]) * kEs), cs = (uint32_t)(p.cs[1] * kCs);
    const uint32_t lx = d0 * kEs, lo = (rot ? first ? d0 + half : d0 - half : d0) * kEs, lc = (rot ? d0 : 0) * kCs;
    Row8<DT> x[kQ];
    auto load_block = [&](int rb) {
        Row8<DT> o[kQ];
        Row8<CDT> c[kQ], sn[kQ];
        const unsigned char* at = src + rb * (long long)rs;
        const unsigned char* atc = ac + ao + rb * (long long)cs;
        const unsigned char* ats = as + ao + rb * (long long)cs;
        const int last = n - 1 - rb;
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
            const uint32_t r = kHeads ? hg : q * 4 + g < last ? q * 4 + g : last;
            x[q].load(at, r * rs + lx);
            if constexpr (kTurn) {
                const uint32_t ro = kHeads ? lc : r * cs + lc;
                o[q].load(at, r * rs + lo);
                c[q].load(atc, ro);
                sn[q].load(ats, ro);
            }
        }
        uint32_t m = 0;
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
            if constexpr (kTurn) rotate8<DT, CDT>(x[q], o[q], c[q], sn[q], first, rot);
            x[q].fold(m);
        }
        if (ballot(beyond<DT>(m))) {  // rare
            m = 0;
#pragma unroll
            for (int q = 0; q < kQ; ++q) x[q].fold_finite(m);
        }
        return m;
    };
    auto larger = [](uint32_t a, uint32_t b) {
        if constexpr (DT == kF32) return a > b ? a : b;
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                      __builtin_bit_cast(u16x2, b)));
    };
    uint32_t m = 0;
    const int rb0 = rank * kRows, rstep = team * kRows;
    if constexpr (kHeads) m = load_block(0);
    else
        for (int rb = rb0; rb < n; rb += rstep) m = larger(m, load_block(rb));
#pragma unroll
    for (int d = 1; d < (kHeads ? 16 : kWave); d <<= 1) m = larger(m, (uint32_t)__shfl_xor((int)m, d, kWave));
    if (team > 1) {
        if (lane == 0) s_max[rank] = m;
        __syncthreads();
        m = 0;
        for (int i = 0; i < team; ++i) m = larger(m, s_max[i]);
        if (!store) return;
    }
    const int b = exponent_after<DT>(m, row0 == 0, old);
    const bool mine = !kHeads || hg == g;
    const bool raise = b > old && row0 != 0 && old != 255;
    if constexpr (kHeads) {
        if (ballot(raise)) {
            for (int r = 0; r < p.bs; ++r)
                if (raise && mine && r != row0) raise_row(cache + r * rstride + (g << 7) + d0, old, b);
        }
    } else if (raise) {
        for (int r = rank * 4 + g; r < p.bs; r += team * 4)
            if (r < row0 || r >= row0 + n) raise_row(cache + r * rstride + d0, old, b);
    }
    const uint32_t rnext = kHeads ? 128u : (uint32_t)rstride;
    auto store_block = [&](int rb) {
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
            const uint32_t r = q * 4 + g;
            const u32x2 y = x[q].bytes(b);
            if (kHeads ? mine : (int)r < n - rb)
                *reinterpret_cast<u32x2*>(cache + (row0 + rb) * rstride + (r * rnext + d0)) = y;
        }
    };
    if (kHeads || n <= rstep) {
        store_block(rb0);
    } else {
        for (int rb = rb0; rb < n; rb += rstep) {
            load_block(rb);
            store_block(rb);
        }
    }
    if ((lane & (kHeads ? 15 : 63)) == 0 && rank == 0 && mine && b != old) sc[hg] = (unsigned char)b;
}

constexpr int kAppWaves = 8;      // most waves of a workgroup
constexpr int kAppTile = 32;      // most tokens of a workgroup
constexpr int kAppScan = 8;       // slots that a thread compares at a time
constexpr int kAppMap = 1024;     // rows of a page whose last tokens are listed

}  // namespace

// A run: tokens of the call in consecutive rows of one page.  A workgroup finds the runs
// that start among its `tile` tokens, then its waves take (run, KV head, K or V) units:
// the largest magnitude of the written rows gives the page's exponent, rows that were
// held under a smaller one are rounded again, and the new rows are written.  That needs
// the page to itself: all slots of the call are compared with the run's page (they are
// few bytes beside the rows), and where other tokens of the page exist -- a page in
// several runs, a slot named twice -- the first token's workgroup writes them all, the
// last token of a slot winning.
//
// Bound by its chain of dependent reads while the call is small: slots (the tile's and
// those compared, read together), then rows, angles and exponents together.  32 single
// tokens, 8 KV heads: 6 us; 548 tokens of decodes and prompts, 4 KV heads, pages of 24: 9 us
// (138 with a page of tokens to a workgroup, whose decodes went one after the other).
// Large calls are bound by VALU issue and the chain, 2 rounds of units a wave, and near the
// end by HBM: 8188 tokens of four prompts, 8 KV heads, 54 MB: 25 us cold, 17 warm (3.2
// TB/s), 55 with branches around the loads, which waited for each.  The comparisons grow
// with the square of the call: 32768 tokens take 64 us, of which about 20 are those.
template <int DT, int CDT>
__global__ __launch_bounds__(kAppWaves * kWave, DT == kF32 || CDT == kF32 ? 2 : 4)
void dv_kv_append8(const Append8Params p, int T) {
    __shared__ uint32_t s_max[2][kAppWaves];
    __shared__ int s_tok[kAppMap];
    __shared__ int s_other[kAppTile];  // 1: the run's page has tokens outside it; 2: earlier ones
    const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6), nthreads = blockDim.x;
    const long long nslots = (long long)p.nblocks * p.bs;
    const bool small = nslots <= 0xffffffffll;
    auto row_of = [&](long long s) { return small ? (int)((uint32_t)s % (uint32_t)p.bs) : (int)(s % p.bs); };
    // workgroups in a row take tiles a page apart: runs recur at that distance, and
    // workgroups go round the XCDs and CUs, some of which would else find runs only
    const int groups = (int)gridDim.x / p.apart;
    const int t0 = ((int)blockIdx.x % groups * p.apart + (int)blockIdx.x / groups) * p.tile;
    if (t0 >= T) return;
    // lane i of each wave: the slot of token t0 - 1 + i
    long long win = -1;
    {
        const int t = t0 - 1 + lane;
        if (t >= 0 && t < T) win = p.slots[t];
    }
    long long sl[kAppScan];
    auto load_scan = [&](int c) {
#pragma unroll
        for (int j = 0; j < kAppScan; ++j) {
            const int u = c + j * nthreads + tid;
            sl[j] = p.slots[u < T ? u : T - 1];
        }
    };
    load_scan(0);
    if (tid < kAppTile) s_other[tid] = 0;
    __syncthreads();
    // 1. runs of the tile.  more: bit i: lane i's token goes on with lane i - 1's run.
    const bool in = win >= 0 && win < nslots;
    const int wrow = in ? row_of(win) : 0;
    const bool head = p.S < T && (t0 - 1 + lane) % p.S == 0;  // runs end with a sequence's tokens
    const long long prev = __shfl_up(win, 1, kWave);
    const uint64_t more = ballot(in && lane > 0 && prev == win - 1 && wrow != 0 && !head);
    uint64_t starts = ballot(in && lane > 0 && lane <= p.tile) & ~more;
    const int nrun = __builtin_popcountll(starts);
    if (nrun == 0) return;
    auto run_at = [&](int l, int& t, long long& base, int& row0, int& n) {
        t = t0 - 1 + l;
        row0 = __builtin_amdgcn_readlane(wrow, l);
        const long long s = ((long long)__builtin_amdgcn_readlane((int)(win >> 32), l) << 32) |
                            (uint32_t)__builtin_amdgcn_readlane((int)win, l);
        base = s - row0;
        const uint64_t stop = l < 63 ? ~more >> (l + 1) : 0;  // (zeros come in behind lane 63)
        n = 1 + (stop ? __builtin_ctzll(stop) : 63 - l);
        if (l + n < 64) return;
        // the window's end: on by what memory says, 64 tokens at a time
        const int here = p.S - t % p.S;
        const int most = p.bs - row0 < here ? p.bs - row0 : here;
        while (n < most) {
            const int k = n + lane;
            const uint64_t bm = ballot(k < most && p.slots[t + (k < most ? k : 0)] == s + k);
            const int good = bm == ~0ull ? 64 : __builtin_ctzll(~bm);
            n += good;
            if (good < 64) break;
        }
    };
    // 2. tokens of the runs' pages elsewhere in the call
    for (int c = 0; c < T; c += kAppScan * nthreads) {
        if (c > 0) load_scan(c);
        uint64_t left = starts;
        for (int i = 0; i < nrun; ++i) {
            int t, row0, n, found = 0;
            long long base;
            run_at(__builtin_ctzll(left), t, base, row0, n);
            left &= left - 1;
#pragma unroll
            for (int j = 0; j < kAppScan; ++j) {
                const int u = c + j * nthreads + tid;
                const bool same = (unsigned long long)sl[j] - (unsigned long long)base < (unsigned long long)p.bs;
                if (same && u < T && (u < t || u >= t + n)) found |= u < t ? 2 : 1;
            }
            if (found) atomicOr(&s_other[i], found);
        }
    }
    __syncthreads();
    // 3. units: K or V of a run, of one KV head, or of four heads where the run is a token
    const int nwaves = (nthreads >> 6) * (int)gridDim.y;
    int next = (int)blockIdx.y * (nthreads >> 6) + wv;  // this wave's unit, counted from the run's first
    int turn = 0;  // which of s_max: a wave may be a unit behind
    for (int i = 0; i < nrun; ++i, starts &= starts - 1) {
        const int other = s_other[i];
        if (other & 2) continue;  // the page's first token lies in an earlier run
        int t, row0, n;
        long long base;
        run_at(__builtin_ctzll(starts), t, base, row0, n);
        if (other) {  // the last token of each row (a maximum: the same in any order)
            __syncthreads();  // an earlier run's list is done with
            for (int r = tid; r < kAppMap; r += nthreads) s_tok[r] = -1;
            __syncthreads();
            for (int k = t + tid; k < T; k += nthreads) {
                const unsigned long long r = (unsigned long long)p.slots[k] - (unsigned long long)base;
                if (r < (unsigned long long)p.bs && r < (unsigned long long)kAppMap) atomicMax(&s_tok[r], k);
            }
            __syncthreads();
        }
        const bool fast = !other && p.vec, heads = fast && n == 1;
        const int per_kv = heads ? (p.Hkv + 3) >> 2 : p.Hkv;
        // a run of many rows is shared by `team` waves, which wait for one another: every
        // wave goes through the same number of units then
        const int team = fast && n > kAppRows ? p.team : 1;
        const int rank = wv % team, ahead = team > 1 ? wv / team : 0;
        const int stride = nwaves / team;
        int u0 = team > 1 ? (int)blockIdx.y * ((nthreads >> 6) / team) : next;
        for (; u0 < 2 * per_kv; u0 += stride) {
            const bool store = u0 + ahead < 2 * per_kv;
            const int u = store ? u0 + ahead : u0;
            const bool isk = u < per_kv;
            const int h = (isk ? u : u - per_kv) * (heads ? 4 : 1);
            const int page = small ? (int)((uint32_t)base / (uint32_t)p.bs) : (int)(base / p.bs);
            unsigned char* cache = (isk ? p.kc : p.vc) + ((base * p.Hkv + h) << 7);
            const long long rstride = (long long)p.Hkv << 7;
            unsigned char* sc = (isk ? p.ks : p.vs) + (long long)page * p.Hkv + h;
            if (fast) {
                // (without a rotation there are no angles to read)
                const bool turns = isk && p.R > 0;
                if (heads) {
                    if (turns) write_run<DT, CDT, true, 0>(p, isk, t, row0, n, h, lane, cache, sc);
                    else write_run<DT, CDT, false, 0>(p, isk, t, row0, n, h, lane, cache, sc);
                } else {
                    uint32_t* sm = s_max[turn] + wv - rank;
                    turn ^= team > 1;
                    if (turns)
                        write_run<DT, CDT, true, 4>(p, isk, t, row0, n, h, lane, cache, sc, team, rank, sm, store);
                    else
                        write_run<DT, CDT, false, 4>(p, isk, t, row0, n, h, lane, cache, sc, team, rank, sm, store);
                }
                continue;
            }
            // The general form: a row at a time, two elements a lane, read again to be written.
            // Rows [r0, r1) of the page may have a token; tok(r): the one written there (-1: none).
            const int r0 = other ? 0 : row0, r1 = other ? p.bs : row0 + n;
            auto tok = [&](int r) {
                if (!other) return r >= row0 && r < row0 + n ? t + r - row0 : -1;
                if (r < kAppMap) return uniform(s_tok[r]);
                int last = -1;
                for (int k = t; k < T; k += kWave) {
                    const uint64_t at = ballot(k + lane < T && p.slots[k + lane < T ? k + lane : t] == base + r);
                    if (at) last = k + 63 - __builtin_clzll(at);
                }
                return last;
            };
            float x[2];
            const int old = *sc;
            float amax = 0.0f;
            for (int r = r0; r < r1; ++r) {
                const int rt = tok(r);
                if (rt < 0) continue;
                load_pair<DT, CDT>(p, isk, rt, h, 2 * lane, x);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float a = __builtin_fabsf(x[e]);
                    amax = a > amax ? a : amax;  // (NaN compares false)
                }
            }
#pragma unroll
            for (int d = 1; d < kWave; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d, kWave));
            const bool fresh = tok(0) >= 0 || old == 255;
            const int want = exponent_of(amax);
            const int b = fresh || want > old ? want : old;
            const bool raise = !fresh && b > old;
            for (int r = raise ? 0 : r0; r < (raise ? p.bs : r1); ++r) {
                const int rt = tok(r);
                uint16_t* to = reinterpret_cast<uint16_t*>(cache + r * rstride) + lane;
                if (rt >= 0) {
                    load_pair<DT, CDT>(p, isk, rt, h, 2 * lane, x);
                    x[0] = __builtin_amdgcn_ldexpf(x[0], 127 - b);
                    x[1] = __builtin_amdgcn_ldexpf(x[1], 127 - b);
                } else if (raise) {
                    const f32x2 y = __builtin_amdgcn_cvt_pk_f32_fp8((int)*to, false);
                    x[0] = old ? __builtin_amdgcn_ldexpf(y[0], old - b) : 0.0f;
                    x[1] = old ? __builtin_amdgcn_ldexpf(y[1], old - b) : 0.0f;
                } else {
                    continue;
                }
                *to = (uint16_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
            }
            if (lane == 0 && b != old) *sc = (unsigned char)b;
        }
        if (team == 1) next = u0 - 2 * per_kv;
    }
}

namespace {

template <int DT, int CDT>
hipError_t append8_go(Append8Params p, hipStream_t stream) {
    const long long T = (long long)p.W * p.S;
    // as many workgroups as the device holds at a time: a token each while there are few
    p.tile = (int)((T + 511) / 512 < kAppTile ? (T + 511) / 512 : kAppTile);
    // waves that share a long run: one for each kAppRows rows of a page
    p.team = 1;
    while (p.team < kAppWaves && p.team * kAppRows < p.bs) p.team *= 2;
    const int units = 2 * p.Hkv;
    const int waves = units * p.team < kAppWaves ? units * p.team : kAppWaves;
    const int teams = waves / p.team;
    const long long tiles = (T + p.tile - 1) / p.tile;
    // the heads of long runs are spread over workgroups where few have a run
    const long long busy = T / (p.tile > p.bs ? p.tile : p.bs) + 1;
    long long split = (units + teams - 1) / teams;
    if (split > 512 / busy) split = 512 / busy > 1 ? 512 / busy : 1;
    const long long apart = (p.bs + p.tile - 1) / p.tile;
    p.apart = (int)(apart < tiles ? apart : tiles);
    const dim3 grid((unsigned)((tiles + p.apart - 1) / p.apart * p.apart), (unsigned)split);
    hipLaunchKernelGGL((dv_kv_append8<DT, CDT>), grid, dim3(waves * kWave), 0, stream, p, (int)T);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_append8(int dtype, int rope_dtype, const Append8Params& base, hipStream_t stream) {
    Append8Params p = base;
    if (p.S == 1) {  // one row of tokens
        p.S = p.W;
        p.W = 1;
        p.kst[2] = p.kst[0];
        p.vst[2] = p.vst[0];
        p.cs[1] = p.cs[0];
    }
    if (p.W == 1) p.kst[0] = p.vst[0] = p.cs[0] = 0;  // (strides of a single index say nothing)
    if (p.Hkv == 1) p.kst[1] = p.vst[1] = 0;
    const int es = dtype == kF32 ? 4 : 2, cs = rope_dtype == kF32 ? 4 : 2;
    auto al = [](const void* q) { return ((uintptr_t)q & 15) == 0; };
    auto step = [](long long n, int bytes, bool near) {
        return n * bytes % 16 == 0 && (!near || (n >= 0 && n * bytes < (1ll << 27)));
    };
    bool vec = al(p.k) && al(p.v);
    for (int i = 0; i < 3; ++i) vec = vec && step(p.kst[i], es, i > 0) && step(p.vst[i], es, i > 0);
    // (the elements half a rotation away start at whole words: half of R is eight or a multiple)
    if (p.R > 0)
        vec = vec && p.R % 16 == 0 && al(p.cosv) && al(p.sinv) && step(p.cs[0], cs, false) && step(p.cs[1], cs, true);
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
