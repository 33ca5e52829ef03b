// gfx950 decode attention with fused query RoPE over a paged cache held in 8 bits:
// E4M3 bytes [num_blocks, block_size, Hkv, 128] and one exponent byte b per page and KV
// head, so that a cached element is byte * 2^(b - 127) (b = 0: zero, 255: NaN).  Rows, views,
// rotation, work split and merge are the 16-bit decode's (dv_decode.hip).
//
//  * One wave owns one KV head and its 16 query heads of one row over a range of the
//    row's keys; up to eight such waves (KV heads, pick_hpw8) make a workgroup.
//  * A stage is 32 keys: 4 KiB of K, 4 KiB of V and the 64 exponent bytes of its rows,
//    moved by nine direct-to-LDS loads into a ring of two stages private to the wave.  The
//    exponents travel with their rows, so pages of any size may end inside a stage.
//  * K bytes are widened to the 16-bit MFMA operand (every E4M3 number is one of bf16 and
//    of fp16): S^T = K Q^T on 16x16x32 MFMA, and the page's 2^(b - 127) multiplies the
//    fp32 score.  V^T comes from the transposing 8-bit LDS read, widened to bf16, and V's
//    2^(b - 127) multiplies the probability before it is rounded (a power of two: the
//    rounding is the same with and without).
//  * Precision: bf16 calls take one operand for Q and P, as the 16-bit decode does, and
//    hold partial results as fp16 under a power of two per row (store_partial).  fp16
//    calls take Q as it is against K in fp16, and P as a bf16 pair hi + lo (16 bits).
//    fp32 calls take Q, its row scaled by a power of two, as an fp16 pair and P as three
//    bf16 numbers, 24 bits either way: the products with exact K and V lose nothing that
//    fp32 arithmetic keeps (V under exponents below 18 aside, whose weights' last part
//    leaves bf16).
//
// Bound by HBM on long caches and by starts on short ones: 4 x 131072 keys of 8 KV heads
// in fp16, 1.07 GB, 169 us (6.4 TB/s; reads alone reach 6.9); 32 ragged sequences of 1k -
// 8k keys in bf16, 320 MB, 60 us (5.3); one sequence of 3001 keys 10.8; 96 fp32 rows over 73
// MB 65, half of it VALU issue and MFMAs (24 of a stage's 40 are P's three parts).
#pragma once

#include "dv_common.h"
#include "dv_device.h"
#include "dv_schedule.h"
#include "dv_stream.h"

namespace dv {
namespace q8 {

constexpr int kRowB = kHeadDim;                 // bytes of a cached row
constexpr int kTile = kStep * kRowB;            // 32 rows of K (or V)
constexpr int kScaleB = 64 * 4;                 // exponent bytes of 32 K rows, then of 32 V rows, a word each
constexpr int kStage = 2 * kTile + kScaleB;
constexpr int kLoads = 9;                       // direct-to-LDS loads per stage

// A wave holds NT query tiles (16 heads of a token each), one or, in 16-bit types, two;
// two waves to a SIMD, with two stages each in LDS and accumulators in VGPRs (as the
// kernels' file is compiled).  fp32 with two tiles (whose operands alone are 128
// registers) had the SIMD to itself: 100 MB of cache took 39 us for two tokens, where rows
// of one token take 17.5 us each.  (A launch's schedule lies in LDS too, 8 bytes a row above
// 64 rows: from 688 rows on, 112 / 304 with one / two KV heads to a workgroup, fewer than
// eight waves fit a CU.)
constexpr int kWaves = 8;                       // per CU
constexpr int kRing = 2;
constexpr int kWaveLds = kRing * kStage + stream::kPc * 4;

// MFMA operands of a query (or probability) value: 16-bit parts that sum to it.
template <int DT> constexpr int kQParts = DT == kF32 ? 2 : 1;
template <int DT> constexpr int kPParts = DT == kF32 ? 3 : DT == kF16 ? 2 : 1;
template <int DT> constexpr int kKType = DT == kBF16 ? kBF16 : kF16;

// Eight E4M3 bytes as four words of 16-bit pairs, exactly.
template <int T16>
__device__ inline u32x4 widen8(u32x2 b) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int w = (int)b[i];
        if constexpr (T16 == kF16) {
            r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
            r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
        } else {
            r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
            r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
        }
    }
    return r;
}

__device__ inline u32x2 lds_read8_at(uint32_t addr) {
    typedef __attribute__((address_space(3))) const u32x2 lds_u32x2;
    return *(lds_u32x2*)(uintptr_t)addr;
}

// Transposing 8-bit read: within each 16-lane block, result lane i, byte j = byte i % 8 at
// the address supplied by block lane i / 8 + 2 * j.
__device__ inline u32x2 lds_read_tr8_at(uint32_t addr) {
    typedef __attribute__((ext_vector_type(2))) int i32x2;
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(uintptr_t)addr));
}

// Where the 16-byte pieces of a row lie: XOR-swizzled by the row, so that the rows that
// one operand read touches spread over the 64 banks (K: rows n, a lane each; V: rows
// g * 4 + j and 16 + g * 4 + j of a 16-lane block).
__device__ inline int swz_k(int row) { return (row >> 1) & 7; }
__device__ inline int swz_v(int row) { return ((row >> 1) & 3) | ((row >> 2) & 4); }

// 2^(b - 127) of an exponent byte (0 and 255: settle_row).
__device__ inline float power_of(uint32_t b) { return __uint_as_float(b << 23); }

// This lane's byte offset from a stage's row bases: load i moves rows 8i .. 8i + 7 (lane /
// 8); with i odd (K) or above 1 (V) the swizzle is the same but for bit 2: offset ^ 64.
__device__ inline uint32_t lane_offset(const DecodeParams& p) {
    const int lane = threadIdx.x & 63;
    const int r = lane >> 3, c = lane & 7;
    return (uint32_t)r * ((uint32_t)p.Hkv * kRowB) + (uint32_t)((c ^ swz_k(r)) * 16);
}

// Issues the loads of the stage holding keys [l, l + 32) into the ring slot at LDS address
// sbase; returns the visibility mask of its keys.  P2 (pages of a power of two of at
// least 16 rows): a stage of 32 visible keys that starts at a multiple of 16 lies in at most
// two pages, one for each half, so its row bases are scalar and no lane looks a row up
// (32 ragged sequences: 9 + 140 instructions per stage instead of 9 + 250).
template <bool P2, bool kAsk, bool kAny>
__device__ inline uint32_t issue(const DecodeParams& p, const stream::View& v, uint32_t lo, const int* pc,
                                 uint32_t sbase, int l) {
    const int lane = threadIdx.x & 63;
    // (positions are 31 bits: rows of views that start behind that are absent)
    const uint32_t pos0 = (uint32_t)v.off + (uint32_t)l;
    const bool whole = l + kStep <= v.b && pos0 <= 0x7fffffffu - (uint32_t)(kStep - 1);
    if constexpr (P2) {
        if ((!kAsk || p.bs_shift >= 4) && whole && stream::full_stage_in_cache((int)pos0, p.bs_shift, v.lp0)) {
            const uint32_t pos = pos0, in = (1u << p.bs_shift) - 1u;
            const int pg0 = uniform(pc[(int)(pos >> p.bs_shift) - v.lp0]);
            const int pg1 = uniform(pc[(int)((pos + 16) >> p.bs_shift) - v.lp0]);
            if (pg0 >= 0 && pg1 >= 0) {
                const uint32_t r0 = ((uint32_t)pg0 << p.bs_shift) + (pos & in);
                const uint32_t r1 = ((uint32_t)pg1 << p.bs_shift) + ((pos + 16) & in);
                const unsigned long long row[2] = {(unsigned long long)(r0 * (uint32_t)p.Hkv + (uint32_t)v.hkv) << 7,
                                                   (unsigned long long)(r1 * (uint32_t)p.Hkv + (uint32_t)v.hkv) << 7};
                const unsigned long long kb = (unsigned long long)v.k, vb = (unsigned long long)v.v;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned long long r =
                        row[i >> 1] + (unsigned long long)((uint32_t)(i & 1) * ((uint32_t)p.Hkv << 10));
                    dma16_kv(kb + r, (i & 1) ? lo ^ 64u : lo, sbase + (uint32_t)(i * 1024), vb + r,
                             (i >> 1) ? lo ^ 64u : lo, sbase + (uint32_t)(kTile + i * 1024));
                }
                const uint32_t pg = (uint32_t)((lane & 16) ? pg1 : pg0);
                dma1((lane < 32 ? p.ks : p.vs) + (pg * (uint32_t)p.Hkv + (uint32_t)v.hkv),
                     sbase + (uint32_t)(2 * kTile));
                return 0xffffffffu;
            }
        }
    }
    const int ol = opaque_tid() & 63;  // (lane-dependent values are computed here, not held)
    // Pages of 16 rows or more: 32 visible keys lie in at most three, whose bases are scalar;
    // a lane picks its row's.  (kAny: stages that the first form does not take are common.)
    if (kAny && p.bs >= 16 && p.bs < (1 << 28) && whole) {
        uint32_t q, r;
        page_split(p, pos0, q, r);
        const int at = uniform((int)q) - v.lp0, r0 = uniform((int)r);
        const int more = (r0 + kStep - 1 >= p.bs ? 1 : 0) + (r0 + kStep - 1 >= 2 * p.bs ? 1 : 0);
        if (at >= 0 && at + more < stream::kPc) {
            int pg[3];
#pragma unroll
            for (int j = 0; j < 3; ++j) pg[j] = uniform(pc[at + (j < more ? j : more)]);
            if (pg[0] >= 0 && pg[1] >= 0 && pg[2] >= 0) {
                uint32_t base[3];  // of key 0, as if its page held all keys
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    base[j] = ((uint32_t)(pg[j] - j) * (uint32_t)p.bs + (uint32_t)r0) * (uint32_t)p.Hkv +
                              (uint32_t)v.hkv;
                const int t1 = p.bs - r0, t2 = 2 * p.bs - r0;  // first keys of the second and third page
                auto pick = [&](int k, uint32_t a, uint32_t b, uint32_t c) { return k >= t1 ? k >= t2 ? c : b : a; };
                const uint32_t lrow = (uint32_t)(ol >> 3) * (uint32_t)p.Hkv;
                // piece of a row; the swizzle of other loads' rows differs in bit 2 (lane_offset)
                const uint32_t piece = (uint32_t)(((ol & 7) ^ swz_k(ol >> 3)) * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t row = pick(i * 8 + (ol >> 3), base[0], base[1], base[2]) + lrow +
                                         (uint32_t)(i * 8) * (uint32_t)p.Hkv;
                    const unsigned long long off = (unsigned long long)row * kRowB;
                    dma16(v.k + (off | ((i & 1) ? piece ^ 64u : piece)), sbase + (uint32_t)(i * 1024));
                    dma16(v.v + (off | ((i >> 1) ? piece ^ 64u : piece)), sbase + (uint32_t)(kTile + i * 1024));
                }
                const uint32_t page = pick(ol & 31, (uint32_t)pg[0], (uint32_t)pg[1], (uint32_t)pg[2]);
                dma1((ol < 32 ? p.ks : p.vs) + (page * (uint32_t)p.Hkv + (uint32_t)v.hkv),
                     sbase + (uint32_t)(2 * kTile));
                return 0xffffffffu;
            }
        }
    }
    // page and in-page offset of the row of key l + k, or page -1
    auto find = [&](int k, uint32_t& r) {
        const int pos = (int)(pos0 + (uint32_t)k);
        uint32_t q;
        page_split(p, (uint32_t)(pos > 0 ? pos : 0), q, r);
        const uint32_t idx = q - (uint32_t)v.lp0;
        const int page = pc[idx < (uint32_t)stream::kPc ? idx : (uint32_t)(stream::kPc - 1)];
        return l + k < v.b && pos >= 0 && idx < (uint32_t)stream::kPc ? page : -1;
    };
    const unsigned char* ka[4];
    const unsigned char* va[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = i * 8 + (ol >> 3);
        uint32_t r;
        const int page = find(k, r);
        const uint32_t row = ((uint32_t)page * (uint32_t)p.bs + r) * (uint32_t)p.Hkv + (uint32_t)v.hkv;
        const unsigned long long off = (unsigned long long)row * kRowB;
        const int pk = ((ol & 7) ^ swz_k(k)) * 16, pv = ((ol & 7) ^ swz_v(k)) * 16;
        ka[i] = page >= 0 ? v.k + off + pk : g_zero_row + pk;
        va[i] = page >= 0 ? v.v + off + pv : g_zero_row + pv;
    }
    uint32_t r;
    const int page = find(ol & 31, r);
    const unsigned char* sb = ol < 32 ? p.ks : p.vs;
    const unsigned char* sa = page >= 0 ? sb + ((uint32_t)page * (uint32_t)p.Hkv + (uint32_t)v.hkv) : g_zero_row;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        dma16(ka[i], sbase + (uint32_t)(i * 1024));
        dma16(va[i], sbase + (uint32_t)(kTile + i * 1024));
    }
    dma1(sa, sbase + (uint32_t)(2 * kTile));
    return (uint32_t)uniform((int)(uint32_t)ballot(page >= 0 && lane < 32));
}

// A query row's 16-bit MFMA operands: lane (g, n) holds dims c * 32 + g * 8 .. + 8 of head n.
// fp32: times 2^k, k such that the head's largest magnitude lies in [2^14, 2^15), as hi + lo:
// hi is within 2^-12 of the element, lo within 2^-12 of what hi leaves (or 2^-25 of 2^15);
// bias: k + 127.
template <int DT>
struct QOp {
    u32x4 q[kQParts<DT>][4];
    int bias;
};

// A score from the product with K's bytes and its row's exponent byte.  fp32: 2^-k with it in
// one step, so that neither leaves the floats where their product does not (one VALU
// instruction and an integer subtraction, as the multiplication by 2^(b - 127) takes).
template <int DT>
__device__ inline float score(float x, uint32_t e, const QOp<DT>& q) {
    if constexpr (DT == kF32) return __builtin_amdgcn_ldexpf(x, (int)e - q.bias);
    else return x * power_of(e);
}

// Eight consecutive elements as floats (16-byte aligned).
template <int DT>
__device__ inline void load_run8(const typename Tr<DT>::raw* x, float (&f)[8]) {
    if constexpr (DT == kF32) {
        const f32x4 a = ld16f(x), b = ld16f(x + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = a[i];
            f[4 + i] = b[i];
        }
    } else {
        const u32x4 a = ld16(x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = Tr<DT>::tof((uint16_t)(a[i] & 0xffffu));
            f[2 * i + 1] = Tr<DT>::tof((uint16_t)(a[i] >> 16));
        }
    }
}

// The rotated query of token `row` in view f, dims [d0, d0 + 8) of one head, in rotate_run's
// arithmetic; `wide`: the rotation pairs whole runs and cos/sin are 16-byte aligned.
template <int DT>
__device__ inline void rotated8(const typename Tr<DT>::raw* q, const float* cs, const float* sn, int R, int d0,
                                bool wide, typename Tr<DT>::raw (&r)[8]) {
#pragma clang fp contract(off)
    const int half = R >> 1;
    float x[8];
    load_run8<DT>(q + d0, x);
    if (!wide) {  // element by element (static indices: the run stays in registers)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = d0 + i;
            if (d < R) {
                const bool first = d < half;
                const int ci = first ? d : d - half;
                const float o = Tr<DT>::tof(q[first ? d + half : ci]);
                const float a = x[i] * cs[ci], b = o * sn[ci];
                x[i] = first ? a - b : a + b;
            }
        }
    } else if (d0 < R) {
        const bool first = d0 < half;
        const int ci = first ? d0 : d0 - half;
        float o[8], c[8], s[8];
        load_run8<DT>(q + (first ? d0 + half : ci), o);
        load_run8<kF32>(cs + ci, c);
        load_run8<kF32>(sn + ci, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = x[i] * c[i], b = o[i] * s[i];
            x[i] = first ? a - b : a + b;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = Tr<DT>::fromf(x[i]);
}

// A run's operands as loaded: the run, the one it pairs with, cos and sin.
template <int DT>
struct QRun {
    static constexpr int kWords = (int)sizeof(typename Tr<DT>::raw) / 2;  // 16-byte words of eight elements
    u32x4 x[kWords], o[kWords];
    f32x4 c[2], s[2];
    __device__ static inline float at(const u32x4 (&w)[kWords], int i) {
        if constexpr (DT == kF32) return __uint_as_float(w[i >> 2][i & 3]);
        else return Tr<DT>::tof((uint16_t)(w[0][i >> 1] >> (16 * (i & 1))));
    }
};

// The rotated query of token `row` in view f, a wave's 16 heads.  kAhead: the loads of all four
// runs are in flight at once, 96 registers; else a run at a time.  Kernels of two tokens to
// a wave take the first (24 sequences x 4 tokens, R = 128: 61.8 -> 57.0 us; decodes beside
// prompt chunks 182 -> 176); rows of one token wait for their stages longer than for the
// runs (batch and long decodes the same, fp32 69 -> 72).
template <int DT, int QM, int RM, bool kAhead>
__device__ inline void load_q(const DecodeParams& p, int row, int f, int hkv, QOp<DT>& o) {
#pragma clang fp contract(off)
    using raw = typename Tr<DT>::raw;
    // (addresses from an opaque lane: computed here, not held in registers from the start)
    const int lane = opaque_tid() & 63;
    const int g = lane >> 4, n = lane & 15;
    const int h = hkv * kGqa + n;
    const raw* q;
    long long co;
    if (QM == kQRotFull) {
        const int w = row / p.S, s = row - (row / p.S) * p.S;
        q = reinterpret_cast<const raw*>(p.q) + (((long long)w * p.Hq + h) * p.S + s) * kHeadDim;
        co = (((long long)f * p.W + w) * p.S + s) * p.R;
    } else {
        q = reinterpret_cast<const raw*>(p.q) + ((long long)row * p.Hq + h) * kHeadDim;
        co = ((long long)f * p.T + row) * (p.R >> 1);
    }
    const float *cs = p.cosv + co, *sn = p.sinv + co;
    const bool wide = (p.R & 15) == 0 &&
                      ((reinterpret_cast<uintptr_t>(p.cosv) | reinterpret_cast<uintptr_t>(p.sinv)) & 15) == 0;
    raw r[4][8];
    if (kAhead && wide && p.R > 0) {
        const int half = p.R >> 1;
        QRun<DT> u[4];
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {  // (lanes behind the rotation load their own run and the first angles)
            const int d0 = cc * 32 + g * 8;
            const bool rot = d0 < p.R, first = d0 < half;
            const int od = rot ? first ? d0 + half : d0 - half : d0, ci = rot ? first ? d0 : d0 - half : 0;
#pragma unroll
            for (int i = 0; i < QRun<DT>::kWords; ++i) {
                u[cc].x[i] = ld16(reinterpret_cast<const unsigned char*>(q + d0) + 16 * i);
                u[cc].o[i] = ld16(reinterpret_cast<const unsigned char*>(q + od) + 16 * i);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                u[cc].c[i] = ld16f(cs + ci + 4 * i);
                u[cc].s[i] = ld16f(sn + ci + 4 * i);
            }
        }
        compiler_fence();
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
            const int d0 = cc * 32 + g * 8;
            const bool rot = d0 < p.R, first = d0 < half;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = QRun<DT>::at(u[cc].x, i);
                const float a = x * u[cc].c[i >> 2][i & 3], b = QRun<DT>::at(u[cc].o, i) * u[cc].s[i >> 2][i & 3];
                const float y = first ? a - b : a + b;
                r[cc][i] = Tr<DT>::fromf(rot ? y : x);
            }
        }
    } else {
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
            compiler_fence();  // one run's loads at a time
            rotated8<DT>(q, cs, sn, p.R, cc * 32 + g * 8, wide, r[cc]);
        }
    }
    if constexpr (DT == kF32) {
        float amax = 0.0f;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = __builtin_fabsf(r[cc][i]);
                amax = a < DV_INF && a > amax ? a : amax;
            }
        amax = rows4_max(amax);
        int k = 15 - __builtin_amdgcn_frexp_expf(amax);  // amax = m * 2^e, m in [0.5, 1); 0: e = 0
        k = k < 100 ? k : 100;
        o.bias = k + 127;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float a = __builtin_amdgcn_ldexpf(r[cc][2 * t], k);
                const float b = __builtin_amdgcn_ldexpf(r[cc][2 * t + 1], k);
                const uint32_t hi = pack2<kF16>(a, b);
                o.q[0][cc][t] = hi;
                o.q[1][cc][t] = pack2<kF16>(a - Tr<kF16>::tof((uint16_t)(hi & 0xffffu)),
                                            b - Tr<kF16>::tof((uint16_t)(hi >> 16)));
            }
    } else {
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
#pragma unroll
            for (int t = 0; t < 4; ++t) o.q[0][cc][t] = (uint32_t)r[cc][2 * t] | ((uint32_t)r[cc][2 * t + 1] << 16);
    }
}

// P^T operands of a lane's eight probabilities times their rows' V scales, and the row
// sum's share of them.
template <int DT>
struct POp {
    u32x4 w[kPParts<DT>];
};

template <int DT>
__device__ inline POp<DT> p_scaled(const float (&pr)[8], const uint32_t (&vs)[8], float& l) {
    POp<DT> o;
    if constexpr (DT == kBF16) {
        // the normaliser sums the rounded weights, as p_operands does
        float ps = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ps = dot2_ones<kBF16>(pack2<kBF16>(pr[2 * i], pr[2 * i + 1]), ps);
        l += ps;
    } else {
        float ps = pr[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) ps += pr[i];
        l += ps;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = pr[2 * i] * power_of(vs[2 * i]), b = pr[2 * i + 1] * power_of(vs[2 * i + 1]);
#pragma unroll
        for (int k = 0; k < kPParts<DT>; ++k) {
            const uint32_t w = pack2<kBF16>(a, b);
            o.w[k][i] = w;
            if (k + 1 < kPParts<DT>) {
                a -= __uint_as_float(w << 16);
                b -= __uint_as_float(w & 0xffff0000u);
            }
        }
    }
    return o;
}

struct State {
    f32x4 o[8];  // O^T: lane (g, n) holds dims c * 16 + g * 4 + i of head n
    float m, l;
};

// This lane's LDS offsets within a stage (128-byte aligned): K operand slice 0 of row n
// (slice cc: ^ 32 cc; row 16 + n: 16 rows further, same swizzle), V^T operand slice 0
// (slice cc: ^ 16 cc), exponents.
struct ReadOff {
    uint32_t k, v, s;
};
__device__ inline ReadOff read_offsets() {
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, n = lane & 15;
    ReadOff o;
    o.k = (uint32_t)(n * kRowB + (((g >> 1) ^ swz_k(n)) * 16) + (g & 1) * 8);
    // k = g * 8 + j <-> key (j / 4) * 16 + g * 4 + j % 4, as the scores' lanes hold them
    const int j = n >> 1;
    const int row = (j >> 2) * 16 + g * 4 + (j & 3);
    o.v = (uint32_t)(kTile + row * kRowB + swz_v(row) * 16 + (n & 1) * 8);
    o.s = (uint32_t)(2 * kTile + g * 16);
    return o;
}

// Exponent bytes of this lane's eight K (or, 128 bytes further, V) rows.
__device__ inline void read_exponents(uint32_t at, uint32_t (&e)[8]) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        const u32x4 a = lds_read16_at(at + (uint32_t)(kb * 64));
#pragma unroll
        for (int i = 0; i < 4; ++i) e[kb * 4 + i] = a[i];
    }
}

// Exponents that are no power of two to multiply with: 0, an empty page, whose elements are
// zeros whatever its bytes are, and 255, no number.  A stage that has such rows among its keys
// gets them rewritten, as zeros or NaN under 2^0: so a NaN byte does not survive the first,
// and the weight 0 of a key that another tile sees stays 0 times the second (0 times infinity
// would be NaN).  e: the exponent of this lane's row: K row `lane`, V row lane - 32.
__device__ inline uint32_t exponent_at(uint32_t slot) {
    typedef __attribute__((address_space(3))) const uint32_t lds_w;
    return *(lds_w*)(uintptr_t)(slot + (uint32_t)(2 * kTile) + (uint32_t)(opaque_tid() & 63) * 4);
}
__device__ inline void settle_row(uint32_t slot, uint32_t e) {
    typedef __attribute__((address_space(3))) uint32_t lds_w;
    typedef __attribute__((address_space(3))) u32x4 lds_w4;
    const uint32_t lane = (uint32_t)(opaque_tid() & 63);
    if (e - 1u >= 254u) {
        const uint32_t x = e ? 0x7f7f7f7fu : 0u;
#pragma unroll
        for (int i = 0; i < kRowB / 16; ++i)
            *(lds_w4*)(uintptr_t)(slot + lane * kRowB + (uint32_t)(i * 16)) = u32x4{x, x, x, x};
        *(lds_w*)(uintptr_t)(slot + (uint32_t)(2 * kTile) + lane * 4) = 127u;
    }
    compiler_fence();
}

// One stage for NT tiles: scores, softmax, O^T += V^T P^T.  okm: the stage's keys that hold
// rows; mask[t]: those that tile t sees.
template <int DT, int NT>
__device__ inline void compute(State (&st)[NT], uint32_t slot, const ReadOff& ro, uint32_t okm,
                               const uint32_t (&mask)[NT], const QOp<DT> (&q)[NT], float l2scale) {
    f32x4 s[NT][2];
    uint32_t ks[8];
    uint32_t e = exponent_at(slot);
    while (true) {  // (twice where rows are rewritten; before the scores, the look at e would be waited for)
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const u32x4 k = widen8<kKType<DT>>(
                    lds_read8_at(((slot + ro.k) ^ (uint32_t)(cc * 32)) + (uint32_t)(kb * 16 * kRowB)));
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < kQParts<DT>; ++j) s[t][kb] = Tr<kKType<DT>>::mma(k, q[t].q[j][cc], s[t][kb]);
            }
        read_exponents(slot + ro.s, ks);
        if (!(ballot(e - 1u >= 254u) & (((uint64_t)okm << 32) | okm))) break;
        settle_row(slot, e);
        e = 127u;
    }
    POp<DT> pB[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[t][0][i] = score<DT>(s[t][0][i], ks[i], q[t]);
            s[t][1][i] = score<DT>(s[t][1][i], ks[4 + i], q[t]);
        }
        float pr[8];
        softmax32<false>(st[t].o, st[t].m, st[t].l, s[t][0], s[t][1], mask[t], l2scale, pr);
        uint32_t vs[8];
        read_exponents(slot + ro.s + 128, vs);
        pB[t] = p_scaled<DT>(pr, vs, st[t].l);
    }
    // a key that some tile sees and another does not takes part there with weight 0, which
    // a NaN would survive: its V is cleared for the tile that does not see it
    bool part = false;
    if constexpr (NT > 1) {
#pragma unroll
        for (int t = 0; t < NT; ++t) part |= (mask[t] & okm) != okm;
    }
    if (NT > 1 && part) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int cc = 0; cc < 8; ++cc) {
            const u32x4 v = widen8<kBF16>(lds_read_tr8_at((slot + ro.v) ^ (uint32_t)(cc * 16)));
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint32_t mg = mask[t] >> (g * 4);
                u32x4 x;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t b = mg >> ((i >> 1) * 16 + (i & 1) * 2);
                    x[i] = v[i] & (((b & 1u) ? 0xffffu : 0u) | ((b & 2u) ? 0xffff0000u : 0u));
                }
#pragma unroll
                for (int k = 0; k < kPParts<DT>; ++k) st[t].o[cc] = Tr<kBF16>::mma(x, pB[t].w[k], st[t].o[cc]);
            }
        }
    } else {
#pragma unroll
        for (int cc = 0; cc < 8; ++cc) {
            const u32x4 v = widen8<kBF16>(lds_read_tr8_at((slot + ro.v) ^ (uint32_t)(cc * 16)));
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < kPParts<DT>; ++k) st[t].o[cc] = Tr<kBF16>::mma(v, pB[t].w[k], st[t].o[cc]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) mfma_settle(st[t].o);
}

// A row group: ntok tokens of sequence w, the first being row `lin` of the token axis.
// NT = 1: a group is a row (token).  Varlen groups of several tokens come from the table
// of dv_varlen_groups: block rg % p.sub of entry rg / p.sub; entries of more tokens than
// the blocks hold are not this launch's.
struct Group {
    int w, lin, ntok;
};
template <int RM, int NT>
__device__ inline Group group_of(const DecodeParams& p, int rg) {
    Group g;
    if (RM == kRowVarlen) {
        const int e = rg / p.sub, b = (rg - e * p.sub) * NT;
        const int4 x = reinterpret_cast<const int4*>(p.vgroups)[e];
        const int n = x.y <= p.sub * NT ? x.y - b : 0;
        g.w = x.z;
        g.lin = x.x + b;
        g.ntok = n < 0 ? 0 : n < NT ? n : NT;
        return g;
    }
    const int nsb = (p.S + NT - 1) / NT;
    g.w = rg / nsb;
    const int s0 = (rg - g.w * nsb) * NT;
    g.ntok = p.S - s0 < NT ? p.S - s0 : NT;
    g.lin = g.w * p.S + s0;
    return g;
}

// Keys of view f that some token of the group sees, and of the whole group (summed over the
// views, as the pieces walk them).
template <int RM, int NT>
__device__ inline int group_view_vis(const DecodeParams& p, int f, const Group& g) {
    int best = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int v = view_vis<kKvPaged>(p, f, row_loc<RM>(p, g.lin + (t < g.ntok ? t : 0), f));
        best = v > best ? v : best;
    }
    return best;
}
template <int RM, int NT>
__device__ inline long long group_visible(const DecodeParams& p, int rg) {
    if constexpr (NT == 1) {
        return row_visible<kKvPaged, RM>(p, rg);
    } else {
        const Group g = group_of<RM, NT>(p, rg);
        long long n = 0;
        if (g.ntok == 0) return 0;
        for (int f = 0; f < p.F; ++f) n += group_view_vis<RM, NT>(p, f, g);
        return n;
    }
}

// One wave: KV head hkv over visible keys [v0, v1) of one row group.
// NT tiles, of a launch whose groups hold up to GT tokens.
template <int DT, int QM, int RM, int NT, int GT, bool MV, bool P2>
__device__ __forceinline__ void piece(const DecodeParams& p, unsigned char* wlds, int rg, int hkv, long long v0,
                                      long long v1, bool final_out, int slot, int wv, long long row_keys) {
    constexpr int R = kRing;
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, n = lane & 15;
    const uint32_t ring = __builtin_amdgcn_readfirstlane(lds_addr(wlds));
    int* pc = reinterpret_cast<int*>(wlds + R * kStage);
    Group gr;
    if constexpr (GT == 1) {
        gr.w = RM == kRowVarlen ? varlen_seq(p, rg) : rg / p.S;
        gr.lin = rg;
        gr.ntok = 1;
    } else {
        gr = group_of<RM, GT>(p, rg);
        gr.w = uniform(gr.w);
        gr.lin = uniform(gr.lin);
        gr.ntok = uniform(gr.ntok);
    }
    const int w = gr.w;
    const uint32_t lo = lane_offset(p);
    const ReadOff ro = read_offsets();

    State st[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int c = 0; c < 8; ++c) st[t].o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        st[t].m = -DV_INF;
        st[t].l = 0.0f;
    }

    auto one_view = [&](int f, int vis, long long P, long long off) {
        const long long a = v0 > P ? v0 : P;
        const long long bnd = v1 < P + vis ? v1 : P + vis;
        const int l0 = (int)(a - P), l1 = (int)(bnd - P);
        stream::View v;
        v.hkv = hkv;
        v.k = reinterpret_cast<const unsigned char*>(p.kc);
        v.v = reinterpret_cast<const unsigned char*>(p.vc);
        // (past 31 bits on either side: all positions below 0, absent)
        v.off = (int)(off < 0x80000000ll && off >= -0x80000000ll ? off : -0x80000000ll);
        int vis_t[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            vis_t[t] = vis;
            if constexpr (NT > 1)
                vis_t[t] = t < gr.ntok ? uniform(view_vis<kKvPaged>(p, f, row_loc<RM>(p, gr.lin + t, f))) : 0;
        }
        QOp<DT> q[NT];
        // sub-ranges whose pages fit the page cache, whole stages
        long long span = ((long long)(stream::kPc - 2) * p.bs) & ~(long long)(kStep - 1);
        span = span < (1ll << 30) ? (span < kStep ? kStep : span) : 1ll << 30;
        for (int sa = l0; sa < l1;) {
            const int sb = (long long)l1 - sa > span ? (int)(sa + span) : l1;
            v.b = sb;
            uint32_t lpa, lpz, r;
            auto at = [&](long long l) {
                const long long pos = v.off + l;
                return pos < 0 ? 0u : pos < 0x7fffffffll ? (uint32_t)pos : 0x7fffffffu;
            };
            page_split(p, at(sa), lpa, r);
            page_split(p, at(sb - 1ll), lpz, r);
            v.lp0 = (int)lpa;
            stream::fill_pages(p, p.bt + (long long)w * p.maxB, pc, (int)(lpz - lpa) + 1,
                               [&](int i) { return lpa + (uint32_t)i; });
            const int ns = (sb - sa + kStep - 1) / kStep;
            auto load_stage = [&](int at, int l) {
                return issue<P2, (GT > 1), (MV || !P2)>(p, v, lo, pc, ring + (uint32_t)(at * kStage), l);
            };
            uint32_t m[R];  // masks of the stages in flight, the one computed next first
#pragma unroll
            for (int k = 0; k < R; ++k) m[k] = 0;
#pragma unroll 1
            for (int k = 0; k < R && k < ns; ++k) {
                const uint32_t x = load_stage(k, sa + k * kStep);
#pragma unroll
                for (int j = 0; j < R; ++j) m[j] = j == k ? x : m[j];
            }
            if (sa == l0) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    compiler_fence();
                    load_q<DT, QM, RM, (GT > 1)>(p, gr.lin + (t < gr.ntok ? t : 0), f, hkv, q[t]);
                    // settled here: a load still pending at the loop would make the compiler
                    // wait for all vector memory in every step
#pragma unroll
                    for (int k = 0; k < kQParts<DT>; ++k)
#pragma unroll
                        for (int cc = 0; cc < 4; ++cc) asm volatile("" : "+v"(q[t].q[k][cc]));
                }
            }
            int cur = 0;  // ring slot of stage s
            for (int s = 0; s < ns; ++s) {
                // stage s landed: at most the R - 1 after it may be in flight
                if (s + R <= ns) wait_vmcnt<(R - 1) * kLoads>();
                else wait_vmcnt<0>();
                uint32_t mask[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    mask[t] = m[0];
                    if constexpr (NT > 1) {
                        const int lim = vis_t[t] - (sa + s * kStep);
                        mask[t] &= lim >= kStep ? 0xffffffffu : lim <= 0 ? 0u : (1u << lim) - 1u;
                    }
                }
                compute<DT, NT>(st, ring + (uint32_t)(cur * kStage), ro, m[0], mask, q, p.l2scale);
#pragma unroll
                for (int k = 0; k + 1 < R; ++k) m[k] = m[k + 1];
                lds_wait();  // the slot's reads are complete before it is refilled
                if (s + R < ns)
                    m[R - 1] = load_stage(cur, sa + (s + R) * kStep);
                cur = cur + 1 == R ? 0 : cur + 1;
            }
            sa = sb;
        }
    };
    if constexpr (!MV) {
        if (v0 < v1) one_view(0, (int)row_keys, 0ll, 0ll);
    } else if constexpr (GT == 1) {
        if (v0 < v1)
            for_views_blocks<kKvPaged, RM>(p, rg, v0, v1, [&](int f, int vis, long long P, long long off) {
                one_view(f, uniform(vis), uniform(P), uniform(off));
            });
    } else {
        long long P = 0, off = 0;
        for (int f = 0; f < p.F && P < v1; ++f) {
            const int vis = uniform(group_view_vis<RM, GT>(p, f, gr));
            if (vis > 0 && P + vis > v0) one_view(f, vis, P, off);
            P += vis;
            off += p.fl[f];
        }
    }

    // epilogue: total over the four lane groups, normalise, base-2 log-sum-exp
    const int h = hkv * kGqa + n;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (t >= gr.ntok) continue;
        const float lt = rows4_sum(st[t].l);
        const float inv = lt > 0.0f ? 1.0f / lt : 0.0f;
        if (final_out) {
            using raw = typename Tr<DT>::raw;
            raw* o;
            if (RM == kRowVarlen) {
                o = reinterpret_cast<raw*>(p.out) + ((long long)(gr.lin + t) * p.Hq + h) * kHeadDim;
            } else {
                const int s = gr.lin + t - w * p.S;
                o = reinterpret_cast<raw*>(p.out) + (((long long)w * p.Hq + h) * p.S + s) * kHeadDim;
            }
            // a NaN score: the row is NaN, not the zeros of a row without keys
            const float scale = lt != lt ? lt : inv;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const int d = c * 16 + g * 4;
                if constexpr (DT == kF32)
                    *reinterpret_cast<f32x4*>(o + d) = st[t].o[c] * scale;
                else
                    *reinterpret_cast<u32x2*>(o + d) = u32x2{pack2<DT>(st[t].o[c][0] * scale, st[t].o[c][1] * scale),
                                                             pack2<DT>(st[t].o[c][2] * scale, st[t].o[c][3] * scale)};
            }
        } else {
            store_partial<DT>(p.part + (long long)slot * p.slot_floats, p.hpw * GT * kGqa, (wv * GT + t) * kGqa + n, g,
                              st[t].o, inv, row_lse(st[t].m, lt));
        }
    }
}

}  // namespace q8

// MV: calls of several views (or none), whose pieces may start anywhere.  P2: pages of a
// power of two of at least 16 rows (NT > 1: looked up, one kernel for all calls).
template <int DT, int QM, int RM, int NT, bool MV, bool P2>
__global__ __launch_bounds__(q8::kWaves * kWave) void dv_decode8(const DecodeParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((128u - (lds_addr(smem_raw) & 127u)) & 127u);  // (ReadOff)
    __shared__ long long s_scan[q8::kWaves];
    const int wv = uniform((int)(threadIdx.x >> 6));
    const int HPW = p.hpw;
    long long* s_pref = reinterpret_cast<long long*>(smem + HPW * q8::kWaveLds);
    unsigned char* wlds = smem + wv * q8::kWaveLds;
    run_schedule<true, MV ? 1 : kStep, 1, NT == 1>(
        p, p.Hkv / HPW, s_pref, s_scan, [&](int row) { return q8::group_visible<RM, NT>(p, row); },
        [&](int row, int hg, long long v0, long long v1, bool fin, int slot, long long rk) {
            if (wv >= HPW) return;
            const int h = uniform(hg) * HPW + wv;
            // packed calls mix groups of one token with others
            if (RM == kRowVarlen && NT == 2 && uniform(q8::group_of<RM, NT>(p, row).ntok) == 1)
                q8::piece<DT, QM, RM, 1, NT, MV, P2>(p, wlds, uniform(row), h, uniform(v0), uniform(v1),
                                                     uniform((int)fin) != 0, uniform(slot), wv, uniform(rk));
            else
                q8::piece<DT, QM, RM, NT, NT, MV, P2>(p, wlds, uniform(row), h, uniform(v0), uniform(v1),
                                                      uniform((int)fin) != 0, uniform(slot), wv, uniform(rk));
        });
}

// Merge of the pieces of row groups of several tokens (NT = 1: dv_merge).  Block (segment,
// KV head, token): thread t -> head t / 16, dims [(t % 16) * 8, + 8).
template <int DT, int RM, int NT>
__global__ __launch_bounds__(256) void dv_merge8(const DecodeParams p) {
    using raw = typename Tr<DT>::raw;
    const int t = blockIdx.x % NT;
    const int sw = blockIdx.x / NT;
    const int sg = sw / p.hpw, wi = sw - sg * p.hpw;
    const int base = p.dir[2 * sg], cnt = p.dir[2 * sg + 1];
    if (cnt == 1) return;
    const int NHG = p.Hkv / p.hpw;
    const int r = sg / NHG, hkv = (sg - r * NHG) * p.hpw + wi;
    const q8::Group gr = q8::group_of<RM, NT>(p, p.row_begin + r);
    if (t >= gr.ntok) return;
    const int n = threadIdx.x >> 4;
    const int d[1] = {(int)(threadIdx.x & 15) * 8};
    const int h = hkv * kGqa + n;
    raw* o = reinterpret_cast<raw*>(p.out) + d[0];
    if (RM == kRowVarlen) o += ((long long)(gr.lin + t) * p.Hq + h) * kHeadDim;
    else o += (((long long)gr.w * p.Hq + h) * p.S + gr.lin + t - gr.w * p.S) * kHeadDim;
    float v[1][8];
    merge_runs<DT, 1>(p.part, p.slot_floats, p.hpw * NT * kGqa, (wi * NT + t) * kGqa + n, d, base, cnt, v);
    store_run8<DT>(o, v[0]);
}

// The launch of rows [p.row_begin, p.row_begin + p.nrows) and their merge.
template <int DT, int QM, int RM, int NT, bool MV, bool P2>
hipError_t launch8_one(DecodeParams p, int device, long long cap, int cus, hipStream_t stream) {
    const void* kern = reinterpret_cast<const void*>(&dv_decode8<DT, QM, RM, NT, MV, P2>);
    // (up to 64 rows the schedule's sums stay in registers)
    auto lds_of = [](int hpw, int nrows) {
        return 128 + (size_t)hpw * q8::kWaveLds + (nrows > kWave ? (size_t)(nrows + 1) * sizeof(long long) : 0);
    };
    static std::atomic<unsigned long long> attr_done{0};
    hipError_t e = once_per_device(attr_done, device, [&] {
        return hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                                   160 * 1024 - 512);
    });
    if (e != hipSuccess) return e;
    // workgroups that are all resident at once
    const size_t lds = lds_of(p.hpw, p.nrows);
    const int fit = (int)(160 * 1024 / (lds + 512));
    const int most = q8::kWaves / p.hpw;
    const long long nwg = (long long)cus * (fit < most ? fit : most);
    p.nwg = (int)(nwg < cap ? nwg : cap < 1 ? 1 : cap);
    hipLaunchKernelGGL((dv_decode8<DT, QM, RM, NT, MV, P2>), dim3(p.nwg), dim3(p.hpw * kWave), lds, stream, p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    if constexpr (NT == 1) {
        return launch_merge(DT, RM, p, stream);
    } else {
        const int nseg = p.nrows * (p.Hkv / p.hpw);
        hipLaunchKernelGGL((dv_merge8<DT, RM, NT>), dim3(nseg * p.hpw * NT), dim3(256), 0, stream, p);
        return hipGetLastError();
    }
}

}  // namespace dv
