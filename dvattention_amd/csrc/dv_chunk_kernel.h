// gfx950 multi-query ("chunk") attention with fused query RoPE: S >= 2 query
// tokens per sequence that share one K/V stream (chunked prefill, speculative
// verification).  Same operator semantics as the decode kernel
// (src/kernels/paged_kernel_v21.cuh:17-374 and kernel_v21.cuh:17-367 in the
// reference repository, which re-read K/V once per query token: grid.y = W*S,
// paged_kernel_v21.cuh:391); here each K/V row is read once per block of 16
// tokens.
//
//  * Workgroup = eight waves, two per SIMD, on one (sequence, 16-token block,
//    KV head) and a contiguous range of its visible keys.  Wave w owns tokens
//    2w and 2w+1: two 16-row query tiles (16 heads each), so a K/V stage read
//    from LDS feeds 32 query rows per wave and 256 per workgroup.  Groups of at
//    most eight tokens split the keys instead (KS wave sets, stream_range).
//  * K/V pages stream through an 8-stage LDS ring filled by direct-to-LDS loads
//    (global_load_lds_dwordx4, non-temporal): 32 keys x 256 B of K and of V per
//    stage, one eighth issued by each wave, seven stages ahead of the one
//    computed, completion tracked with vmcnt and one workgroup barrier per stage.
//  * Per stage and tile: S^T = K Q^T on 16x16x32 MFMA (8 per tile), online
//    softmax per query row, O^T += V^T P^T (8 MFMA per tile, 16 for fp16: see
//    p_operands); the K and V^T operands of a stage are read from LDS once per
//    wave and kept in registers for both tiles.
//  * MFMA / VALU overlap inside the wave: the two tiles (A = 0, B = 1) run half
//    a stage apart.  Each half-stage issues one tile's MFMAs (S of B and P V of
//    B's previous stage, or P V of A and S of A's next stage) while the other
//    tile's softmax runs on the VALU, so the two use disjoint registers and the
//    matrix core has work during the softmax; the second wave on the SIMD fills
//    what one wave's dependences leave idle.
//  * Rows are causal-masked per token (key l visible iff l <= locations[f,w,s]).
//  * The balanced split / LSE merge is the decode kernel's (equal key chunks per
//    workgroup, fp32 partial slots, dv_merge_chunk).
// The 16-bit multi-query kernel (dv_chunk.hip) and its form for caches held in 8 bits
// (dv_chunk8.hip), as templates.
#pragma once

#include <type_traits>

#include "dv_chunk.h"

namespace dv {
namespace chunk {

// Workgroup barrier that is also a compiler memory and scheduling barrier: no
// LDS access or MFMA moves across it.
__device__ inline void wg_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// swizzled 16-byte piece positions inside a 256-byte key row
__device__ inline int swz_k(int key, int piece) { return piece ^ (key & 15); }
__device__ inline int swz_v(int key, int piece) { return piece ^ ((key & 7) << 1); }

// ---- 8-bit caches (KV8) ---------------------------------------------------------
//
// The stage loop computes on 16-bit tiles, as for a 16-bit cache; they are made from the
// 8-bit rows in LDS, once per workgroup: bytes that every wave widened for itself would
// cost 64 conversions per wave and stage, this takes eight.  Waves 0 .. 3 bring eight rows
// of K each, waves 4 .. 7 of V (16 bytes per lane, and the exponent byte of the lane's
// row), into a raw ring of their own, seven stages ahead; one stage before its turn a
// wave widens its rows -- E4M3 times a power of two, exact in bf16 (in fp16 calls, whose K
// takes fp16, a number beyond that type's range or spacing is rounded to it) -- into one of three
// 16-bit slots.  Three, so that a slot outlives its stage by a barrier and V can be read
// from it again (mask_v).
constexpr int kWideSlots = 3;
constexpr int kRawStages = 8;
constexpr int kRawWave = 64 * 16 + 64 * 4;  // a wave's share of a raw stage: rows, then exponents
constexpr int kRawBytes = kWaves * kRawWave;
template <bool KV8> constexpr int kLdsRing = KV8 ? kWideSlots * kStageBytes + kRawStages * kRawBytes : kRingBytes;

// Per-lane constants of the loop, held in a register each (what derives from them is
// computed where it is used, as is 16 * lane: a register more and fp16 calls read query
// operands back from memory in every stage): the LDS offsets of this lane's K and V^T operands
// in a slot and of its widened piece.
struct Off8 {
    uint32_t k, v, w;
};
__device__ inline uint32_t lane_times_16() { return (uint32_t)(opaque_tid() & 63) * 16; }
__device__ inline Off8 offsets8() {
    const int lane = threadIdx.x & 63, wv = uniform((int)(threadIdx.x >> 6));
    const int g = lane >> 4, n = lane & 15;
    const int k0 = g * 4 + (n >> 2);
    const int kl = (wv & 3) * 8 + (lane >> 3), piece = (lane & 7) * 2;
    Off8 o;
    o.k = (uint32_t)(n * 256 + 16 * (g ^ (n & 3)) + 64 * (n >> 2));
    o.v = (uint32_t)(kKvBytes + k0 * 256 + 16 * ((n & 3) >> 1) + (n & 1) * 8 + 32 * (k0 & 7));
    o.w = (uint32_t)((wv < 4 ? 0 : kKvBytes) + kl * 256 + (wv < 4 ? swz_k(kl, piece) : swz_v(kl, piece)) * 16);
    asm volatile("" : "+v"(o.k), "+v"(o.v), "+v"(o.w));
    return o;
}

// This wave's share of raw stage st (keys kb0 .. kb0 + 31 of the range): lane -> row 8 *
// (wave % 4) + lane / 8, 16-byte piece lane % 8.
template <bool P2>
__device__ inline void issue_raw(const DecodeParams& p, const Range& r, const int* pages, uint32_t raw, int st,
                                 int kb0) {
    const int wv = uniform((int)(threadIdx.x >> 6));
    const uint32_t base = raw + (uint32_t)((st % kRawStages) * kRawBytes + wv * kRawWave);
    const uint32_t lane16 = lane_times_16();
    const int lrow = (int)(lane16 >> 7);
    const int l = kb0 + (wv & 3) * 8 + lrow;
    const uint32_t pos = (uint32_t)(r.off + kb0 + (wv & 3) * 8) + (uint32_t)lrow;
    uint32_t lp, rr;
    if (P2) {
        lp = pos >> p.bs_shift;
        rr = pos & ((1u << p.bs_shift) - 1u);
    } else {
        lp = pos / (uint32_t)p.bs;
        rr = pos - lp * (uint32_t)p.bs;
    }
    const uint32_t idx = lp - r.lp0;
    const unsigned char* c = wv < 4 ? r.k : r.v;
    const unsigned char* e = wv < 4 ? p.ks : p.vs;
    // (one path: a branch here would part the MFMAs that this is computed beside)
    const int pg = pages[idx < (uint32_t)kPageCap ? idx : (uint32_t)(kPageCap - 1)];
    const bool ok = l < r.b && idx < (uint32_t)kPageCap && pg >= 0;
    const uint32_t h = ((uint32_t)pg * (uint32_t)p.bs + rr) * (uint32_t)p.Hkv + (uint32_t)r.hkv;
    const unsigned char* a = (ok ? c + ((unsigned long long)h << 7) : zrow) + (lane16 & 127u);
    const unsigned char* s = ok ? e + ((uint32_t)pg * (uint32_t)p.Hkv + (uint32_t)r.hkv) : zrow;
    dma16(a, __builtin_amdgcn_readfirstlane(base));
    dma1(s, __builtin_amdgcn_readfirstlane(base + 64 * 16));
}

// The wave's share of landed raw stage st, widened into the 16-bit slot at LDS address
// `slot`, at the places where a 16-bit stage has its pieces: K in the queries' type, V in
// bf16.
template <int DT>
__device__ inline void widen(uint32_t slot, uint32_t raw, int st, const Off8& o) {
    const int wv = uniform((int)(threadIdx.x >> 6));
    const uint32_t base = raw + (uint32_t)((st % kRawStages) * kRawBytes + wv * kRawWave);
    typedef __attribute__((address_space(3))) const uint32_t lds_u32;
    const uint32_t lane16 = lane_times_16();
    u32x4 x = lds_read16_at(base + lane16);
    const uint32_t e = *(lds_u32*)(uintptr_t)(base + 64 * 16 + (lane16 >> 2));
    if (ballot(e == 0)) {  // an exponent of 0: a page of zeros (or no page)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = e ? x[i] : 0u;
    }
    const float s = __uint_as_float(e << 23);
    u32x4 w[2];
    if (DT == kF16 && wv < 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i >> 1][(i & 1) * 2] =
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x[i], s, false));
            w[i >> 1][(i & 1) * 2 + 1] =
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x[i], s, true));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i >> 1][(i & 1) * 2] =
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x[i], s, false));
            w[i >> 1][(i & 1) * 2 + 1] =
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x[i], s, true));
        }
    }
    // (both swizzles keep a row's pieces 2i and 2i + 1 side by side, in one order or the other)
    typedef __attribute__((address_space(3))) u32x4 lds_w;
    const uint32_t at = slot + o.w;
    *(lds_w*)(uintptr_t)at = w[0];
    *(lds_w*)(uintptr_t)(at ^ 16u) = w[1];
}

// fp16 calls over 8-bit caches: the weights as two bf16 numbers, 16 bits of each whatever
// its size (an fp16 pair ends at 2^-25 of the row's largest).
__device__ inline POperand p_operands_pair(const float (&pr)[8], float& l) {
    POperand o;
    float ps = pr[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) ps += pr[i];
    l += ps;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = pack2<kBF16>(pr[2 * i], pr[2 * i + 1]);
        o.hi[i] = w;
        o.lo[i] = pack2<kBF16>(pr[2 * i] - __uint_as_float(w << 16), pr[2 * i + 1] - __uint_as_float(w & 0xffff0000u));
    }
    return o;
}

// Issue this wave's eighth of stage `st` (keys [kb0, kb0+32) of the range): key
// rows 4*wave .. 4*wave+3 of K and of V, lane -> (row lane/16, 16-byte piece).
template <int KVM, bool P2>
__device__ inline void issue_stage(const DecodeParams& p, const Range& r, const int* pages, uint32_t ring,
                                   int st, int kb0) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int pos = lane & 15;
    const uint32_t sbase = ring + (uint32_t)(st % kStages) * kStageBytes;
    const int kl = wv * 4 + (lane >> 4);
    const int gk = swz_k(kl, pos), gv = swz_v(kl, pos);
    const uint32_t koff = (uint32_t)(wv * 4) * 256;
    const unsigned char* ka;
    const unsigned char* va;
    if (KVM == kKvPaged && P2 && r.pages_ok && kb0 + kStep <= r.b) {
        // interior stage of a range whose pages are all valid: no visibility
        // test and no zero rows
        const uint32_t pos_l = (uint32_t)(r.off + kb0 + kl);
        const int pg = pages[(pos_l >> p.bs_shift) - r.lp0];
        const uint32_t rowidx = (((uint32_t)pg << p.bs_shift) + (pos_l & ((1u << p.bs_shift) - 1u))) *
                                    (uint32_t)p.Hkv + (uint32_t)r.hkv;
        const unsigned long long boff = (unsigned long long)rowidx << 8;
        ka = r.k + boff + gk * 16;
        va = r.v + boff + gv * 16;
    } else {
        const long long row = row_of<KVM, P2>(p, r, pages, kb0 + kl);
        ka = row >= 0 ? r.k + row + gk * 16 : zrow + gk * 16;
        va = row >= 0 ? r.v + row + gv * 16 : zrow + gv * 16;
    }
    dma16(ka, __builtin_amdgcn_readfirstlane(sbase + koff));
    dma16(va, __builtin_amdgcn_readfirstlane(sbase + kKvBytes + koff));
}

struct Tile {
    f32x4 o[8];
    float m, l;
    // -max(m, -FLT_MAX), the exponent offset of every stage: kept beside m and
    // updated only where m changes (sm_raise), not recomputed per stage
    float nm;
};

// Query tiles of this wave's tokens tok0 .. tok0 + ntile - 1 of group gr for
// view f, staged through LDS (the K/V ring is idle between view ranges): raw
// q rows arrive by direct-to-LDS loads, each lane rotates whole (d, d + R/2)
// pairs in place (src/rope.cuh:18-51 and :67-114: first R/2 cos/sin entries of
// the token's full-width row, or its half-width varlen row; separately rounded
// fp32 products and sum, rounded to the storage type; dims >= R untouched),
// then lane (g, n) reads Q[n][c*32 + g*8 + 0..7] of every tile.  Wave-private
// LDS region: 8 KiB.  A row's 16-byte pieces are XOR-swizzled by the head, like
// the K rows: the rotation and the operand reads touch the same piece of 16 rows
// at once, which unswizzled rows (256 B apart) serialised 16-fold on one group of
// banks -- 4.5-6 us of every piece for the eight waves together, 1.6-2.5 with the swizzle.
// Key split: the KS waves of the same tokens share one region, each staging and
// rotating the heads [kg * 16 / KS, + 16 / KS); read_q_tiles follows a barrier.
template <int DT, int QM, int RM, int KS>
__device__ inline void stage_q_tiles(const DecodeParams& p, unsigned char* qreg, float* csreg, const Grp& gr,
                                     int tok0, int ntile, int kg, int f, int hkv) {
#pragma clang fp contract(off)
    using raw = typename Tr<DT>::raw;
    const int lane = opaque_tid() & 63;
    const uint32_t qbase = lds_addr(qreg);
    const int half = p.R >> 1;
    // every load is issued before the first is waited for: cos/sin of both tiles
    // on clamped, in-bounds indices (a branch around a load waits for it at once)
    float cv[kTiles], sv[kTiles];
    const bool rot = QM != kQPre && half > 0;
    if (rot && ntile > 0) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const long long row = (long long)f * tok_axis<RM>(p) + gr.lin + tok0 + (t < ntile ? t : 0);
            const long long co = (QM == kQRotHalf ? row * half : row * p.R) + (lane < half ? lane : 0);
            cv[t] = p.cosv[co];
            sv[t] = p.sinv[co];
        }
    }
    for (int t = 0; t < ntile; ++t) {
#pragma unroll
        for (int i4 = 0; i4 < 4 / KS; ++i4) {
            const int i = kg * (4 / KS) + i4;
            const int hn = i * 4 + (lane >> 4);
            const int h = hkv * kGqa + hn;
            const raw* q = reinterpret_cast<const raw*>(p.q) + q_row<QM, RM>(p, gr, tok0 + t, h, f);
            dma16(q + ((lane & 15) ^ hn) * 8, __builtin_amdgcn_readfirstlane(qbase + (uint32_t)(t * 4096 + i * 1024)));
        }
    }
    if (rot && ntile > 0) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            csreg[t * 128 + lane] = cv[t];
            csreg[t * 128 + 64 + lane] = sv[t];
        }
    }
    wait_vmcnt<0>();
    compiler_fence();
    if (p.qsign) {  // a negative scale (fold_scale); the rotation keeps the sign
        for (int t = 0; t < ntile; ++t)
            for (int i = kg * (4 / KS); i < (kg + 1) * (4 / KS); ++i)
                *reinterpret_cast<u32x4*>(qreg + t * 4096 + i * 1024 + lane * 16) ^= p.qsign;
        compiler_fence();
    }
    if (rot) {
        constexpr int kLanes = 4 * KS;  // lanes per head
        const int hn = kg * (kGqa / KS) + lane / kLanes, q = lane % kLanes;
        for (int t = 0; t < ntile; ++t) {
            raw* x = reinterpret_cast<raw*>(qreg + t * 4096 + hn * 256);
            auto at = [&](int e) { return x + ((e ^ (hn << 3)) & 127); };  // element e of the row
            const float* cs = csreg + t * 128;
            const float* sn = cs + 64;
            if ((half & 7) == 0) {
                for (int j0 = q * 8; j0 < half; j0 += 8 * kLanes) {
                    u32x4* pa4 = reinterpret_cast<u32x4*>(at(j0));
                    u32x4* pb4 = reinterpret_cast<u32x4*>(at(j0 + half));
                    const u32x4 a = *pa4, b = *pb4;
                    u32x4 ya, yb;
#pragma unroll
                    for (int e2 = 0; e2 < 4; ++e2) {
                        uint32_t wa = 0, wb = 0;
#pragma unroll
                        for (int hl = 0; hl < 2; ++hl) {
                            const int e = e2 * 2 + hl;
                            const float x1 = Tr<DT>::tof((raw)((a[e2] >> (16 * hl)) & 0xffffu));
                            const float x2 = Tr<DT>::tof((raw)((b[e2] >> (16 * hl)) & 0xffffu));
                            const float c = cs[j0 + e], s = sn[j0 + e];
                            const float a1 = x1 * c, b1 = x2 * s;
                            const float a2 = x2 * c, b2 = x1 * s;
                            wa |= (uint32_t)Tr<DT>::fromf(a1 - b1) << (16 * hl);
                            wb |= (uint32_t)Tr<DT>::fromf(a2 + b2) << (16 * hl);
                        }
                        ya[e2] = wa;
                        yb[e2] = wb;
                    }
                    *pa4 = ya;
                    *pb4 = yb;
                }
            } else {
                for (int j = q; j < half; j += kLanes) {
                    raw *xa = at(j), *xb = at(j + half);
                    const float x1 = Tr<DT>::tof(*xa), x2 = Tr<DT>::tof(*xb);
                    const float c = cs[j], s = sn[j];
                    const float a1 = x1 * c, b1 = x2 * s;
                    const float a2 = x2 * c, b2 = x1 * s;
                    *xa = Tr<DT>::fromf(a1 - b1);
                    *xb = Tr<DT>::fromf(a2 + b2);
                }
            }
        }
        compiler_fence();
    }
}

__device__ inline void read_q_tiles(const unsigned char* qreg, int ntile, u32x4 (&qB)[kTiles][4]) {
    const int lane = opaque_tid() & 63;
    const int g = lane >> 4, n = lane & 15;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
        if (t < ntile)
#pragma unroll
            for (int cc = 0; cc < 4; ++cc)
                qB[t][cc] = *reinterpret_cast<const u32x4*>(qreg + t * 4096 + n * 256 + (((cc * 4 + g) ^ n) << 4));
    compiler_fence();
}

// frag / view_vis: the views' tensors and visible key counts (dv_stream.h)

// K operand of one stage (A of S^T = K Q^T): lo[cc] holds key n, hi[cc] key
// 16 + n, dims cc*32 + g*8 .. +8 (lane (g, n)).  The K swizzle only flips
// address bits 6-7 of the row base, so slice cc is at kbase ^ (64 cc).
struct KOp {
    u32x4 lo[4], hi[4];
};

// V^T operand of one stage (A of O^T += V^T P^T), 16-dim slice cc: block lane
// sl -> key g*4 + sl/4 (and + 16), dims cc*16 + (sl%4)*4 (transposing reads);
// the V swizzle only flips address bits 5-7, so slice cc is at vbase ^ (32 cc).
struct VOp {
    u32x4 v[8];
};

__device__ inline void read_k_at(uint32_t kbase, KOp& k) {
#pragma unroll
    for (int cc = 0; cc < 4; ++cc) {
        k.lo[cc] = lds_read16_at(kbase ^ (uint32_t)(64 * cc));
        k.hi[cc] = lds_read16_at((kbase ^ (uint32_t)(64 * cc)) + 16 * 256);
    }
}

__device__ inline void read_k(const unsigned char* kt, KOp& k) {
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, n = lane & 15;
    read_k_at(lds_addr(kt) + (uint32_t)(n * 256 + 16 * (g ^ (n & 3)) + 64 * (n >> 2)), k);
}

__device__ inline void read_v_at(uint32_t vbase, VOp& v) {
#pragma unroll
    for (int cc = 0; cc < 8; ++cc) {
        const u32x2 a0 = lds_read_tr16_at(vbase ^ (uint32_t)(32 * cc));
        const u32x2 a1 = lds_read_tr16_at((vbase ^ (uint32_t)(32 * cc)) + 16 * 256);
        v.v[cc] = u32x4{a0[0], a0[1], a1[0], a1[1]};
    }
}

// Scores of one tile: s0 keys 0-15, s1 keys 16-31 (S^T, lane (g, n): keys
// g*4 + i of head n).
template <int DT>
__device__ inline void qk_tile(const KOp& k, const u32x4 (&q)[4], f32x4& s0, f32x4& s1) {
    s0 = f32x4{0.f, 0.f, 0.f, 0.f};
    s1 = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int cc = 0; cc < 4; ++cc) {
        s0 = Tr<DT>::mma(k.lo[cc], q[cc], s0);
        s1 = Tr<DT>::mma(k.hi[cc], q[cc], s1);
    }
}

// O^T += V^T P^T for one tile.
template <int DT, bool KV8 = false>
__device__ inline void pv_tile(const VOp& v, const POperand& pB, Tile& t) {
    constexpr int VT = KV8 ? kBF16 : DT;
#pragma unroll
    for (int cc = 0; cc < 8; ++cc) t.o[cc] = Tr<VT>::mma(v.v[cc], pB.hi, t.o[cc]);
    if constexpr (DT == kF16) {
#pragma unroll
        for (int cc = 0; cc < 8; ++cc) t.o[cc] = Tr<VT>::mma(v.v[cc], pB.lo, t.o[cc]);
    }
}

// Visibility of the 32 keys of the stage starting at kb0: the range end, and,
// when some page of the sub-range is missing, page validity (a scalar branch
// around a few instructions; the loop itself is not duplicated).
template <int KVM, bool P2, int KS>
__device__ inline uint32_t stage_mask(const DecodeParams& p, const Range& r, const int* pages, int sbnd, int kb0) {
    const int nin = sbnd - kb0;
    uint32_t m = nin >= 32 ? 0xffffffffu : ((1u << (KS > 1 && nin < 0 ? 0 : nin)) - 1u);  // KS > 1: stages past the end
    if (!r.pages_ok) {
        const int lane = threadIdx.x & 63;
        const bool kv_ok = row_of<KVM, P2>(p, r, pages, kb0 + (lane & 31)) >= 0;
        m &= (uint32_t)ballot(kv_ok && lane < 32);
    }
    return m;
}

__device__ inline void read_v(const unsigned char* vt, VOp& v) {
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, sl = lane & 15;
    const int k0 = g * 4 + (sl >> 2);
    read_v_at(lds_addr(vt) + (uint32_t)(k0 * 256 + 16 * ((sl & 3) >> 1) + (sl & 1) * 8 + 32 * (k0 & 7)), v);
}

// V^T operand with the keys cleared that a tile does not see (bit k of mask: key k): their
// weight is 0, which a NaN of another token's row would survive.  A lane holds keys
// g*4 + i and 16 + g*4 + i, 16 bits each.
__device__ inline void mask_v(VOp& v, uint32_t mask) {
    const int lane = opaque_tid() & 63;
    const uint32_t mg = mask >> ((lane >> 4) * 4);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t b = mg >> ((i >> 1) * 16 + (i & 1) * 2);
        w[i] = ((b & 1u) ? 0xffffu : 0u) | ((b & 2u) ? 0xffff0000u : 0u);
        asm volatile("" : "+v"(w[i]));  // (a branch around it stays one)
    }
#pragma unroll
    for (int cc = 0; cc < 8; ++cc)
#pragma unroll
        for (int i = 0; i < 4; ++i) v.v[cc][i] &= w[i];
}

// Scores of invisible keys set to -inf (mask bit k = key k; lane (g, n) holds
// keys g*4 + i and 16 + g*4 + i): a partially visible stage only, so full
// stages spend nothing on masks.  They are scaled later, by a positive number (fold_scale).
__device__ inline void mask_scores(f32x4& s0, f32x4& s1, uint32_t mask) {
    const int lane = threadIdx.x & 63;
    const uint32_t mg = mask >> ((lane >> 4) * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        s0[i] = ((mg >> i) & 1u) ? s0[i] : -DV_INF;
        s1[i] = ((mg >> (16 + i)) & 1u) ? s1[i] : -DV_INF;
    }
}

// Online softmax of two tiles over one 32-key stage, in two straight-line
// parts so that the MFMAs of the other tile group can be interleaved with it
// (a branch ends the scheduling region).  Scores of invisible keys are -inf
// already (mask_scores).  Part 1: base-2 exponents against the running max
// (lane (g, n) holds keys g*4 + i and 16 + g*4 + i of head n); returns the
// lane's largest, so the caller can ask whether some row exceeds its max by
// more than kMaxSlack or has no max yet -- then sm_raise (rare) raises the max
// to the rows' maximum, rescales the accumulators and recomputes the
// exponents.  Part 2 (sm_finish): the probabilities, the row sums and the P^T
// operands.  Same arithmetic as softmax32 + p_operands.
__device__ inline float sm_exponents(const Tile& t, const f32x4& s0, const f32x4& s1, float l2, float (&pr)[8]) {
    // a row with no max yet (m = -inf) subtracts -FLT_MAX instead (t.nm): a
    // visible key's exponent is then huge (the row takes sm_raise) and an
    // invisible key's stays -inf, where -inf - (-inf) would be NaN
    const float nm = t.nm;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        pr[i] = __builtin_fmaf(s0[i], l2, nm);
        pr[4 + i] = __builtin_fmaf(s1[i], l2, nm);
    }
    // shaped for three-operand maxima: max3(max3(0,1,2), max3(3,4,5), max(6,7)),
    // four instructions where a balanced pairwise tree compiled to five
    const float a = fmaxf(fmaxf(pr[0], pr[1]), pr[2]), b = fmaxf(fmaxf(pr[3], pr[4]), pr[5]);
    return fmaxf(fmaxf(a, b), fmaxf(pr[6], pr[7]));
}

__device__ inline void sm_raise(Tile& t, const f32x4& s0, const f32x4& s1, float l2, float (&pr)[8]) {
    float sc[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sc[i] = s0[i] * l2;
        sc[4 + i] = s1[i] * l2;
    }
    const float mx = rows4_max(
        fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7]))));
    if (ballot(mx > t.m + kMaxSlack)) {
        const float mnew = fmaxf(t.m, mx);
        const float alpha = mnew == -DV_INF ? 1.0f : __builtin_amdgcn_exp2f(t.m - mnew);
        t.l *= alpha;
#pragma unroll
        for (int c = 0; c < 8; ++c) t.o[c] *= alpha;
        t.m = mnew;
        t.nm = -fmaxf(mnew, -3.402823466e38f);
    }
    const float mm = t.m == -DV_INF ? 0.0f : t.m;  // p = 0 while the row has no visible key
#pragma unroll
    for (int i = 0; i < 8; ++i) pr[i] = sc[i] - mm;
}

template <int DT, bool KV8 = false>
__device__ inline POperand sm_finish(Tile& t, float (&pr)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) pr[i] = __builtin_amdgcn_exp2f(pr[i]);
    if constexpr (KV8 && DT == kF16) return p_operands_pair(pr, t.l);
    else return p_operands<DT>(pr, t.l);
}

// Register tie: the values are complete at this point in program order (the
// compiler may not move their computation past it, e.g. across a workgroup
// barrier into the next half-stage).  Only the words the P V MFMAs read are
// tied: bf16 has no residual operand, and tying its (zero) lo made the
// compiler rebuild and copy four zero registers every half-stage.
template <int DT>
__device__ inline void settle(POperand& a) {
    asm volatile("" : "+v"(a.hi));
    if constexpr (DT == kF16) asm volatile("" : "+v"(a.lo));
}

// Key split KS (1, 2 or 4): a row group of few tokens leaves waves without
// tokens, and the arithmetic of 16 tokens per stage, not the loads, bound calls
// of 2 .. 8 tokens.  So KS sets of kWaves / KS waves hold the same tokens and
// take every KS-th stage: wave set kg computes stages kg, kg + KS, ... and one
// step of the loop covers KS stages of the ring; the sets' tiles are combined
// at the end of a piece (combine_split).  Steps in flight: the ring's steps
// less one for KS = 1, every step of the ring for KS > 1.  32 sequences of
// 4608 keys, 8 KV heads, bf16, same call without the split -> with it: 4 tokens
// 194 -> 117 us (5.2 TB/s), 8 tokens 194 -> 131 us.
template <int KS> constexpr int lead() { return KS == 1 ? kAhead : kStages / KS; }

// Keys [sa, sbnd) of the current view for this wave's two tiles (A = tile 0,
// B = tile 1): the stage loop.  Ring slot i % kStages holds stage i.  Per
// stage i, in every wave:
//   H1(i): MFMA O_B += V(i-1) P_B(i-1) beside A's exponents; MFMA S_B(i) =
//          K(i) Q_B^T and read V(i) beside A's probabilities
//   own loads of stage i+1 landed; workgroup barrier
//   H2(i): read K(i+1); MFMA O_A += V(i) P_A(i) beside B's exponents; MFMA
//          S_A(i+1) = K(i+1) Q_A^T and the loads of stage i+kAhead beside B's
//          probabilities
// so each wave's instruction stream alternates MFMAs of one tile with the
// softmax of the other, and the two waves of a SIMD issue both at once.  The
// loads of H2(i) refill slots of step i (KS > 1) or i-1 only: the barrier of
// step i is reached by every wave with its reads of every stage <= i complete
// (K(i) is read in H2(i-1), the V reads of H1 are waited for before the barrier).  One
// K and one V^T operand set live in registers: K(i+1) is read after the MFMAs
// of K(i) are issued, V(i) after those of V(i-1).  A's accumulators are
// rescaled in H1 and written by MFMAs issued in H2 (and B's the other way
// round), so a softmax never touches registers an MFMA of the same half-stage
// writes; mfma_settle before each softmax covers the MFMA -> VALU dependence
// across the half-stage boundary.  Invisible keys get -inf scores only on a
// partially visible stage (a uniform branch between the interleaved regions).
template <int DT, int KVM, bool P2, int KS>
__device__ inline void stream_range(const DecodeParams& p, const Range& r, const int* pages, unsigned char* smem,
                                    int sa, int sbnd, int kg, const int (&vis_t)[kTiles],
                                    const u32x4 (&qB)[kTiles][4], Tile (&tl)[kTiles]) {
    constexpr int kLead = lead<KS>();
    constexpr int kDma = kDmaPerStage * KS;  // loads per wave and step
    const uint32_t ring = lds_addr(smem);
    const int nsteps = (sbnd - sa + KS * kStep - 1) / (KS * kStep);
    const float l2 = p.loop_scale;
    // prologue: steps 0 .. kLead-1.  Past the end, KS = 1 issues rows of zeros; with a
    // key split such steps issue nothing (a view of 30 keys would pay for the
    // addresses of 12 stages and not 4: 2 tokens, 4 sequences, six such views, 8 KV
    // heads 112.5 -> 99.6 us; six of 150 keys 55 -> 50.5).
#pragma unroll
    for (int s = 0; s < kLead; ++s) {
        if (KS > 1 && s >= nsteps) break;
#pragma unroll
        for (int st = s * KS; st < (s + 1) * KS; ++st) issue_stage<KVM, P2>(p, r, pages, ring, st, sa + st * kStep);
    }
    if (KS == 1 || nsteps >= kLead) wait_vmcnt<kDma * (kLead - 1)>();  // own share of step 0 landed
    else wait_vmcnt<0>();
    wg_barrier();

    KOp kop;
    VOp vop;
#pragma unroll
    for (int cc = 0; cc < 8; ++cc) vop.v[cc] = u32x4{0u, 0u, 0u, 0u};  // the first P V adds 0 * 0
    f32x4 sa0, sa1, sb0, sb1;
    POperand pa = {}, pb = {};
    read_k(smem + kg * kStageBytes, kop);
    qk_tile<DT>(kop, qB[0], sa0, sa1);

    for (int i = 0; i < nsteps; ++i) {
        const int st = i * KS + kg;  // this wave's stage of the step
        const int kb0 = sa + st * kStep;
        const unsigned char* slot = smem + (st % kStages) * kStageBytes;
        const uint32_t okm = stage_mask<KVM, P2, KS>(p, r, pages, sbnd, kb0);
        const uint32_t mka = okm & token_mask(vis_t[0], kb0), mkb = okm & token_mask(vis_t[1], kb0);
        float pr[8];
        // ---- H1(i)
        if (mka != 0xffffffffu) mask_scores(sa0, sa1, mka);
        mfma_settle(tl[0].o);
        pv_tile<DT>(vop, pb, tl[1]);  // zero at i = 0
        float lmx = sm_exponents(tl[0], sa0, sa1, l2, pr);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);  // VALU
        }
        if (ballot(lmx > kMaxSlack)) sm_raise(tl[0], sa0, sa1, l2, pr);
        qk_tile<DT>(kop, qB[1], sb0, sb1);
        read_v(slot + kKvBytes, vop);
        pa = sm_finish<DT>(tl[0], pr);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS read
            __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);  // VALU
        }
        settle<DT>(pa);
        lds_wait();
        // own share of step i + 1 landed (with a key split, fewer loads follow it near
        // the end)
        if (KS == 1 || i + kLead <= nsteps) wait_vmcnt<kDma * (kLead - 2)>();
        else wait_vmcnt<0>();
        wg_barrier();
        if (KS > 1 && i + kLead < nsteps) {
            // the loads of step i + kLead, into the slots of step i (free since the
            // barrier): at once, as no later step is in flight when KS = 4; one
            // stage at a time, the addresses of all do not fit the registers
#pragma unroll 1
            for (int q = (i + kLead) * KS; q < (i + kLead + 1) * KS; ++q)
                issue_stage<KVM, P2>(p, r, pages, ring, q, sa + q * kStep);
        }
        // ---- H2(i) (past the end, step i + 1 holds rows of zeros or what the slot
        // held before: K and S_A of the next stage need no branch, the last ones go
        // unused)
        read_k(smem + ((st + KS) % kStages) * kStageBytes, kop);
        if (mkb != 0xffffffffu) mask_scores(sb0, sb1, mkb);
        mfma_settle(tl[1].o);
        pv_tile<DT>(vop, pa, tl[0]);
        lmx = sm_exponents(tl[1], sb0, sb1, l2, pr);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
            __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);  // VALU
        }
        if (ballot(lmx > kMaxSlack)) sm_raise(tl[1], sb0, sb1, l2, pr);
        qk_tile<DT>(kop, qB[0], sa0, sa1);
        pb = sm_finish<DT>(tl[1], pr);
        // the loads of stage i + kAhead (into the slot of stage i - 1, free since
        // the barrier), their address arithmetic beside the MFMAs
        if constexpr (KS == 1) issue_stage<KVM, P2>(p, r, pages, ring, i + kLead, sa + (i + kLead) * kStep);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);  // VALU
        }
        settle<DT>(pb);
    }
    // P V of B's last stage
    mfma_settle(tl[1].o);
    pv_tile<DT>(vop, pb, tl[1]);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) mfma_settle(tl[t].o);
    wait_vmcnt<0>();  // the trailing zero-row stages land before the ring is reused
    __syncthreads();
}

// The same loop over an 8-bit cache (KS = 1): stage i + 1 is widened in H1(i), complete
// before the barrier after which K(i + 1) is read.  Two loops, one after the other in the
// same pipeline: stages that both tiles see whole (no masks at all), then those from the
// first that some tile sees in part -- the last ones of a causal chunk -- where scores are
// masked and each tile's V operand too.  In one loop, the masked operand would cost the
// common stages 32 registers, which there are not (two prompt chunks of 2048 tokens over
// 4100 keys, 8 KV heads: 2898 us in one loop, 1240 so, 0.72 PFLOP/s; a 16-bit cache of
// these sizes takes 1090).  Bound by VALU issue, six instructions to an MFMA, and the
// barrier of each stage: of the SIMDs' time MFMAs run for a third.  Widening between the
// first MFMAs of a stage instead of after them made no difference.
template <int DT, bool P2>
__device__ inline void stream_range8(const DecodeParams& p, const Range& r, const int* pages, unsigned char* smem,
                                     int sa, int sbnd, int ntile, const int (&vis_t)[kTiles],
                                     const u32x4 (&qB)[kTiles][4], Tile (&tl)[kTiles]) {
    constexpr int kLead = lead<1>();
    constexpr int kDma = kDmaPerStage;  // of a raw stage: rows and exponents
    const uint32_t ring = lds_addr(smem);
    const uint32_t raw = ring + kWideSlots * kStageBytes;
    const int nsteps = (sbnd - sa + kStep - 1) / kStep;
    const float l2 = p.loop_scale;
    const Off8 o8 = offsets8();
    // stages that every tile of this wave sees whole
    int seen = sbnd;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
        if (t < ntile && vis_t[t] < seen) seen = vis_t[t];
    const int nfull = r.pages_ok && seen > sa ? (seen - sa) / kStep : 0;
#pragma unroll
    for (int s = 0; s < kLead; ++s) issue_raw<P2>(p, r, pages, raw, s, sa + s * kStep);
    wait_vmcnt<kDma * (kLead - 1)>();  // own share of stage 0 landed
    widen<DT>(ring, raw, 0, o8);
    lds_wait();
    wg_barrier();

    KOp kop;
    VOp vop;
#pragma unroll
    for (int cc = 0; cc < 8; ++cc) vop.v[cc] = u32x4{0u, 0u, 0u, 0u};  // the first P V adds 0 * 0
    f32x4 sa0, sa1, sb0, sb1;
    POperand pa = {}, pb = {};
    read_k_at(ring + o8.k, kop);
    qk_tile<DT>(kop, qB[0], sa0, sa1);
    uint32_t mkb_last = 0xffffffffu;  // what B saw of the stage whose P V is still to come
    uint32_t at = 0, next = kStageBytes;  // slots of stages i and i + 1

    auto step = [&](auto masked, int i) {
        constexpr bool kMask = decltype(masked)::value;
        const int kb0 = sa + i * kStep;
        uint32_t mka = 0xffffffffu, mkb = 0xffffffffu;
        float pr[8];
        // ---- H1(i)
        if constexpr (kMask) {
            const uint32_t okm = stage_mask<kKvPaged, P2, 1>(p, r, pages, sbnd, kb0);
            mka = okm & token_mask(vis_t[0], kb0);
            mkb = okm & token_mask(vis_t[1], kb0);
            if (mka != 0xffffffffu) mask_scores(sa0, sa1, mka);
            if (mkb_last != 0xffffffffu) mask_v(vop, mkb_last);
            mkb_last = mkb;
        }
        mfma_settle(tl[0].o);
        pv_tile<DT, true>(vop, pb, tl[1]);  // zero at i = 0
        float lmx = sm_exponents(tl[0], sa0, sa1, l2, pr);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);  // VALU
        }
        if (ballot(lmx > kMaxSlack)) sm_raise(tl[0], sa0, sa1, l2, pr);
        qk_tile<DT>(kop, qB[1], sb0, sb1);
        read_v_at(ring + at + o8.v, vop);
        pa = sm_finish<DT, true>(tl[0], pr);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS read
            __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);  // VALU
        }
        settle<DT>(pa);
        // own share of stage i + 1 landed: widened here, where K(i)'s registers are free
        wait_vmcnt<kDma * (kLead - 2)>();
        __builtin_amdgcn_sched_barrier(0);
        widen<DT>(ring + next, raw, i + 1, o8);
        lds_wait();
        wg_barrier();
        // ---- H2(i)
        read_k_at(ring + next + o8.k, kop);
        if constexpr (kMask) {
            if (mkb != 0xffffffffu) mask_scores(sb0, sb1, mkb);
            if (mka != 0xffffffffu) mask_v(vop, mka);
        }
        mfma_settle(tl[1].o);
        pv_tile<DT, true>(vop, pa, tl[0]);
        lmx = sm_exponents(tl[1], sb0, sb1, l2, pr);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
            __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);  // VALU
        }
        if (ballot(lmx > kMaxSlack)) sm_raise(tl[1], sb0, sb1, l2, pr);
        qk_tile<DT>(kop, qB[0], sa0, sa1);
        pb = sm_finish<DT, true>(tl[1], pr);
        issue_raw<P2>(p, r, pages, raw, i + kLead, sa + (i + kLead) * kStep);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);  // VALU
        }
        settle<DT>(pb);
        if constexpr (kMask) {
            if (mka != 0xffffffffu) read_v_at(ring + at + o8.v, vop);  // whole again, for B
        }
        at = next;
        next = next == (kWideSlots - 1) * kStageBytes ? 0u : next + kStageBytes;
    };
    int i = 0;
#pragma unroll 1
    for (; i < nfull; ++i) step(std::false_type{}, i);
#pragma unroll 1
    for (; i < nsteps; ++i) step(std::true_type{}, i);
    // P V of B's last stage
    if (mkb_last != 0xffffffffu) mask_v(vop, mkb_last);
    mfma_settle(tl[1].o);
    pv_tile<DT, true>(vop, pb, tl[1]);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) mfma_settle(tl[t].o);
    wait_vmcnt<0>();  // the trailing stages land before the ring is reused
    __syncthreads();
}

// Key split: wave kg's tiles of the same tokens (kg = 0 .. KS - 1, waves
// kg * kWaves/KS + tp) combined into those of kg = 0, through the idle ring:
// lane by lane, O and the lane's row sum scaled to the common maximum (fp32).
template <int KS>
__device__ inline void combine_split(unsigned char* smem, int wv, int kg, int ntile, Tile (&tl)[kTiles]) {
    constexpr int kPairs = kWaves / KS;  // waves per key subset
    constexpr int kRec = 10 * 1024;      // per (wave, tile): 8 x 1 KiB of O, then m and l
    static_assert((kWaves - kPairs) * kTiles * kRec <= kRingBytes + kPageCap * 4, "LDS of the combination");
    const int lane = threadIdx.x & 63;
    auto rec = [&](int k, int t) {  // record of tile t of the wave with subset k >= 1 of these tokens
        return smem + (((k - 1) * kPairs + wv % kPairs) * kTiles + t) * kRec;
    };
    if (kg > 0) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            if (t >= ntile) continue;
            unsigned char* b = rec(kg, t);
#pragma unroll
            for (int c = 0; c < 8; ++c) *reinterpret_cast<f32x4*>(b + c * 1024 + lane * 16) = tl[t].o[c];
            float* ml = reinterpret_cast<float*>(b + 8 * 1024);
            ml[lane] = tl[t].m;
            ml[64 + lane] = tl[t].l;
        }
    }
    __syncthreads();
    if (kg == 0) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            if (t >= ntile) continue;
            float mk[KS], M = tl[t].m;
#pragma unroll
            for (int k = 1; k < KS; ++k) {
                mk[k] = reinterpret_cast<const float*>(rec(k, t) + 8 * 1024)[lane];
                M = fmaxf(M, mk[k]);
            }
            // an empty subset (-inf) -> weight 0; with no maximum in any, all have
            // it, and what a NaN left in a subset's sums stays
            const float Mf = M == -DV_INF ? 0.0f : M;
            const float s0 = __builtin_amdgcn_exp2f(tl[t].m - Mf);
            tl[t].l *= s0;
#pragma unroll
            for (int c = 0; c < 8; ++c) tl[t].o[c] *= s0;
#pragma unroll
            for (int k = 1; k < KS; ++k) {
                const float sk = __builtin_amdgcn_exp2f(mk[k] - Mf);
                tl[t].l += sk * reinterpret_cast<const float*>(rec(k, t) + 8 * 1024)[64 + lane];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    tl[t].o[c] += sk * *reinterpret_cast<const f32x4*>(rec(k, t) + c * 1024 + lane * 16);
            }
            tl[t].m = M;
        }
    }
    __syncthreads();  // the records are read before the ring is filled again
}

// One workgroup: keys [v0, v1) of row group rg for KV head hkv.
template <int DT, int QM, int KVM, bool P2, int RM, int KS, bool KV8>
__device__ void chunk_piece(const DecodeParams& p, unsigned char* smem, int* pages, int rg, int hkv, long long v0,
                            long long v1, bool final_out, int slot, long long row_keys) {
    const int wv = uniform((int)(threadIdx.x >> 6));
    Grp gr = group_of<RM>(p, rg);
    gr.w = uniform(gr.w);
    gr.s0 = uniform(gr.s0);
    gr.lin = uniform(gr.lin);
    gr.ntok = uniform(gr.ntok);
    const int w = gr.w;
    const int kg = KS == 1 ? 0 : wv / (kWaves / KS);                // this wave's key subset
    const int tok0 = (KS == 1 ? wv : wv % (kWaves / KS)) * kTiles;  // and first token of the group
    const int ntile = gr.ntok - tok0 < kTiles ? (gr.ntok - tok0 > 0 ? gr.ntok - tok0 : 0) : kTiles;

    Tile tl[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
#pragma unroll
        for (int c = 0; c < 8; ++c) tl[t].o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        tl[t].m = -DV_INF;
        tl[t].l = 0.0f;
        tl[t].nm = 3.402823466e38f;
    }

    long long P = 0, off = 0;
    for (int f = 0; f < p.F && P < v1; ++f) {
        // visible keys per tile (wave-uniform: the stage masks and their branches
        // stay scalar), and of this view for the block: the union over its tokens,
        // for a single view the row's keys, counted by the schedule
        int vis_t[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int last = gr.ntok - 1;  // >= 0: a group without tokens has no piece
            const int v = uniform(view_vis<KVM>(p, f, loc_of<RM>(p, f, gr, tok0 + t < last ? tok0 + t : last)));
            vis_t[t] = t < ntile ? v : 0;
        }
        const int vis_blk = p.F == 1 ? (int)row_keys : uniform(group_view_vis<KVM, RM>(p, f, gr));
        long long a = v0 > P ? v0 : P;
        long long bnd = v1 < P + vis_blk ? v1 : P + vis_blk;
        if constexpr (KV8) {  // rows at positions outside 31 bits are absent (issue_raw counts in 32)
            a = a > P - off ? a : P - off;
            bnd = bnd < P - off + 0x80000000ll ? bnd : P - off + 0x80000000ll;
        }
        if (a < bnd) {
            const int la = (int)(a - P), lb = (int)(bnd - P);
            Range r;
            r.w = w;
            r.hkv = hkv;
            if (KVM == kKvPaged) {
                r.k = reinterpret_cast<const unsigned char*>(p.kc);
                r.v = reinterpret_cast<const unsigned char*>(p.vc);
                r.off = off;
                r.bstride = 0;
                r.L = 0;
            } else {
                const FragDesc& fd = frag<KVM>(p, f);
                r.k = reinterpret_cast<const unsigned char*>(fd.k);
                r.v = reinterpret_cast<const unsigned char*>(fd.v);
                r.off = 0;
                r.bstride = fd.bstride * w;
                r.L = fd.L;
            }
            u32x4 qB[kTiles][4] = {};
            // sub-ranges whose page ids fit the LDS page cache
            const int span = KVM == kKvPaged ? subrange_keys(p.bs) : 1 << 30;
            for (int sa = la, sbnd; sa < lb; sa = sbnd) {
                sbnd = subrange_end(sa, lb, span);
                r.b = sbnd;
                int pg[kPageIt];
                uint32_t lpl = 0;
                r.lp0 = 0;
                if (KVM == kKvPaged) {
                    lpl = logical_page(p, off + sbnd - 1);
                    r.lp0 = logical_page(p, off + sa);
                    fetch_pages(p, p.bt + (long long)w * p.maxB, r.lp0, lpl, pg);
                }
                // the ring is idle here (previous range drained): stage the query tiles
                // in it, their round trip beside the page ids'
                unsigned char* qreg = smem + (KS == 1 ? wv : wv % (kWaves / KS)) * (kTiles * 4096);
                if (sa == la) {
                    stage_q_tiles<DT, QM, RM, KS>(
                        p, qreg, reinterpret_cast<float*>(smem + kWaves * kTiles * 4096 + wv * kTiles * 512), gr, tok0,
                        ntile, kg, f, hkv);
                    if (KS == 1) read_q_tiles(qreg, ntile, qB);
                }
                // every position and page of the sub-range is valid; the page ids are
                // written and the query tiles read (KS > 1: staged)
                bool ok = true;
                if (KVM == kKvPaged)
                    ok = store_pages(p, pages, r.lp0, lpl, pg) && position_in_range(off + sa) &&
                         position_in_range(off + sbnd - 1);
                r.pages_ok = __syncthreads_and(ok) != 0;
                if (KS > 1 && sa == la) {
                    read_q_tiles(qreg, ntile, qB);
                    __syncthreads();
                }
                if constexpr (KV8) stream_range8<DT, P2>(p, r, pages, smem, sa, sbnd, ntile, vis_t, qB, tl);
                else stream_range<DT, KVM, P2, KS>(p, r, pages, smem, sa, sbnd, kg, vis_t, qB, tl);
            }
        }
        P += vis_blk;
        off += p.fl[f];
    }

    if constexpr (KS > 1) combine_split<KS>(smem, wv, kg, ntile, tl);

    // epilogue: per tile, normalise and write the output or a partial slot
    {
    const int lane = opaque_tid() & 63;
    const int g = lane >> 4, n = lane & 15;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        if (t >= ntile || kg > 0) continue;
        const float lt = rows4_sum(tl[t].l);
        const float inv = lt > 0.0f ? 1.0f / lt : 0.0f;
        const int h = hkv * kGqa + n;
        if (final_out) {
            using raw = typename Tr<DT>::raw;
            raw* o = reinterpret_cast<raw*>(p.out) + out_row<RM>(p, gr, tok0 + t, h);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const u32x2 pk = {pack2<DT>(tl[t].o[c][0] * inv, tl[t].o[c][1] * inv),
                                  pack2<DT>(tl[t].o[c][2] * inv, tl[t].o[c][3] * inv)};
                *reinterpret_cast<u32x2*>(o + c * 16 + g * 4) = pk;
            }
        } else {
            const int tb = tok0 + t;  // token within the block
            store_partial<DT>(p.part + (long long)slot * p.slot_floats, kTokBlk * kGqa, tb * kGqa + n, g, tl[t].o,
                              inv, row_lse(tl[t].m, lt));
        }
    }
    }
}

// P2: paged with a power-of-two block_size (shift and mask instead of a
// division in the stage loop's row addressing).  KS = 0 (varlen): the key split of
// each row group follows from its own tokens, four wave sets up to kFewTok tokens
// and none above (decodes beside prompt chunks, and the last tokens of a chunk).
template <int DT, int QM, int KVM, bool P2, int RM, int KS, bool KV8 = false>
__global__ __launch_bounds__(kThreads) void dv_chunk(const DecodeParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    // the ring starts at a 256-byte aligned LDS address (the XOR addressing of
    // the MFMA operands needs address bits 0-7 of every tile base clear)
    unsigned char* smem = smem_raw + ((256u - (lds_addr(smem_raw) & 255u)) & 255u);
    int* pages = reinterpret_cast<int*>(smem + kLdsRing<KV8>);
    long long* s_scan = reinterpret_cast<long long*>(smem + kLdsRing<KV8> + kPageCap * 4);  // kWaves entries
    long long* s_pref = s_scan + kWaves;
    const int NHG = p.Hkv;  // one KV head per workgroup

    if constexpr (KS > 0) {
        run_schedule(p, NHG, s_pref, s_scan,
                     [&](int rg) {
                         // (varlen over an 8-bit cache: groups of few tokens go another way)
                         if (KV8 && RM == kRowVarlen && group_of<RM>(p, rg).ntok <= kFewTok) return 0ll;
                         return group_visible<KVM, RM>(p, rg);
                     },
                     [&](int rg, int hg, long long v0, long long v1, bool fin, int slot, long long rk) {
                         chunk_piece<DT, QM, KVM, P2, RM, KS, KV8>(p, smem, pages, uniform(rg), uniform(hg), uniform(v0),
                                                              uniform(v1), uniform((int)fin) != 0, uniform(slot),
                                                              uniform(rk));
                     });
    } else {
        // the schedule counts units, even for a group without the split, odd with it
        // (one unit more than its keys': both sides of a cut round down alike, so it
        // never makes a key)
        run_schedule<false, 1, kLongKeyCost>(
                     p, NHG, s_pref, s_scan,
                     [&](int rg) {
                         const long long v = group_visible<KVM, RM>(p, rg);
                         const bool split =
                             group_of<RM>(p, rg).ntok <= kFewTok && v >= (long long)kSplitVarlenKeys * p.F;
                         return split ? v * kShortKeyCost + 1 : v * kLongKeyCost;
                     },
                     [&](int rg, int hg, long long v0, long long v1, bool fin, int slot, long long rk) {
                         if (uniform((int)rk & 1))
                             chunk_piece<DT, QM, KVM, P2, RM, 4, KV8>(p, smem, pages, uniform(rg), uniform(hg),
                                                                 uniform(v0 / kShortKeyCost),
                                                                 uniform(v1 / kShortKeyCost), uniform((int)fin) != 0,
                                                                 uniform(slot), uniform(rk / kShortKeyCost));
                         else
                             chunk_piece<DT, QM, KVM, P2, RM, 1, KV8>(p, smem, pages, uniform(rg), uniform(hg),
                                                                 uniform(v0 / kLongKeyCost),
                                                                 uniform(v1 / kLongKeyCost), uniform((int)fin) != 0,
                                                                 uniform(slot), uniform(rk / kLongKeyCost));
                     });
    }
}

// The scale as the stage loops take it: positive, its sign in the queries' (exact), so that a
// hidden score of -inf stays one when it is scaled.  Zero becomes the smallest float, 2^-149:
// a finite score then adds less than 2^-21 to an exponent.
inline void fold_scale(DecodeParams& p) {
    p.qsign = p.l2scale < 0.0f ? 0x80008000u : 0u;
    p.loop_scale = p.l2scale == 0.0f ? __FLT_DENORM_MIN__ : __builtin_fabsf(p.l2scale);
}

template <bool KV8 = false>
inline size_t lds_bytes(int nrows) {
    return 256 + (size_t)kLdsRing<KV8> + (size_t)kPageCap * 4 + (size_t)(kWaves + nrows + 1) * sizeof(long long);
}

}  // namespace chunk
}  // namespace dv
