// gfx950 decode attention with fused query RoPE over a paged cache held in 8 bits:
// E4M3 bytes [num_blocks, block_size, Hkv, 128] and one exponent byte b per page and KV
// head, so that a cached element is byte * 2^(b - 127) (b = 0: zero).  Rows, views,
// rotation, work split and merge are the 16-bit decode's (dv_decode.hip).
//
//  * One wave owns one KV head and its 16 query heads of one row over a range of the
//    row's keys; up to four such waves (KV heads) make a workgroup.
//  * A stage is 32 keys: 4 KiB of K, 4 KiB of V and the 64 exponent bytes of its rows,
//    moved by nine direct-to-LDS loads into a ring of four stages private to the wave,
//    three of them in flight beside the one computed.  The exponents travel with their
//    rows, so pages of any size may end inside a stage.
//  * K bytes are widened to the 16-bit MFMA operand (every E4M3 number is one of bf16 and
//    of fp16): S^T = K Q^T on 16x16x32 MFMA, and the page's 2^(b - 127) multiplies the
//    fp32 score.  V^T comes from the transposing 8-bit LDS read, widened to bf16, and V's
//    2^(b - 127) multiplies the probability before it is rounded (a power of two: the
//    rounding is the same with and without).
//  * Precision: bf16 calls take one operand for Q and P, as the 16-bit decode does.  fp16
//    calls take Q as it is against K in fp16, and P as a bf16 pair hi + lo (16 bits).
//    fp32 calls take Q and P as three bf16 numbers each, which hold 24 bits: the products
//    with exact K and V lose nothing that fp32 arithmetic keeps.
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
constexpr int kRing = 4;                        // stages per wave
constexpr int kLoads = 9;                       // direct-to-LDS loads per stage
constexpr int kWaveLds = kRing * kStage + stream::kPc * 4;

// MFMA operands of a query (or probability) value: 16-bit parts that sum to it.
template <int DT> constexpr int kQParts = DT == kF32 ? 3 : 1;
template <int DT> constexpr int kPParts = DT == kF32 ? 3 : DT == kF16 ? 2 : 1;
template <int DT> constexpr int kKType = DT == kF16 ? kF16 : kBF16;

// A byte per lane from global memory into the LDS word at lds_base + 4 * lane.
__device__ inline void dma1(const void* gptr, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, off" ::"v"(gptr), "s"(lds_base)
                 : "memory", "m0");
}

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

// 2^(b - 127) of an exponent byte (0: zero).
__device__ inline float power_of(uint32_t b) { return __uint_as_float(b << 23); }

// Issues the loads of the stage holding keys [l, l + 32) into the ring slot at LDS address
// sbase; returns the visibility mask of its keys.
__device__ inline uint32_t issue(const DecodeParams& p, const stream::View& v, const int* pc, uint32_t sbase, int l) {
    const int lane = threadIdx.x & 63;
    // page and in-page offset of the row of key l + k, or page -1
    auto find = [&](int k, uint32_t& r) {
        const int pos = v.off + l + k;
        uint32_t q, x;
        page_split(p, (uint32_t)(pos > 0 ? pos : 0), q, x);
        const uint32_t idx = q - (uint32_t)v.lp0;
        const int page = pc[idx < (uint32_t)stream::kPc ? idx : (uint32_t)(stream::kPc - 1)];
        r = x;
        return l + k < v.b && pos >= 0 && idx < (uint32_t)stream::kPc ? page : -1;
    };
    const unsigned char* ka[4];
    const unsigned char* va[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = i * 8 + (lane >> 3);
        uint32_t r;
        const int page = find(k, r);
        const uint32_t row = ((uint32_t)page * (uint32_t)p.bs + r) * (uint32_t)p.Hkv + (uint32_t)v.hkv;
        const unsigned long long off = (unsigned long long)row * kRowB;
        const int pk = ((lane & 7) ^ swz_k(k)) * 16, pv = ((lane & 7) ^ swz_v(k)) * 16;
        ka[i] = page >= 0 ? v.k + off + pk : g_zero_row + pk;
        va[i] = page >= 0 ? v.v + off + pv : g_zero_row + pv;
    }
    uint32_t r;
    const int page = find(lane & 31, r);
    const unsigned char* sb = lane < 32 ? p.ks : p.vs;
    const unsigned char* sa = page >= 0 ? sb + (unsigned long long)page * (uint32_t)p.Hkv + v.hkv : g_zero_row;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        dma16(ka[i], sbase + (uint32_t)(i * 1024));
        dma16(va[i], sbase + (uint32_t)(kTile + i * 1024));
    }
    dma1(sa, sbase + (uint32_t)(2 * kTile));
    return (uint32_t)ballot(page >= 0 && lane < 32);
}

// A query row's 16-bit MFMA operands: lane (g, n) holds dims c * 32 + g * 8 .. + 8 of head n.
template <int DT>
struct QOp {
    u32x4 q[kQParts<DT>][4];
};

// fp32: the three bf16 numbers that sum to x (each part rounds what the ones before left).
__device__ inline void split3(float x, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    const uint16_t h = Tr<kBF16>::fromf(x);
    const float r = x - Tr<kBF16>::tof(h);
    const uint16_t m = Tr<kBF16>::fromf(r);
    const uint16_t l = Tr<kBF16>::fromf(r - Tr<kBF16>::tof(m));
    hi = h;
    mid = m;
    lo = l;
}

template <int DT, int QM, int RM>
__device__ inline void load_q(const DecodeParams& p, int row, int f, int hkv, QOp<DT>& o) {
    if constexpr (DT != kF32) {
        load_q16<DT, QM, RM>(p, row, f, hkv, o.q[0]);
    } else {
        const int lane = threadIdx.x & 63;
        const int g = lane >> 4, n = lane & 15;
        const int h = hkv * kGqa + n;
        const float* q;
        long long co;
        if (QM == kQRotFull) {
            const int w = row / p.S, s = row - (row / p.S) * p.S;
            q = reinterpret_cast<const float*>(p.q) + (((long long)w * p.Hq + h) * p.S + s) * kHeadDim;
            co = (((long long)f * p.W + w) * p.S + s) * p.R;
        } else {
            q = reinterpret_cast<const float*>(p.q) + ((long long)row * p.Hq + h) * kHeadDim;
            co = ((long long)f * p.T + row) * (p.R >> 1);
        }
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
            float r[8];
            rotate_run<kF32, 8>(q, p.cosv + co, p.sinv + co, p.R, cc * 32 + g * 8, r);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                uint32_t a[3], b[3];
                split3(r[2 * t], a[0], a[1], a[2]);
                split3(r[2 * t + 1], b[0], b[1], b[2]);
#pragma unroll
                for (int k = 0; k < 3; ++k) o.q[k][cc][t] = a[k] | (b[k] << 16);
            }
        }
    }
}

// P^T operands of a lane's eight probabilities times their rows' V scales, and the row
// sum's share of them.
template <int DT>
struct POp {
    u32x4 w[kPParts<DT>];
};

template <int DT>
__device__ inline POp<DT> p_scaled(const float (&pr)[8], const float (&vs)[8], float& l) {
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
        float a = pr[2 * i] * vs[2 * i], b = pr[2 * i + 1] * vs[2 * i + 1];
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

// One stage.
template <int DT>
__device__ inline void compute(State& st, uint32_t slot, uint32_t mask, const QOp<DT>& q, float l2scale) {
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, n = lane & 15;
    f32x4 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        s[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int row = kb * 16 + n;
        const uint32_t base = slot + (uint32_t)(row * kRowB + (g & 1) * 8);
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
            const u32x4 k = widen8<kKType<DT>>(
                lds_read8_at(base + (uint32_t)(((cc * 2 + (g >> 1)) ^ swz_k(row)) * 16)));
#pragma unroll
            for (int j = 0; j < kQParts<DT>; ++j) s[kb] = Tr<kKType<DT>>::mma(k, q.q[j][cc], s[kb]);
        }
    }
    float vs[8];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        const u32x4 a = lds_read16_at(slot + (uint32_t)(2 * kTile + (kb * 16 + g * 4) * 4));
        const u32x4 b = lds_read16_at(slot + (uint32_t)(2 * kTile + (32 + kb * 16 + g * 4) * 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[kb][i] *= power_of(a[i]);
            vs[kb * 4 + i] = power_of(b[i]);
        }
    }
    float pr[8];
    softmax32<false>(st.o, st.m, st.l, s[0], s[1], mask, l2scale, pr);
    const POp<DT> pB = p_scaled<DT>(pr, vs, st.l);
    // V^T operand of dims [cc * 16, + 16): k = g * 8 + j <-> key (j / 4) * 16 + g * 4 + j % 4
    const int j = n >> 1;
    const int row = (j >> 2) * 16 + g * 4 + (j & 3);
    const uint32_t base = slot + (uint32_t)(kTile + row * kRowB + (n & 1) * 8);
#pragma unroll
    for (int cc = 0; cc < 8; ++cc) {
        const u32x4 v = widen8<kBF16>(lds_read_tr8_at(base + (uint32_t)((cc ^ swz_v(row)) * 16)));
#pragma unroll
        for (int k = 0; k < kPParts<DT>; ++k) st.o[cc] = Tr<kBF16>::mma(v, pB.w[k], st.o[cc]);
    }
    mfma_settle_acc(st.o);
}

// One wave: KV head hkv over visible keys [v0, v1) of one row.
template <int DT, int QM, int RM, bool MV>
__device__ __forceinline__ void piece(const DecodeParams& p, unsigned char* wlds, int row, int hkv, long long v0, long long v1,
                      bool final_out, int slot, int wv, long long row_keys) {
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, n = lane & 15;
    const uint32_t ring = __builtin_amdgcn_readfirstlane(lds_addr(wlds));
    int* pc = reinterpret_cast<int*>(wlds + kRing * kStage);
    const int w = RM == kRowVarlen ? varlen_seq(p, row) : row / p.S;

    State st;
#pragma unroll
    for (int c = 0; c < 8; ++c) st.o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    st.m = -DV_INF;
    st.l = 0.0f;

    auto one_view = [&](int f, int vis, long long P, long long off) {
        const long long a = v0 > P ? v0 : P;
        const long long bnd = v1 < P + vis ? v1 : P + vis;
        const int l0 = (int)(a - P), l1 = (int)(bnd - P);
        stream::View v;
        v.hkv = hkv;
        v.k = reinterpret_cast<const unsigned char*>(p.kc);
        v.v = reinterpret_cast<const unsigned char*>(p.vc);
        v.off = (int)off;
        QOp<DT> q;
        // sub-ranges whose pages fit the page cache, whole stages
        long long span = ((long long)(stream::kPc - 2) * p.bs) & ~(long long)(kStep - 1);
        span = span < (1ll << 30) ? (span < kStep ? kStep : span) : 1ll << 30;
        for (int sa = l0; sa < l1;) {
            const int sb = (long long)l1 - sa > span ? (int)(sa + span) : l1;
            v.b = sb;
            uint32_t lpa, lpz, r;
            const int pa = v.off + sa, pz = v.off + sb - 1;
            page_split(p, pa > 0 ? (uint32_t)pa : 0u, lpa, r);
            page_split(p, pz > 0 ? (uint32_t)pz : 0u, lpz, r);
            v.lp0 = (int)lpa;
            stream::fill_pages(p, p.bt + (long long)w * p.maxB, pc, (int)(lpz - lpa) + 1,
                               [&](int i) { return lpa + (uint32_t)i; });
            const int ns = (sb - sa + kStep - 1) / kStep;
            uint32_t m0 = 0, m1 = 0, m2 = 0;
            m0 = issue(p, v, pc, ring, sa);
            if (ns > 1) m1 = issue(p, v, pc, ring + kStage, sa + kStep);
            if (ns > 2) m2 = issue(p, v, pc, ring + 2 * kStage, sa + 2 * kStep);
            if (sa == l0) {
                load_q<DT, QM, RM>(p, row, f, hkv, q);
                // settled here: a load still pending at the loop would make the compiler
                // wait for all vector memory in every step
#pragma unroll
                for (int k = 0; k < kQParts<DT>; ++k)
#pragma unroll
                    for (int cc = 0; cc < 4; ++cc) asm volatile("" : "+v"(q.q[k][cc]));
            }
            for (int s = 0; s < ns; ++s) {
                if (s + 2 < ns) wait_vmcnt<2 * kLoads>();
                else if (s + 1 < ns) wait_vmcnt<kLoads>();
                else wait_vmcnt<0>();
                uint32_t m3 = 0;
                lds_wait();  // the reads of stage s - 1 are complete before its slot is refilled
                if (s + 3 < ns)
                    m3 = issue(p, v, pc, ring + (uint32_t)(((s + 3) & (kRing - 1)) * kStage), sa + (s + 3) * kStep);
                compute<DT>(st, ring + (uint32_t)((s & (kRing - 1)) * kStage), m0, q, p.l2scale);
                m0 = m1;
                m1 = m2;
                m2 = m3;
            }
            lds_wait();
            sa = sb;
        }
    };
    if constexpr (!MV) {
        if (v0 < v1) one_view(0, (int)row_keys, 0ll, 0ll);
    } else if (v0 < v1) {
        for_views_blocks<kKvPaged, RM>(p, row, v0, v1, [&](int f, int vis, long long P, long long off) {
            one_view(f, uniform(vis), uniform(P), uniform(off));
        });
    }

    // epilogue: total over the four lane groups, normalise, base-2 log-sum-exp
    const float lt = rows4_sum(st.l);
    const float inv = lt > 0.0f ? 1.0f / lt : 0.0f;
    const int h = hkv * kGqa + n;
    if (final_out) {
        using raw = typename Tr<DT>::raw;
        raw* o;
        if (RM == kRowVarlen) {
            o = reinterpret_cast<raw*>(p.out) + ((long long)row * p.Hq + h) * kHeadDim;
        } else {
            const int s = row - w * p.S;
            o = reinterpret_cast<raw*>(p.out) + (((long long)w * p.Hq + h) * p.S + s) * kHeadDim;
        }
        if (lt != lt)  // a NaN score: the row is NaN, not the zeros of a row without keys
#pragma unroll
            for (int c = 0; c < 8; ++c) st.o[c] = f32x4{lt, lt, lt, lt};
        const float scale = lt != lt ? 1.0f : inv;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int d = c * 16 + g * 4;
            if constexpr (DT == kF32)
                *reinterpret_cast<f32x4*>(o + d) = st.o[c] * scale;
            else
                *reinterpret_cast<u32x2*>(o + d) = u32x2{pack2<DT>(st.o[c][0] * scale, st.o[c][1] * scale),
                                                         pack2<DT>(st.o[c][2] * scale, st.o[c][3] * scale)};
        }
    } else {
        store_partial<DT>(p.part + (long long)slot * p.slot_floats, p.hpw * kGqa, wv * kGqa + n, g, st.o, inv,
                          row_lse(st.m, lt));
    }
}

}  // namespace q8

// MV: calls of several views (or none), whose pieces may start anywhere.
template <int DT, int QM, int RM, bool MV>
__global__ __launch_bounds__(256) void dv_decode8(const DecodeParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ long long s_scan[4];
    const int wv = uniform((int)(threadIdx.x >> 6));
    const int HPW = p.hpw;
    long long* s_pref = reinterpret_cast<long long*>(smem + HPW * q8::kWaveLds);
    unsigned char* wlds = smem + wv * q8::kWaveLds;
    run_schedule<true, MV ? 1 : kStep, 1, true>(
        p, p.Hkv / HPW, s_pref, s_scan, [&](int row) { return row_visible<kKvPaged, RM>(p, row); },
        [&](int row, int hg, long long v0, long long v1, bool fin, int slot, long long rk) {
            if (wv < HPW)
                q8::piece<DT, QM, RM, MV>(p, wlds, uniform(row), uniform(hg) * HPW + wv, uniform(v0), uniform(v1),
                                      uniform((int)fin) != 0, uniform(slot), wv, uniform(rk));
        });
}

// ---- host side --------------------------------------------------------------------

namespace {

template <int DT, int QM, int RM, bool MV>
hipError_t launch8_one(DecodeParams p, int device, long long cap, int cus, hipStream_t stream) {
    const void* kern = reinterpret_cast<const void*>(&dv_decode8<DT, QM, RM, MV>);
    auto lds_of = [](int hpw, int nrows) {
        return (size_t)hpw * q8::kWaveLds + (size_t)(nrows + 1) * sizeof(long long);
    };
    static std::atomic<unsigned long long> attr_done{0};
    hipError_t e = once_per_device(attr_done, device, [&] {
        return hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)lds_of(kMaxWavesPerWg, kMaxRows));
    });
    if (e != hipSuccess) return e;
    // workgroups that are all resident at once: four waves fill a CU's LDS
    const long long nwg = (long long)cus * (kMaxWavesPerWg / p.hpw);
    p.nwg = (int)(nwg < cap ? nwg : cap < 1 ? 1 : cap);
    hipLaunchKernelGGL((dv_decode8<DT, QM, RM, MV>), dim3(p.nwg), dim3(p.hpw * kWave), lds_of(p.hpw, p.nrows), stream,
                       p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    return launch_merge(DT, RM, p, stream);
}

template <int DT, int QM, int RM>
hipError_t launch8(const DecodeParams& p, int device, long long cap, int cus, hipStream_t stream) {
    if (p.F == 1) return launch8_one<DT, QM, RM, false>(p, device, cap, cus, stream);
    return launch8_one<DT, QM, RM, true>(p, device, cap, cus, stream);
}

}  // namespace

hipError_t launch_decode8(int dtype, int qmode, int rowmode, const DecodeParams& base, int nrows_total,
                          long long max_keys_per_row, void* workspace, size_t ws_bytes, hipStream_t stream) {
    if (nrows_total <= 0 || base.Hkv <= 0) return hipSuccess;
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    if (ws_bytes < decode_workspace_bytes(nrows_total, base.Hkv, device, dtype)) return hipErrorInvalidValue;
    DecodeParams p = base;
    p.hpw = pick_hpw(p.Hkv);
    const int nhg = p.Hkv / p.hpw;
    p.slot_floats = p.hpw * kGqa * (kHeadDim + 1);
    const int cus = device_cu_count(device);
    // decode_workspace_bytes' layout: slots of as many workgroups and segments as a launch has
    const long long nseg_cap = (long long)(nrows_total < kMaxRows ? nrows_total : kMaxRows) * nhg;
    const long long slots_cap = (long long)cus * (8 / p.hpw) + nseg_cap;
    const size_t part_bytes = ((size_t)(slots_cap * p.slot_floats * 4) + 255) & ~(size_t)255;
    unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
    p.part = reinterpret_cast<float*>(ws);
    p.dir = reinterpret_cast<int*>(ws + part_bytes);
    p.piece_cost = kPieceCost;
    p.skew_pm = xcd_skew_pm();
    const bool varlen = rowmode == kRowVarlen;
    if (varlen != (qmode == kQRotHalf)) return hipErrorInvalidValue;
    for (int r0 = 0; r0 < nrows_total; r0 += kMaxRows) {
        p.row_begin = r0;
        p.nrows = nrows_total - r0 < kMaxRows ? nrows_total - r0 : kMaxRows;
        const long long cap =
            ((long long)p.nrows * nhg * (max_keys_per_row + p.piece_cost) + p.min_keys - 1) / p.min_keys;
        switch (dtype) {
            case kBF16: e = varlen ? launch8<kBF16, kQRotHalf, kRowVarlen>(p, device, cap, cus, stream)
                                   : launch8<kBF16, kQRotFull, kRowWS>(p, device, cap, cus, stream); break;
            case kF16: e = varlen ? launch8<kF16, kQRotHalf, kRowVarlen>(p, device, cap, cus, stream)
                                  : launch8<kF16, kQRotFull, kRowWS>(p, device, cap, cus, stream); break;
            case kF32: e = varlen ? launch8<kF32, kQRotHalf, kRowVarlen>(p, device, cap, cus, stream)
                                  : launch8<kF32, kQRotFull, kRowWS>(p, device, cap, cus, stream); break;
            default: e = hipErrorInvalidValue;
        }
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace dv
