// Attention of the drafted nodes of token trees (dvattn_tree_paged_sdpa): the part
// beside the committed cache.
//
// Node s of sequence w sees the committed keys that its locations allow and, of the
// drafted rows, its ancestors and itself.  With x the base-2 scores,
//   out = sum_{l seen} 2^(x_l - m) v_l / sum_{l seen} 2^(x_l - m),
// and the sum splits into the committed keys, the same for every node of a tree, and
// a handful of ancestors that differ from node to node.  The committed part is the
// multi-query kernel's (dv_chunk / dv_chunk32: each K/V row read once per 16 nodes,
// every piece left as a partial result with its log-sum-exp); dv_merge_tree joins the
// pieces and adds the ancestors, whose rows it looks up one by one.  A drafted row
// that a node does not see is never loaded for it, so what siblings and absent nodes
// left in the cache, NaN included, cannot reach its output, as 0 * NaN would.
//
// Work per node is its depth, not the tree's size: a mask over all drafted rows on
// the matrix units would multiply S^2 pairs of which a tree of depth d sees S * d.
#include "dv_chunk.h"

namespace dv {
namespace chunk {

// Eight elements of a row as fp32.
template <int DT>
struct Run8 {
    u32x4 w[DT == kF32 ? 2 : 1];
    __device__ inline void load(const void* row, int d) {
        const unsigned char* b = reinterpret_cast<const unsigned char*>(row) + (long long)d * Tr<DT>::kBytes;
        w[0] = ld16(b);
        if constexpr (DT == kF32) w[1] = ld16(b + 16);
    }
    __device__ inline float operator[](int e) const {
        if constexpr (DT == kF32) return __uint_as_float(w[e >> 2][e & 3]);
        else return Tr<DT>::tof((uint16_t)(w[0][e >> 1] >> (16 * (e & 1))));
    }
};

// Ancestors, and committed pieces, whose rows are loaded together.  Four: eight would
// hold 76-100 registers instead of 64, fewer blocks per CU for a kernel that waits for
// memory (16 trees of 64 nodes: 51 us with eight, 35 with four; few long sequences with
// 30 pieces per segment: 9.1 and 10.0).
constexpr int kTreeBatch = 4;

// Block (segment, node of the group): thread t -> head t / 16, dims [(t % 16) * 8, +8).
// LDS: the sequence's parents, then the node's ancestors as cache rows, which the first
// wave looks up while the others join the committed pieces.  An absent node (its
// path leaves the tree at an entry that is no earlier node and not -1) writes zeros.
template <int DT>
__global__ __launch_bounds__(256) void dv_merge_tree(const DecodeParams p, int ntb) {
    using raw = typename Tr<DT>::raw;
    extern __shared__ int s_tree[];
    __shared__ int s_count;
    const int sg = blockIdx.x / ntb;
    const int tb = blockIdx.x - sg * ntb;
    const int r = sg / p.Hkv, hkv = sg - r * p.Hkv;
    const Grp gr = group_of<kRowWS>(p, p.row_begin + r);
    if (tb >= gr.ntok) return;
    const int tid = threadIdx.x;
    const int n = tid >> 4, d = (tid & 15) * 8;
    const int s = gr.s0 + tb, w = gr.w;
    const int h = hkv * kGqa + n;
    int* s_par = s_tree;
    int* s_row = s_tree + p.S;

    for (int i = tid; i < p.S; i += 256) s_par[i] = p.parents[(long long)w * p.S + i];
    const int base = p.dir[2 * sg], cnt = p.dir[2 * sg + 1];
    const int tv = p.tree_views[w], first = p.tree_rows[w];
    const bool has_view = tv >= 0 && tv < p.F;
    const long long row = ((long long)(has_view ? tv : 0) * p.W + w) * p.S + s;
    __syncthreads();
    if (tid < kWave) {
        int count = 0;
        if (tid == 0) {
            // every step goes to an earlier node, so the walk ends
            int j = s;
            for (;;) {
                const int up = s_par[j];
                s_row[count++] = j;
                if (up == -1) break;
                if (up < -1 || up >= j) {
                    count = -1;
                    break;
                }
                j = up;
            }
            s_count = count;
        }
        count = uniform(count);
        // ancestors -> cache rows (-1: not in the view, on no valid page, or at most the
        // node's location and so among the committed keys already)
        long long off = 0, len = 0;
        int loc = -1;
        if (has_view && count > 0) {
            for (int f = 0; f < tv; ++f) off += p.fl[f];
            len = p.fl[tv];
            loc = p.loc[row];
        }
        for (int i = tid; i < count; i += kWave) {
            const long long pos = (long long)first + s_row[i];
            const long long l = pos - off;
            int at = -1;
            if (l >= 0 && l < len && l > loc && pos >= 0) {
                const long long lp = p.bs_shift >= 0 ? pos >> p.bs_shift : (long long)((uint32_t)pos / (uint32_t)p.bs);
                if (lp < p.maxB) {
                    const int page = p.bt[(long long)w * p.maxB + lp];
                    if (page >= 0 && page < p.nblocks) at = (int)(uint32_t)((long long)page * p.bs + (pos - lp * p.bs));
                }
            }
            s_row[i] = at;
        }
    }

    // the committed keys' pieces: running base-2 maximum m, weight sum, weighted sum.
    // A piece that saw no key (-inf) holds nothing, whatever its values are.
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float m = -DV_INF, wsum = 0.0f;
    for (int k0 = 0; k0 < cnt; k0 += kTreeBatch) {
        float lse[kTreeBatch];
        int kx[kTreeBatch];
        Run8<kHalfPartials<DT> ? kF16 : kF32> x[kTreeBatch];
        const int jrow = tb * kGqa + n;
#pragma unroll
        for (int i = 0; i < kTreeBatch; ++i) {
            const bool in = k0 + i < cnt;
            const float* sp = p.part + (long long)(base + (in ? k0 + i : k0)) * p.slot_floats;
            lse[i] = in ? sp[kTokBlk * kGqa * kHeadDim + jrow] : -DV_INF;
            kx[i] = 0;
            if constexpr (kHalfPartials<DT>) {
                kx[i] = reinterpret_cast<const int*>(sp)[kTokBlk * kGqa * (kHeadDim / 2) + jrow];
                x[i].load(reinterpret_cast<const uint16_t*>(sp) + jrow * kHeadDim, d);
            } else {
                x[i].load(sp + jrow * kHeadDim, d);
            }
        }
        float bm = m;
#pragma unroll
        for (int i = 0; i < kTreeBatch; ++i) bm = fmaxf(bm, lse[i]);
        const float bz = bm == -DV_INF ? 0.0f : bm;
        const float sc = __builtin_amdgcn_exp2f(m - bz);
        wsum *= sc;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= sc;
#pragma unroll
        for (int i = 0; i < kTreeBatch; ++i) {
            if (lse[i] == -DV_INF) continue;
            const float wgt = __builtin_amdgcn_exp2f(lse[i] - bz);
            wsum += wgt;
            const float wv = __builtin_amdgcn_ldexpf(wgt, -kx[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(wv, x[i][e], v[e]);
        }
        m = bm;
    }
    float q[8];
    if (has_view) {
        raw qr[8];
        const raw* qrow = reinterpret_cast<const raw*>(p.q) + (((long long)w * p.Hq + h) * p.S + s) * kHeadDim;
        rotate_run<DT, 8>(qrow, p.cosv + row * p.R, p.sinv + row * p.R, p.R, d, qr);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = Tr<DT>::tof(qr[e]);
    }
    __syncthreads();
    const int count = s_count;
    raw* o = reinterpret_cast<raw*>(p.out) + out_row<kRowWS>(p, gr, tb, h) + d;
    if (count < 0) {
        const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        store_run8<DT>(o, zero);
        return;
    }

    // the ancestors: a row's 16 lanes hold one head's 128 dims
    const raw* kc = reinterpret_cast<const raw*>(p.kc);
    const raw* vc = reinterpret_cast<const raw*>(p.vc);
    for (int i0 = 0; i0 < count; i0 += kTreeBatch) {
        Run8<DT> kr[kTreeBatch], vr[kTreeBatch];
        bool in[kTreeBatch];
#pragma unroll
        for (int i = 0; i < kTreeBatch; ++i) {
            const int at = uniform(i0 + i < count ? s_row[i0 + i] : -1);
            in[i] = at != -1;
            if (in[i]) {
                const long long e = ((long long)(uint32_t)at * p.Hkv + hkv) * kHeadDim;
                kr[i].load(kc + e, d);
                vr[i].load(vc + e, d);
            }
        }
        float x[kTreeBatch];
        float bm = m;
#pragma unroll
        for (int i = 0; i < kTreeBatch; ++i) {
            x[i] = -DV_INF;
            if (in[i]) {
                float a = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) a = __builtin_fmaf(q[e], kr[i][e], a);
                x[i] = row16_sum(a) * p.l2scale;
                bm = fmaxf(bm, x[i]);
            }
        }
        const float bz = bm == -DV_INF ? 0.0f : bm;
        const float sc = __builtin_amdgcn_exp2f(m - bz);
        wsum *= sc;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= sc;
#pragma unroll
        for (int i = 0; i < kTreeBatch; ++i) {
            if (!in[i]) continue;
            const float wgt = __builtin_amdgcn_exp2f(x[i] - bz);
            wsum += wgt;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(wgt, vr[i][e], v[e]);
        }
        m = bm;
    }
    // no key at all: zeros (a NaN sum stays NaN)
    const float inv = wsum == 0.0f ? 0.0f : 1.0f / wsum;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= inv;
    store_run8<DT>(o, v);
}

}  // namespace chunk

hipError_t launch_merge_tree(int dtype, const DecodeParams& p, int ntb, hipStream_t stream) {
    const dim3 grid((unsigned)(p.nrows * p.Hkv * ntb)), block(256);
    const size_t lds = (size_t)p.S * 2 * sizeof(int);
    switch (dtype) {
        case kBF16: hipLaunchKernelGGL(chunk::dv_merge_tree<kBF16>, grid, block, lds, stream, p, ntb); break;
        case kF16: hipLaunchKernelGGL(chunk::dv_merge_tree<kF16>, grid, block, lds, stream, p, ntb); break;
        case kF32: hipLaunchKernelGGL(chunk::dv_merge_tree<kF32>, grid, block, lds, stream, p, ntb); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace dv
