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
//
// 16 trees of 64 nodes over 8192 keys, 8 KV heads in bf16: 621 us a call (650 TFLOP/s), of
// which the merge is 32-35 and the multi-query kernel the rest (685 TFLOP/s).
//
// Short sequences take one launch instead (dv_tree_small, below).
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

// Node s and its ancestors, from the node up; their number, or -1 for an absent node (its
// path leaves the tree at an entry that is no earlier node and not -1).  Every step goes
// to an earlier node, so the walk ends.
__device__ inline int walk_path(const int* parents, int s, int* path) {
    int count = 0;
    for (;;) {
        const int up = parents[s];
        path[count++] = s;
        if (up == -1) return count;
        if (up < -1 || up >= s) return -1;
        s = up;
    }
}

// Cache row (without its KV head) of stream row pos of sequence w, or -1 if it lies on no
// valid page.
__device__ inline int page_row(const DecodeParams& p, int w, long long pos) {
    if (pos < 0) return -1;
    const long long lp = p.bs_shift >= 0 ? pos >> p.bs_shift : (long long)((uint32_t)pos / (uint32_t)p.bs);
    if (lp >= p.maxB) return -1;
    const int page = p.bt[(long long)w * p.maxB + lp];
    return page >= 0 && page < p.nblocks ? (int)(uint32_t)((long long)page * p.bs + (pos - lp * p.bs)) : -1;
}

// Ancestors, and committed pieces, whose rows are loaded together.  Four: eight would
// hold 76-100 registers instead of 64, fewer blocks per CU for a kernel that waits for
// memory (16 trees of 64 nodes: 51 us with eight, 35 with four; few long sequences with
// 30 pieces per segment: 9.1 and 10.0).
constexpr int kTreeBatch = 4;

// Block (segment, node of the group): thread t -> head t / 16, dims [(t % 16) * 8, +8).
// LDS: the sequence's parents, then the node's ancestors as cache rows, which the first
// wave looks up while the others join the committed pieces.  An absent node writes zeros.
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
            count = walk_path(s_par, s, s_row);
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
            s_row[i] = l >= 0 && l < len && l > loc ? page_row(p, w, pos) : -1;
        }
    }

    // the committed keys' pieces: running base-2 maximum m, weight sum, weighted sum.
    // A piece that saw no key (-inf) holds nothing, whatever its values are; one with a NaN
    // score has a NaN log-sum-exp (row_lse), which reaches the output.
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

// ---- short sequences -------------------------------------------------------------
//
// With few keys the call above is two launches' fixed times (a view's start alone costs a
// workgroup of the first 11 - 13 us).  Here a block of eight waves for each (sequence, KV
// head, node) goes through the list of the node's keys, the committed ones of each view
// and then its path, every view's part rounded up to tiles of 16 entries (so a tile has
// one rotated query):
//   scores S^T = K Q^T by tiles (the waves take turns), left in LDS with each head's
//   maximum; weights 2^(x - m) in place with each head's sum; O^T = V^T P by steps of four
//   keys on 16x16x4 fp32 MFMAs, whatever the cache's type: a lane's 16-byte load of V row
//   4 * step + g is one element of each of the step's MFMAs, so V needs no transposing
//   and the weights no rounding.  Last, the waves' sums are joined in order.
// A list of more than 640 entries, or one that few blocks would have to take in long
// turns, is cut into windows, a block each, whose sums a second launch joins; the path
// goes with the first window.
constexpr int kSmallWaves = 8;
constexpr int kSmallThreads = kSmallWaves * kWave;
constexpr int kSmallAhead = 4;                // V steps under way together
constexpr int kEntries = 640;                 // of a block's list: two blocks share a CU
constexpr int kSmallQueryBytes = 16 * 1024;   // the views' queries in LDS
// Read in place of a list entry without a row: loads without branches can be on their way
// together.
__device__ __align__(16) unsigned char no_row[kHeadDim * 4];
template <int DT> constexpr int kQPieces = kHeadDim * Tr<DT>::kBytes / 64;  // 16-byte pieces of a row per lane

// A window's sums: [16 heads, 128 dims], then each head's maximum and sum of weights.  A
// sum below zero marks an absent node.
constexpr int kSlot = kGqa * kHeadDim + 2 * kGqa;

template <int DT, bool SPLIT>
__global__ __launch_bounds__(kSmallThreads) void dv_tree_small(const DecodeParams p, int windows, int window) {
    using raw = typename Tr<DT>::raw;
    constexpr int kP = kQPieces<DT>;
    constexpr int kRowBytes = kHeadDim * Tr<DT>::kBytes;
    constexpr int kRun = 16 / Tr<DT>::kBytes;     // elements of a piece
    constexpr int kMaxViews = kSmallQueryBytes / (kP * kWave * 16);
    __shared__ __align__(16) float s_x[kEntries * kGqa];
    __shared__ __align__(16) int s_row[kEntries];
    __shared__ int s_par[kEntries];
    __shared__ u32x4 s_q[kMaxViews * kP * kWave];
    __shared__ float s_m[kSmallWaves][kGqa], s_l[kSmallWaves][kGqa];
    __shared__ int s_count;
    const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int hkv = blockIdx.x % p.Hkv;
    const int item = blockIdx.x / p.Hkv;
    const int ws = SPLIT ? item / windows : item;
    const int part = SPLIT ? item - ws * windows : 0;
    const int w = ws / p.S, s = ws - w * p.S;
    for (int i = tid; i < p.S; i += kSmallThreads) s_par[i] = p.parents[(long long)w * p.S + i];
    // per view: its first stream row, and the list's entries before it
    long long off[kMaxViews];
    int at[kMaxViews + 1], seen[kMaxViews];
    const long long rows = (long long)p.maxB * p.bs;
    const int room = windows * window;
    const int tv = p.tree_views[w], first = p.tree_rows[w];
    long long own_off = 0;
    int own_len = 0, own_loc = -1;
    at[0] = 0;
    {
        long long o = 0;
#pragma unroll
        for (int f = 0; f < kMaxViews; ++f) {
            off[f] = o;
            seen[f] = 0;
            if (f < p.F) {
                const int len = p.fl[f], loc = p.loc[((long long)f * p.W + w) * p.S + s];
                const long long most = loc >= len - 1 ? len : (long long)loc + 1;
                long long here = most < rows - o ? most : rows - o;
                // (lengths below zero could make views overlap: the list ends where it ends)
                here = here < room - at[f] ? here : room - at[f];
                seen[f] = here > 0 ? (int)here : 0;
                if (f == tv) {
                    own_off = o;
                    own_len = len;
                    own_loc = loc;
                }
                o += len;
            }
            at[f + 1] = at[f] + (seen[f] + 15) / 16 * 16;
        }
    }
    // this block's committed entries: [lo, lo + base) of the list
    const int lo = SPLIT ? part * window : 0;
    const int rest = at[kMaxViews] - lo;
    const int base = rest < 0 ? 0 : rest < window ? rest : window;
    float* slot = SPLIT ? p.part + ((long long)ws * p.Hkv + hkv) * windows * kSlot + part * kSlot : nullptr;
    if (SPLIT && part > 0 && base == 0) {
        if (tid < 2 * kGqa) slot[kGqa * kHeadDim + tid] = tid < kGqa ? -DV_INF : 0.0f;
        return;
    }
    const bool has_view = tv >= 0 && tv < p.F;
    __syncthreads();
    if (wv == 0) {
        int count = 0;
        if (lane == 0) s_count = count = part > 0 ? 0 : walk_path(s_par, s, s_row + base);
        count = uniform(count);
        if (count > 0)
            for (int i = lane; i < (count + 15) / 16 * 16; i += kWave) {
                int r = -1;
                if (has_view && i < count) {
                    const long long pos = (long long)first + s_row[base + i];
                    const long long l = pos - own_off;
                    if (l >= 0 && l < own_len && l > own_loc) r = page_row(p, w, pos);
                }
                s_row[base + i] = r;
            }
    } else {
        const int t0 = tid - kWave, nt = kSmallThreads - kWave;
        for (int i = t0; i < base; i += nt) {
            int r = -1;
#pragma unroll
            for (int f = 0; f < kMaxViews; ++f)
                if (lo + i >= at[f] && lo + i - at[f] < seen[f]) r = page_row(p, w, off[f] + (lo + i - at[f]));
            s_row[i] = r;
        }
        // the token's 16 heads in the MFMA's operand order, rotated for each view
        for (int i = t0; i < p.F * kP * kWave; i += nt) {
            const int f = i / (kP * kWave), piece = i - f * (kP * kWave);
            const int cc = piece >> 6, h = hkv * kGqa + (piece & 15);
            const raw* qrow = reinterpret_cast<const raw*>(p.q) + (((long long)w * p.Hq + h) * p.S + s) * kHeadDim;
            const long long cs = (((long long)f * p.W + w) * p.S + s) * p.R;
            // (through a register on its way to LDS: kept in LDS, the array is indexed by what
            // each block would fetch from the launch packet, 5 - 13 us of a call)
            raw r[kRun];
            rotate_run<DT, kRun>(qrow, p.cosv + cs, p.sinv + cs, p.R, (cc * 4 + ((piece >> 4) & 3)) * kRun, r);
            u32x4 v;
            __builtin_memcpy(&v, r, 16);
            s_q[i] = v;
        }
    }
    __syncthreads();
    const int count = s_count;
    if (count < 0) {
        raw* o = reinterpret_cast<raw*>(p.out) + (((long long)w * p.Hq + hkv * kGqa) * p.S + s) * kHeadDim;
        if constexpr (SPLIT) {
            if (tid < 2 * kGqa) slot[kGqa * kHeadDim + tid] = tid < kGqa ? -DV_INF : -1.0f;
            return;
        }
        for (int i = tid; i < kGqa * kHeadDim; i += kSmallThreads)
            o[(long long)(i / kHeadDim) * p.S * kHeadDim + i % kHeadDim] = raw(0);
        return;
    }
    const int tiles = (base + count + 15) / 16;

    // scores
    float mx = -DV_INF;
#pragma unroll 2
    for (int t = wv; t < tiles; t += kSmallWaves) {
        const int row = s_row[t * 16 + n];
        u32x4 k[kP];
        const unsigned char* src = (row != -1 ? reinterpret_cast<const unsigned char*>(p.kc) +
                                                    ((unsigned long long)(uint32_t)row * p.Hkv + hkv) * kRowBytes
                                              : no_row) +
                                   g * 16;
#pragma unroll
        for (int cc = 0; cc < kP; ++cc) k[cc] = ld16(src + cc * 64);
        int f = 0;
#pragma unroll
        for (int v = 1; v < kMaxViews; ++v) f = lo + t * 16 >= at[v] ? v : f;
        if (t * 16 >= base) f = has_view ? tv : 0;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int cc = 0; cc < kP; ++cc) {
            const u32x4 q = s_q[(f * kP + cc) * kWave + lane];
            if constexpr (DT == kF32) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    x = Tr<kF32>::mma1(__builtin_bit_cast(f32x4, k[cc])[j], __builtin_bit_cast(f32x4, q)[j], x);
            } else {
                x = Tr<DT>::mma(k[cc], q, x);
            }
        }
        const int4 ids = *reinterpret_cast<const int4*>(s_row + t * 16 + g * 4);
        x[0] = ids.x != -1 ? x[0] * p.l2scale : -DV_INF;
        x[1] = ids.y != -1 ? x[1] * p.l2scale : -DV_INF;
        x[2] = ids.z != -1 ? x[2] * p.l2scale : -DV_INF;
        x[3] = ids.w != -1 ? x[3] * p.l2scale : -DV_INF;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s_x[(t * 16 + g * 4 + i) * kGqa + n] = x[i];
            mx = fmaxf(mx, x[i]);
        }
    }
    mx = rows4_max(mx);
    if (lane < kGqa) s_m[wv][lane] = mx;
    __syncthreads();

    // weights; every thread meets one head only
    float m = -DV_INF;
#pragma unroll
    for (int v = 0; v < kSmallWaves; ++v) m = fmaxf(m, s_m[v][n]);
    const float mz = m == -DV_INF ? 0.0f : m;
    float l = 0.0f;
    for (int i = tid; i < tiles * 16 * kGqa; i += kSmallThreads) {
        const float e = __builtin_amdgcn_exp2f(s_x[i] - mz);
        s_x[i] = e;
        l += e;
    }
    l = rows4_sum(l);
    if (lane < kGqa) s_l[wv][lane] = l;
    __syncthreads();

    // the weighted sums: acc[e] holds dims (g * 4 + i) * 8 + e of head n (fp32: two
    // pieces of four dims, (g * 4 + i) * 4 + e and 64 more)
    f32x4 acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll kSmallAhead
    for (int st = wv; st < tiles * 4; st += kSmallWaves) {
        const int row = s_row[st * 4 + g];
        const float e = s_x[(st * 4 + g) * kGqa + n];
        u32x4 v[DT == kF32 ? 2 : 1];
        const unsigned char* src = (row != -1 ? reinterpret_cast<const unsigned char*>(p.vc) +
                                                    ((unsigned long long)(uint32_t)row * p.Hkv + hkv) * kRowBytes
                                              : no_row) +
                                   n * 16;
        v[0] = ld16(src);
        if constexpr (DT == kF32) v[1] = ld16(src + 256);
        raw r[8];
        __builtin_memcpy(r, v, sizeof(v));
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = Tr<kF32>::mma1(Tr<DT>::tof(r[j]), e, acc[j]);
    }
    __syncthreads();  // the weights are read; their space takes the waves' sums
    f32x4* s_acc = reinterpret_cast<f32x4*>(s_x);
    static_assert(sizeof(s_x) >= kSmallWaves / 2 * 8 * kWave * 16, "half of the waves' sums");
    if (wv >= kSmallWaves / 2)
#pragma unroll
        for (int j = 0; j < 8; ++j) s_acc[((wv - kSmallWaves / 2) * 8 + j) * kWave + lane] = acc[j];
    __syncthreads();
    if (wv < kSmallWaves / 2)
#pragma unroll
        for (int j = 0; j < 8; ++j) s_acc[(wv * 8 + j) * kWave + lane] += acc[j];
    __syncthreads();

    // thread -> head tid / 32, dims [tid % 32 * 4, +4)
    const int h = tid >> 5, d = (tid & 31) * 4;
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < kSmallWaves; ++v) sum += s_l[v][h];
    // no key at all: zeros (a NaN sum stays NaN)
    const float inv = SPLIT ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = DT == kF32 ? (d >> 6) * 4 + j : (d & 7) + j;
        const int r = DT == kF32 ? (d & 63) >> 2 : d >> 3;
        float a = 0.0f;
#pragma unroll
        for (int v = 0; v < kSmallWaves / 2; ++v)
            a += s_x[((v * 8 + e) * kWave + (r >> 2) * 16 + h) * 4 + (r & 3)];
        o[j] = a * inv;
    }
    if constexpr (SPLIT) {
        *reinterpret_cast<f32x4*>(slot + h * kHeadDim + d) = f32x4{o[0], o[1], o[2], o[3]};
        if (tid < kGqa) slot[kGqa * kHeadDim + tid] = m;
        if (d == 0) slot[kGqa * kHeadDim + kGqa + h] = sum;
        return;
    }
    raw* dst = reinterpret_cast<raw*>(p.out) + (((long long)w * p.Hq + hkv * kGqa + h) * p.S + s) * kHeadDim + d;
    if constexpr (DT == kF32) *reinterpret_cast<f32x4*>(dst) = f32x4{o[0], o[1], o[2], o[3]};
    else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
}

// Block (sequence, node, KV head): thread t -> head t / 16, dims [(t % 16) * 8, +8).
template <int DT>
__global__ __launch_bounds__(256) void dv_tree_join(const DecodeParams p, int windows) {
    const int n = threadIdx.x >> 4, d = (threadIdx.x & 15) * 8;
    const int hkv = blockIdx.x % p.Hkv;
    const int ws = blockIdx.x / p.Hkv;
    const int w = ws / p.S, s = ws - w * p.S;
    const float* slots = p.part + ((long long)ws * p.Hkv + hkv) * windows * kSlot;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float m = -DV_INF, sum = 0.0f;
    const bool absent = slots[kGqa * kHeadDim + kGqa + n] < 0.0f;
    for (int k0 = 0; k0 < windows && !absent; k0 += kTreeBatch) {
        float km[kTreeBatch], ks[kTreeBatch];
        Run8<kF32> x[kTreeBatch];
#pragma unroll
        for (int i = 0; i < kTreeBatch; ++i) {
            const bool in = k0 + i < windows;
            const float* sp = slots + (long long)(in ? k0 + i : k0) * kSlot;
            km[i] = in ? sp[kGqa * kHeadDim + n] : -DV_INF;
            ks[i] = in ? sp[kGqa * kHeadDim + kGqa + n] : 0.0f;
            x[i].load(sp + n * kHeadDim, d);
        }
        float bm = m;
#pragma unroll
        for (int i = 0; i < kTreeBatch; ++i) bm = fmaxf(bm, km[i]);
        const float bz = bm == -DV_INF ? 0.0f : bm;
        const float sc = __builtin_amdgcn_exp2f(m - bz);
        sum *= sc;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= sc;
#pragma unroll
        for (int i = 0; i < kTreeBatch; ++i) {
            if (ks[i] == 0.0f) continue;  // no key: the rest of the slot holds nothing
            const float wgt = km[i] == -DV_INF ? 1.0f : __builtin_amdgcn_exp2f(km[i] - bz);
            sum = __builtin_fmaf(wgt, ks[i], sum);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(wgt, x[i][e], v[e]);
        }
        m = bm;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= inv;
    store_run8<DT>(reinterpret_cast<typename Tr<DT>::raw*>(p.out) +
                       (((long long)w * p.Hq + hkv * kGqa + n) * p.S + s) * kHeadDim + d,
                   v);
}

}  // namespace chunk

// Keys and nodes up to which this is the faster way, 8 KV heads of one sequence, us here /
// with the multi-query kernel.  One launch, bf16: 8 nodes on 200 keys 11 / 24; 16 nodes of
// four sequences on 400 keys 23 / 33, of eight (1024 blocks) 43.5 / 46; 64 nodes of four
// sequences on 200 (2048 blocks) 51 / 49.  fp32: 12 / 64, 31 / 92, 56 / 163, 65 / 124.
// Windows, bf16: 8 nodes on 1000 keys 16.6 / 25.6, on 3000 26 / 30; 32 on 1000 30 / 34;
// (more entries, nodes times keys:) 64 on 1000 55 / 41.  fp32: 19 / 56, 35 / 81, 39 / 83,
// 73 / 135; 8 on 8000 84 / 89.
TreePlan tree_plan(int dtype, int F, int W, int S, int Hkv, long long max_keys) {
    using namespace chunk;
    TreePlan t{0, 0};
    if (S > kEntries / 2 || (long long)W * Hkv > (1 << 20) || max_keys > (1 << 24)) return t;
    const long long nodes = (long long)W * Hkv * S;
    const long long view = (long long)kGqa * kHeadDim * (dtype == kF32 ? 4 : 2);  // bytes of a view's queries
    const long long keys = (max_keys + 15ll * F) / 16 * 16 + 16;                  // more than the committed list holds
    const long long path = (S + 15ll) / 16 * 16;
    if (F * view > kSmallQueryBytes) return t;
    if (keys + path <= kEntries && nodes <= (dtype == kF32 ? 4096 : 1024)) return TreePlan{1, (int)keys};
    if (nodes * keys > (dtype == kF32 ? 600 : 288) * 1024ll) return t;
    // Two blocks share a CU and take about as long for entries + 160 (in bf16: 11.7 us for
    // 128 entries, 15.8 for 224, 23 for 416): as many windows as make the rounds of 512
    // blocks shortest, fewer ones where that is even.
    long long best = 0;
    for (long long n = (keys + kEntries - path - 1) / (kEntries - path); n == 1 || n <= (keys + 127) / 128; ++n) {
        const long long window = ((keys + n - 1) / n + 15) / 16 * 16;
        const long long cost = (nodes * n + 511) / 512 * (window + 160);
        if (t.windows == 0 || cost < best) {
            best = cost;
            t = TreePlan{(int)((keys + window - 1) / window), (int)window};
        }
    }
    return t;
}

size_t tree_workspace_bytes(const TreePlan& t, int W, int S, int Hkv) {
    return t.windows > 1 ? (size_t)W * S * Hkv * t.windows * chunk::kSlot * sizeof(float) : 0;
}

namespace {

template <int DT>
hipError_t tree_go(const TreePlan& t, const DecodeParams& p, hipStream_t stream) {
    using namespace chunk;
    const unsigned nodes = (unsigned)(p.W * p.Hkv * p.S);
    if (t.windows == 1) {
        hipLaunchKernelGGL((dv_tree_small<DT, false>), dim3(nodes), dim3(kSmallThreads), 0, stream, p, 1, t.window);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((dv_tree_small<DT, true>), dim3(nodes * t.windows), dim3(kSmallThreads), 0, stream, p,
                       t.windows, t.window);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(dv_tree_join<DT>, dim3(nodes), dim3(256), 0, stream, p, t.windows);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_tree_small(int dtype, const TreePlan& t, const DecodeParams& p, hipStream_t stream) {
    switch (dtype) {
        case kBF16: return tree_go<kBF16>(t, p, stream);
        case kF16: return tree_go<kF16>(t, p, stream);
        case kF32: return tree_go<kF32>(t, p, stream);
        default: return hipErrorInvalidValue;
    }
}

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
