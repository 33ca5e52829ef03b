// Cache-side kernels around the decode path:
//  * dv_kv_append -- rotate the new tokens' keys and write keys and values into
//    their cache rows (the K side of a decode step: attention.py:304 rotates
//    key_states with the model's (cos, sin), attention.py:141-152 appends them to
//    the sequence's own cache).  The same kernel with one (cos, sin) row
//    broadcast over all tokens is merge_caches' constant-offset re-rotation
//    (attention.py:245-251).
//  * dv_view_meta -- per (view, sequence, new token) locations and rotary
//    cos/sin on the device (attention.py:158-186: suffix sums of the segment
//    lengths in each sequence's segment order, then the model's rotary
//    embedding at those positions).
//  * dv_tree_meta -- the same for a step that drafts a token tree per sequence:
//    positions follow a node's depth, and the drafted rows' places.
// All are elementwise and HBM- or launch-bound; one thread per 16-byte run.
#include "dv_common.h"
#include "dv_device.h"

namespace dv {

namespace {

typedef __attribute__((address_space(1))) u32x4 gw_u32x4;

// N elements of X from / to global memory, 16 bytes at a time when the run is
// a multiple of 16 bytes (the launcher checks the alignment).
template <typename X, int N>
__device__ inline void load_run(const X* src, X (&dst)[N]) {
    if constexpr ((sizeof(X) * N) % 16 == 0) {
        constexpr int V = (int)(sizeof(X) * N / 16);
        u32x4 t[V];
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = ld16(reinterpret_cast<const unsigned char*>(src) + 16 * i);
        __builtin_memcpy(dst, t, sizeof(dst));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) dst[i] = src[i];
    }
}

template <typename X, int N>
__device__ inline void store_run(X* dst, const X (&src)[N]) {
    if constexpr ((sizeof(X) * N) % 16 == 0) {
        constexpr int V = (int)(sizeof(X) * N / 16);
        u32x4 t[V];
        __builtin_memcpy(t, src, sizeof(t));
#pragma unroll
        for (int i = 0; i < V; ++i) *(gw_u32x4*)(reinterpret_cast<unsigned char*>(dst) + 16 * i) = t[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) dst[i] = src[i];
    }
}

template <int DT>
__device__ inline float round_to(float f) {
    return Tr<DT>::tof(Tr<DT>::fromf(f));
}

// One rotated element as PyTorch evaluates attention.py:82-88,
// x_rot * cos + rotate_half(x_rot) * sin: each product and the sum are rounded
// to the promoted dtype of (x, cos) -- fp32 if either is fp32, else the 16-bit
// storage type -- and the result to the storage type.  `first`: dims [0, R/2),
// where rotate_half contributes -x[e + R/2].
template <int DT, int CDT>
__device__ inline float rope_elem(float x, float xp, float c, float s, bool first) {
#pragma clang fp contract(off)
    constexpr bool kF32Math = DT == kF32 || CDT == kF32;
    float a = x * c;
    float b = xp * s;
    if constexpr (!kF32Math) {
        a = round_to<DT>(a);
        b = round_to<DT>(b);
    }
    float y = first ? a - b : a + b;
    if constexpr (!kF32Math) y = round_to<DT>(y);
    return y;
}

}  // namespace

// Thread = one run of RUN dims of one (token, KV head) row; consecutive threads
// cover one row, so every warp-wide access is contiguous.  Tokens whose
// position is negative, past the block table row or on an invalid page are not
// written.
template <int DT, int CDT, int RUN>
__global__ __launch_bounds__(256) void dv_kv_append(const AppendParams p, uint32_t nruns, uint32_t runs) {
    using raw = typename Tr<DT>::raw;
    using craw = typename Tr<CDT>::raw;
    // 32-bit index arithmetic: the launcher keeps a launch below 2^31 runs
    const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
    if (idx >= nruns) return;
    const uint32_t hr = idx / runs;
    const int d0 = (int)(idx - hr * runs) * RUN;
    const uint32_t n = hr / (uint32_t)p.Hkv;  // token index w*S + s
    const int h = (int)(hr - n * (uint32_t)p.Hkv);
    const int w = (int)(n / (uint32_t)p.S);
    const int s = (int)(n - (uint32_t)w * (uint32_t)p.S);
    // the token's inputs are loaded first, then the page lookup (positions,
    // then block_tables: two dependent loads) runs while they are in flight
    const int ps = p.pos[n];
    const bool has_k = d0 < p.E, has_v = d0 < p.Ev;
    const bool rot = has_k && d0 < p.R;
    const int half = p.R >> 1;
    const bool first = d0 < half;  // a rotated run lies within one half (R/2 % RUN == 0)
    raw xa[RUN], xb[RUN], vo[RUN];
    craw c[RUN], sn[RUN];
    if (has_k) {
        const raw* x = reinterpret_cast<const raw*>(p.k) + w * p.ks[0] + h * p.ks[1] + s * p.ks[2];
        load_run<raw, RUN>(x + d0, xa);
        if (rot) {
            const long long co = w * p.cs[0] + s * p.cs[1] + d0;
            load_run<raw, RUN>(x + (first ? d0 + half : d0 - half), xb);
            load_run<craw, RUN>(reinterpret_cast<const craw*>(p.cosv) + co, c);
            load_run<craw, RUN>(reinterpret_cast<const craw*>(p.sinv) + co, sn);
        }
    }
    if (has_v)
        load_run<raw, RUN>(reinterpret_cast<const raw*>(p.v) + w * p.vs[0] + h * p.vs[1] + s * p.vs[2] + d0, vo);
    if (ps < 0) return;
    const int lp = ps / p.bs;
    if (lp >= p.maxB) return;
    const int page = p.bt[(long long)w * p.maxB + lp];
    if (has_k && rot) {
#pragma unroll
        for (int e = 0; e < RUN; ++e)
            xa[e] = Tr<DT>::fromf(rope_elem<DT, CDT>(Tr<DT>::tof(xa[e]), Tr<DT>::tof(xb[e]), Tr<CDT>::tof(c[e]),
                                                     Tr<CDT>::tof(sn[e]), first));
    }
    if (page < 0 || page >= p.nblocks) return;
    const long long row = ps - (long long)lp * p.bs;
    if (has_k)
        store_run<raw, RUN>(reinterpret_cast<raw*>(p.kc) + page * p.kcs[0] + row * p.kcs[1] + h * p.kcs[2] + d0, xa);
    if (has_v)
        store_run<raw, RUN>(reinterpret_cast<raw*>(p.vc) + page * p.vcs[0] + row * p.vcs[1] + h * p.vcs[2] + d0, vo);
}

template <int DT, int CDT, int RUN>
hipError_t append_go(const AppendParams& p, hipStream_t stream) {
    const int E = p.E > p.Ev ? p.E : p.Ev;
    const int runs = (E + RUN - 1) / RUN;
    const long long nruns = (long long)p.W * p.S * p.Hkv * runs;
    if (nruns == 0) return hipSuccess;
    if (nruns >= (1ll << 31)) return hipErrorInvalidValue;  // the C ABI rejects such calls first
    const long long blocks = (nruns + 255) / 256;
    hipLaunchKernelGGL((dv_kv_append<DT, CDT, RUN>), dim3((unsigned)blocks), dim3(256), 0, stream, p,
                       (uint32_t)nruns, (uint32_t)runs);
    return hipGetLastError();
}

template <int DT, int CDT>
hipError_t append_dispatch(const AppendParams& p, hipStream_t stream) {
    constexpr int kRun = DT == kF32 ? 4 : 8;
    constexpr int kEs = Tr<DT>::kBytes, kCs = Tr<CDT>::kBytes;
    auto al = [](const void* ptr) { return ((uintptr_t)ptr & 15) == 0; };
    auto st = [](long long stride, int bytes) { return (stride * bytes) % 16 == 0; };
    bool vec = p.E % kRun == 0 && p.Ev % kRun == 0 && (p.R / 2) % kRun == 0;
    vec = vec && al(p.kc) && al(p.vc) && al(p.k) && al(p.v) && al(p.cosv) && al(p.sinv);
    for (int i = 0; i < 3; ++i)
        vec = vec && st(p.kcs[i], kEs) && st(p.vcs[i], kEs) && st(p.ks[i], kEs) && st(p.vs[i], kEs);
    vec = vec && st(p.cs[0], kCs) && st(p.cs[1], kCs);
    if (vec) return append_go<DT, CDT, kRun>(p, stream);
    return append_go<DT, CDT, 1>(p, stream);
}

hipError_t launch_kv_append(int dtype, int rope_dtype, const AppendParams& p, hipStream_t stream) {
    const bool f32rope = rope_dtype == kF32;
    switch (dtype) {
        case kBF16: return f32rope ? append_dispatch<kBF16, kF32>(p, stream) : append_dispatch<kBF16, kBF16>(p, stream);
        case kF16: return f32rope ? append_dispatch<kF16, kF32>(p, stream) : append_dispatch<kF16, kF16>(p, stream);
        case kF32: return append_dispatch<kF32, kF32>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

// Thread = (view f, sequence w, new token s, rotary pair i).  The location of
// view f for sequence w is the total length of w's segments from f's place in
// its segment order to the last one, minus the new tokens, plus s
// (attention.py:167-176 walks the order backwards accumulating lengths that
// already include the new tokens).  cos/sin follow the rotary embedding of
// transformers: angle = fp32(position) * inv_freq[i] (one fp32 product),
// cos/sin of it times the attention scaling, the same value in both halves.
// A view missing from w's order gets location -1 and the identity rotation.
__global__ __launch_bounds__(256) void dv_view_meta(const MetaParams p, long long n, int rh) {
    const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx >= n) return;
    const int i = (int)(idx % rh);
    const long long t = idx / rh;  // (f*W + w)*S + s
    const int s = (int)(t % p.S);
    const long long fw = t / p.S;
    const int w = (int)(fw % p.W);
    const int f = (int)(fw / p.W);
    // the whole row is walked: if f appears more than once, its first place
    // wins, as in the reference, whose backward walk assigns it last.  The row is
    // walked eight segments at a time, their loads issued together (one after the
    // other, a row of five segments was ten dependent round trips: 20 calls on 5 / 8
    // / 16 / 40 segments 64 / 73 / 98 / 182 us, batched 60 / 62 / 75 / 133); rows of
    // up to three one by one (one segment: 47 us, batched 50)
    long long suffix = 0, at = 0;
    bool found = false;
    const int* ord = p.order + (long long)w * p.F;
    if (p.F <= 3) {
        for (int j = p.F - 1; j >= 0; --j) {
            const int g = ord[j];
            if (g >= 0 && g < p.F) suffix += p.fl[g];
            if (g == f) {
                found = true;
                at = suffix;
            }
        }
    } else {
        for (int j0 = p.F - 1; j0 >= 0; j0 -= 8) {
            int g[8], len[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) g[k] = ord[j0 - k > 0 ? j0 - k : 0];
#pragma unroll
            for (int k = 0; k < 8; ++k) len[k] = p.fl[g[k] >= 0 && g[k] < p.F ? g[k] : 0];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (j0 - k < 0) continue;
                if (g[k] >= 0 && g[k] < p.F) suffix += len[k];
                if (g[k] == f) {
                    found = true;
                    at = suffix;
                }
            }
        }
    }
    const int loc = found ? (int)(at - p.S + s) : -1;
    if (i == 0) p.loc[t] = loc;
    if (p.R > 0) {
        float c = 1.0f, sn = 0.0f;
        if (found) {
            const float ang = (float)loc * p.inv_freq[i];
            c = cosf(ang) * p.scaling;
            sn = sinf(ang) * p.scaling;
        }
        if (p.round_dt == kBF16) {
            c = round_to<kBF16>(c);
            sn = round_to<kBF16>(sn);
        } else if (p.round_dt == kF16) {
            c = round_to<kF16>(c);
            sn = round_to<kF16>(sn);
        }
        const long long o = t * p.R;
        p.cosv[o + i] = c;
        p.cosv[o + i + rh] = c;
        p.sinv[o + i] = sn;
        p.sinv[o + i + rh] = sn;
    }
}

hipError_t launch_view_meta(const MetaParams& p, hipStream_t stream) {
    const int rh = p.R > 0 ? p.R / 2 : 1;
    const long long n = (long long)p.F * p.W * p.S * rh;
    if (n == 0) return hipSuccess;
    const long long blocks = (n + 255) / 256;
    hipLaunchKernelGGL(dv_view_meta, dim3((unsigned)blocks), dim3(256), 0, stream, p, n, rh);
    return hipGetLastError();
}

// A step that drafts a tree of S nodes per sequence.  With c(g) the committed tokens
// of view g -- committed[w, g] where given, else fl[g] less the S drafted rows where g is
// some sequence's own (last) view -- and d(s) the depth of node s (0: child of the committed tokens),
//   position[f, w, s] = sum of c + dropped over w's segments from f's place in its order
//                       to the last one, plus d(s),
//   location[f, w, s] = c(f) - 1 (the drafted rows are seen through the tree alone),
//   cos / sin         = cos / sin(fp32(position) * inv_freq[i]) * scaling, as dv_view_meta.
// An absent node (parent neither -1 nor an earlier node, or below such a node) and a
// view missing from the order get location -1 and the identity rotation.
// dropped[w, g] are tokens that were cut from the view: rows count what a cache holds,
// positions what it has seen (the keys that stayed keep their rotation).
//
// Bound by its writes (F W S (4 + 8 R) bytes) and, for small calls, by the launch: 8 nodes
// of one sequence 4.1 us, 32 nodes of 16 sequences over 17 views (8.9 MB) 8.4.
// Block (f, w, tile of kTreeTile nodes): which views are drafted, the order's sum and
// the nodes' depths cost one round of loads each for the whole block and are shared
// in LDS; then thread = RUN rotary pairs of a node, 16-byte stores.
constexpr int kTreeTile = 64;
template <int RUN>
__global__ __launch_bounds__(256) void dv_tree_meta(const TreeMetaParams tp, int tiles) {
    const MetaParams& p = tp.m;
    extern __shared__ int s_meta[];
    int* s_drafted = s_meta;               // [F]: view is some sequence's own
    int* s_par = s_drafted + p.F;          // [S]
    int* s_depth = s_par + p.S;            // [kTreeTile]
    __shared__ int s_place;
    __shared__ long long s_sum;
    const int tid = threadIdx.x;
    const int tile = blockIdx.x % tiles;
    const int fw = blockIdx.x / tiles;
    const int f = fw / p.W, w = fw - (fw / p.W) * p.W;
    const int* ord = p.order + (long long)w * p.F;

    for (int i = tid; i < p.F; i += 256) s_drafted[i] = 0;
    for (int i = tid; i < p.S; i += 256) s_par[i] = tp.parents[(long long)w * p.S + i];
    if (tid == 0) {
        s_place = p.F;
        s_sum = 0;
    }
    __syncthreads();
    for (int v = tid; v < p.W && p.F > 0; v += 256) {
        const int g = p.order[(long long)v * p.F + p.F - 1];
        if (g >= 0 && g < p.F) s_drafted[g] = 1;
    }
    // f's first place in the order (integers: the order of the updates does not matter)
    for (int j = tid; j < p.F; j += 256)
        if (ord[j] == f) atomicMin(&s_place, j);
    __syncthreads();
    auto committed = [&](int g) {
        const long long c = tp.committed ? (long long)tp.committed[(long long)w * p.F + g]
                                         : (long long)p.fl[g] - (s_drafted[g] ? p.S : 0);
        return c > 0 ? c : 0ll;
    };
    const int place = s_place;
    long long mine = 0;
    for (int j = tid; j < p.F; j += 256) {
        const int g = ord[j];
        if (j >= place && g >= 0 && g < p.F)
            mine += committed(g) + (tp.dropped ? (long long)tp.dropped[(long long)w * p.F + g] : 0ll);
    }
    if (mine) atomicAdd(reinterpret_cast<unsigned long long*>(&s_sum), (unsigned long long)mine);
    const int s0 = tile * kTreeTile;
    const int ns = p.F == 0 ? 0 : p.S - s0 < kTreeTile ? p.S - s0 : kTreeTile;
    if (tid < ns) {
        // every step goes to an earlier node, so the walk ends
        int j = s0 + tid, dep = 0;
        for (;;) {
            const int up = s_par[j];
            if (up == -1) break;
            if (up < -1 || up >= j) {
                dep = -1;
                break;
            }
            j = up;
            ++dep;
        }
        s_depth[tid] = dep;
    }
    __syncthreads();
    const bool found = place < p.F;
    if (f == 0 && tile == 0 && tid == 0) {
        // the drafted rows: w's own view, and the stream row of node 0
        const int own = p.F > 0 ? ord[p.F - 1] : -1;
        const bool ok = own >= 0 && own < p.F;
        long long row = 0;
        for (int g = 0; ok && g < own; ++g) row += p.fl[g];
        tp.tree_views[w] = ok ? own : -1;
        tp.tree_rows[w] = ok ? (int)(row + committed(own)) : 0;
    }
    const long long t0 = ((long long)f * p.W + w) * p.S + s0;
    if (tid < ns) p.loc[t0 + tid] = found && s_depth[tid] >= 0 ? (int)committed(f) - 1 : -1;
    const int rh = p.R >> 1;
    const int runs = rh / RUN;
    const long long base = s_sum;
    for (int k = tid; k < ns * runs; k += 256) {
        const int t = k / runs;
        const int i = (k - t * runs) * RUN;
        const int dep = s_depth[t];
        float c[RUN], sn[RUN];
#pragma unroll
        for (int e = 0; e < RUN; ++e) {
            c[e] = 1.0f;
            sn[e] = 0.0f;
            if (found && dep >= 0) {
                const float ang = (float)(int)(base + dep) * p.inv_freq[i + e];
                sincosf(ang, &sn[e], &c[e]);
                c[e] *= p.scaling;
                sn[e] *= p.scaling;
            }
            if (p.round_dt == kBF16) {
                c[e] = round_to<kBF16>(c[e]);
                sn[e] = round_to<kBF16>(sn[e]);
            } else if (p.round_dt == kF16) {
                c[e] = round_to<kF16>(c[e]);
                sn[e] = round_to<kF16>(sn[e]);
            }
        }
        const long long o = (t0 + t) * p.R + i;
        store_run<float, RUN>(p.cosv + o, c);
        store_run<float, RUN>(p.cosv + o + rh, c);
        store_run<float, RUN>(p.sinv + o, sn);
        store_run<float, RUN>(p.sinv + o + rh, sn);
    }
}

hipError_t launch_tree_meta(const TreeMetaParams& p, hipStream_t stream) {
    // (without views or nodes a block per sequence still writes the drafted rows' place)
    const int tiles = p.m.S > 0 ? (p.m.S + kTreeTile - 1) / kTreeTile : 1;
    const long long blocks = (long long)(p.m.F > 0 ? p.m.F : 1) * p.m.W * tiles;
    if (blocks == 0) return hipSuccess;
    if (blocks >= (1ll << 24)) return hipErrorInvalidValue;  // the C ABI rejects such calls first
    const size_t lds = (size_t)(p.m.F + p.m.S + kTreeTile) * sizeof(int);
    auto al = [](const void* ptr) { return ((uintptr_t)ptr & 15) == 0; };
    const bool vec = (p.m.R / 2) % 4 == 0 && al(p.m.cosv) && al(p.m.sinv);
    if (vec) hipLaunchKernelGGL(dv_tree_meta<4>, dim3((unsigned)blocks), dim3(256), lds, stream, p, tiles);
    else hipLaunchKernelGGL(dv_tree_meta<1>, dim3((unsigned)blocks), dim3(256), lds, stream, p, tiles);
    return hipGetLastError();
}

}  // namespace dv
