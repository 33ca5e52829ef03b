// C ABI of libdvattn_amd.so (declared in include/dvattn_amd.h).  Validates the
// arguments the reference's torch binding validated (src/binding.cu:41-296),
// rejects the shapes/dtypes it silently ignored, and launches the gfx950
// kernels on the caller's stream.  No exception crosses this boundary.
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <atomic>
#include <initializer_list>
#include <mutex>
#include <vector>

#include "../../include/dvattn_amd.h"
#include "dv_common.h"
#include "dv_stream.h"

namespace {

thread_local char g_err[512] = "";

dvattn_status fail(dvattn_status st, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return st;
}

dvattn_status ok() {
    g_err[0] = '\0';
    return DVATTN_OK;
}

dvattn_status hip_fail(hipError_t e, const char* what) {
    return fail(DVATTN_ERR_HIP, "%s: %s (%s)", what, hipGetErrorString(e), dv::last_hip_site());
}

bool valid_dtype(int dt) { return dt == DVATTN_F32 || dt == DVATTN_F16 || dt == DVATTN_BF16; }

int log2_exact(int v) {
    if (v <= 0 || (v & (v - 1))) return -1;
    int s = 0;
    while ((1 << s) < v) ++s;
    return s;
}

int current_device(int device) {
    if (device >= 0) return device;
    int d = 0;
    if (hipGetDevice(&d) != hipSuccess) d = 0;
    return d;
}

// Checks shared by the attention entry points: GQA 16, E == Ev == 128
// (paged_kernel_v21.cuh:413, varlen:410, kernel_v21.cuh:400).
dvattn_status check_heads(const dvattn_shape* s) {
    if (s->Hkv <= 0) return fail(DVATTN_ERR_INVALID, "Hkv must be positive (got %d)", s->Hkv);
    if (s->Hq != 16 * s->Hkv)
        return fail(DVATTN_ERR_UNSUPPORTED, "only GQA 16 is implemented (Hq=%d, Hkv=%d)", s->Hq, s->Hkv);
    if (s->E != 128 || s->Ev != 128)
        return fail(DVATTN_ERR_UNSUPPORTED, "only head dims E == Ev == 128 are implemented (E=%d, Ev=%d)", s->E,
                    s->Ev);
    return DVATTN_OK;
}

dvattn_status check_rotary(int R, int E) {
    if (R < 0 || R > E || (R & 1))
        return fail(DVATTN_ERR_UNSUPPORTED, "rotary_dim must be even and in [0, E] (got %d, E=%d)", R, E);
    return DVATTN_OK;
}

dvattn_status check_pages(const dvattn_shape* s) {
    if (s->block_size <= 0) return fail(DVATTN_ERR_INVALID, "block_size must be positive (got %d)", s->block_size);
    if (s->max_blocks_per_seq < 0 || s->num_blocks < 0)
        return fail(DVATTN_ERR_INVALID, "max_blocks_per_seq / num_blocks must be >= 0");
    // the kernels index cache rows (block, slot, KV head) with 32-bit integers
    if ((long long)s->num_blocks * s->block_size * (s->Hkv > 0 ? s->Hkv : 1) >= (1ll << 32))
        return fail(DVATTN_ERR_UNSUPPORTED, "K/V cache of %lld rows exceeds 2^32 rows",
                    (long long)s->num_blocks * s->block_size * s->Hkv);
    return DVATTN_OK;
}

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// The attention kernels move queries, outputs, cache and view rows and partial
// results as 16-byte vectors and LDS DMAs, update 8-byte merge flags in the
// workspace atomically and read the int32 / fp32 arrays as 4-byte words (the
// reference's kernels load 16-byte vectors too, paged_kernel_v21.cuh:58-62,
// unchecked).  A pointer off that alignment is refused here instead of reaching
// a kernel.  Null pointers pass: the null checks are separate.
struct Aligned {
    const void* ptr;
    const char* name;
    unsigned align;
};

unsigned elem_bytes(int dtype) { return dtype == DVATTN_F32 ? 4u : 2u; }

dvattn_status check_aligned(std::initializer_list<Aligned> ptrs) {
    for (const Aligned& a : ptrs)
        if ((uintptr_t)a.ptr & (a.align - 1))
            return fail(DVATTN_ERR_INVALID, "%s must be %u-byte aligned (got %p)", a.name, a.align, a.ptr);
    return DVATTN_OK;
}

// ---- static scratch of dvattn_paged_sdpa_noalloc ------------------------------
// Device memory for the partial results and merge directory of the paged entry
// point, for callers that cannot allocate.  Each GPU the library runs on holds
// its own copy of the array until the process ends.  In host code `scratch`
// names a host-side stand-in, never the device memory: the device address is
// taken once per device with hipGetSymbolAddress and only that address is used.
constexpr size_t kScratchBytes = (size_t)DVATTN_NOALLOC_SCRATCH_BYTES;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];

constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;
void* g_scratch_dev[kMaxDevices] = {};

// Device address of `scratch` on the current device (looked up on the first
// call on that device, with the device current).
dvattn_status scratch_address(void** out) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return fail(DVATTN_ERR_HIP, "hipGetDevice: %s", hipGetErrorString(e));
    if (dev < 0 || dev >= kMaxDevices) return fail(DVATTN_ERR_UNSUPPORTED, "device %d beyond %d", dev, kMaxDevices);
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    if (!g_scratch_dev[dev]) {
        void* ptr = nullptr;
        e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
        if (e != hipSuccess || !ptr)
            return fail(DVATTN_ERR_HIP, "hipGetSymbolAddress(scratch) on device %d: %s", dev, hipGetErrorString(e));
        g_scratch_dev[dev] = ptr;
    }
    *out = g_scratch_dev[dev];
    return DVATTN_OK;
}

size_t contig_table_bytes(int F) {
    return F > dv::kMaxFragArgs ? align256((size_t)F * sizeof(dv::FragDesc)) : 0;
}

}  // namespace

namespace dv {

namespace {

// Option values; kUnset until first read (then from the environment).
constexpr int kUnset = -1;
std::atomic<int> g_options[kOptCount] = {kUnset};

int option_from_env(Option) {
    const char* e = getenv("DVATTN_SMALL_PATH");
    if (!e) return kSmallAuto;
    if (e[0] == '0') return kSmallOff;
    if (strcmp(e, "require") == 0) return kSmallRequire;
    if (strcmp(e, "force") == 0) return kSmallForce;
    return kSmallAuto;
}

}  // namespace

int option(Option o) {
    int v = g_options[o].load(std::memory_order_relaxed);
    if (v == kUnset) {
        int expected = kUnset;
        const int init = option_from_env(o);
        g_options[o].compare_exchange_strong(expected, init, std::memory_order_relaxed);
        v = g_options[o].load(std::memory_order_relaxed);
    }
    return v;
}

void set_option(Option o, int value) { g_options[o].store(value, std::memory_order_relaxed); }

// splitmix64 of a process-wide call counter, 48 bits, nonzero
unsigned long long next_call_tag() {
    static std::atomic<unsigned long long> calls{0x5eed5eedull};
    unsigned long long z = calls.fetch_add(0x9e3779b97f4a7c15ull, std::memory_order_relaxed);
    z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
    z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
    z ^= z >> 31;
    z &= (1ull << 48) - 1ull;
    return z ? z : 1ull;
}

}  // namespace dv

extern "C" {

const char* dvattn_last_error(void) { return g_err; }

dvattn_status dvattn_set_option(const char* name, int value) {
    if (!name) return fail(DVATTN_ERR_INVALID, "dvattn_set_option: null name");
    if (strcmp(name, "small_path") == 0) {
        if (value < dv::kSmallOff || value > dv::kSmallForce)
            return fail(DVATTN_ERR_INVALID, "small_path: 0 (off), 1 (auto), 2 (require) or 3 (force), not %d", value);
        dv::set_option(dv::kOptSmallPath, value);
        return ok();
    }
    return fail(DVATTN_ERR_INVALID, "unknown option \"%s\" (small_path)", name);
}

int dvattn_get_option(const char* name) {
    if (!name) return -1;
    if (strcmp(name, "small_path") == 0) return dv::option(dv::kOptSmallPath);
    return -1;
}

int dvattn_abi_version(void) { return DVATTN_ABI_VERSION; }

// ---------------------------------------------------------------------------
size_t dvattn_paged_sdpa_workspace_size(int dtype, const dvattn_shape* s, int device) {
    if (!s || !valid_dtype(dtype)) return 0;
    if (dv::use_chunk(dtype, s->S)) return dv::chunk_workspace_bytes(s->W, s->S, s->Hkv, current_device(device));
    return dv::decode_workspace_bytes(s->W * s->S, s->Hkv, current_device(device), dtype);
}

dvattn_status dvattn_paged_sdpa(int dtype, void* out, float scale, const int* locations, const void* queries,
                                const float* cosines, const float* sines, const int* fragment_lengths,
                                const void* k_cache, const void* v_cache, const int* block_tables,
                                const dvattn_shape* s, void* workspace, size_t workspace_bytes, void* stream) {
    if (!s) return fail(DVATTN_ERR_INVALID, "shape is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (s->F < 0 || s->W < 0 || s->S < 0) return fail(DVATTN_ERR_INVALID, "negative F/W/S");
    if ((long long)s->W * s->S == 0 || s->Hkv == 0) return ok();  // paged_kernel_v21.cuh:385-386
    dvattn_status st;
    if ((st = check_heads(s)) != DVATTN_OK) return st;
    if ((st = check_rotary(s->rotary_dim, s->E)) != DVATTN_OK) return st;
    if ((st = check_pages(s)) != DVATTN_OK) return st;
    if (!out || !queries) return fail(DVATTN_ERR_INVALID, "null output or query pointer");
    if (s->F > 0 && (!locations || !fragment_lengths || ((!cosines || !sines) && s->rotary_dim > 0)))
        return fail(DVATTN_ERR_INVALID, "null locations / fragment_lengths / cos / sin pointer");
    if (s->num_blocks > 0 && (!k_cache || !v_cache)) return fail(DVATTN_ERR_INVALID, "null k/v cache pointer");
    if (s->max_blocks_per_seq > 0 && !block_tables) return fail(DVATTN_ERR_INVALID, "null block_tables pointer");
    if ((st = check_aligned({{out, "out", 16}, {queries, "queries", 16}, {k_cache, "k_cache", 16},
                             {v_cache, "v_cache", 16}, {workspace, "workspace", 16}, {locations, "locations", 4},
                             {fragment_lengths, "fragment_lengths", 4}, {cosines, "cosines", 4},
                             {sines, "sines", 4}, {block_tables, "block_tables", 4}})) != DVATTN_OK)
        return st;
    const size_t need = dvattn_paged_sdpa_workspace_size(dtype, s, -1);
    if (workspace_bytes < need || (need && !workspace))
        return fail(DVATTN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);

    dv::DecodeParams p;
    memset(&p, 0, sizeof(p));
    p.out = out;
    p.loc = locations;
    p.q = queries;
    p.cosv = cosines;
    p.sinv = sines;
    p.fl = fragment_lengths;
    p.kc = k_cache;
    p.vc = v_cache;
    p.bt = block_tables;
    p.l2scale = scale * 1.4426950408889634f;  // scale / ln 2 (paged_kernel_v21.cuh:47)
    p.F = s->F;
    p.W = s->W;
    p.S = s->S;
    p.Hq = s->Hq;
    p.Hkv = s->Hkv;
    p.R = s->rotary_dim;
    p.bs = s->block_size;
    p.bs_shift = log2_exact(s->block_size);
    p.maxB = s->max_blocks_per_seq;
    p.nblocks = s->num_blocks;
    p.min_keys = dv::kDecodeMinKeys;
    const long long max_keys = (long long)s->max_blocks_per_seq * s->block_size;
    hipError_t e;
    if (dv::use_chunk(dtype, s->S)) {
        p.min_keys = 256;
        e = dv::launch_chunk(dtype, dv::kQRotFull, dv::kKvPaged, p, max_keys, workspace, workspace_bytes,
                             (hipStream_t)stream);
    } else {
        e = dv::launch_decode(dtype, dv::kQRotFull, dv::kKvPaged, dv::kRowWS, p, s->W * s->S, max_keys, workspace,
                              workspace_bytes, (hipStream_t)stream);
    }
    if (e != hipSuccess) return hip_fail(e, "dvattn_paged_sdpa launch");
    return ok();
}

dvattn_status dvattn_paged_sdpa_noalloc(int dtype, void* out, float scale, const int* locations,
                                        const void* queries, const float* cosines, const float* sines,
                                        const int* fragment_lengths, const void* k_cache, const void* v_cache,
                                        const int* block_tables, const dvattn_shape* s, void* stream) {
    if (!s) return fail(DVATTN_ERR_INVALID, "shape is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    const size_t need = dvattn_paged_sdpa_workspace_size(dtype, s, -1);
    if (need > kScratchBytes)
        return fail(DVATTN_ERR_WORKSPACE,
                    "dvattn_paged_sdpa_noalloc: this shape needs %zu bytes of scratch, the static scratch "
                    "holds %zu (use dvattn_paged_sdpa with a workspace)",
                    need, kScratchBytes);
    void* ws = nullptr;
    const dvattn_status st = scratch_address(&ws);
    if (st != DVATTN_OK) return st;
    // nothing in the scratch has to start at zero: every call's kernels write the
    // partial slots and the merge directory before reading them
    return dvattn_paged_sdpa(dtype, out, scale, locations, queries, cosines, sines, fragment_lengths, k_cache,
                             v_cache, block_tables, s, ws, kScratchBytes, stream);
}

// ---------------------------------------------------------------------------
size_t dvattn_varlen_paged_sdpa_workspace_size(int dtype, const dvattn_shape* s, int device) {
    if (!s || !valid_dtype(dtype)) return 0;
    if (dv::use_varlen_chunk(dtype, s->total_q_tokens, s->W))
        return dv::varlen_chunk_workspace_bytes(s->total_q_tokens, s->W, s->Hkv, current_device(device));
    return dv::decode_workspace_bytes(s->total_q_tokens, s->Hkv, current_device(device), dtype);
}

dvattn_status dvattn_varlen_paged_sdpa(int dtype, void* out, float scale, const int* locations,
                                       const void* queries, const float* cosines, const float* sines,
                                       const int* fragment_lengths, const void* k_cache, const void* v_cache,
                                       const int* block_tables, const int* cu_seqlens_q, const int* cu_seqlens_k,
                                       const dvattn_shape* s, void* workspace, size_t workspace_bytes,
                                       void* stream) {
    (void)cu_seqlens_k;  // passed but never read by the reference (binding.cu:279,290)
    if (!s) return fail(DVATTN_ERR_INVALID, "shape is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (s->F < 0 || s->W < 0 || s->total_q_tokens < 0) return fail(DVATTN_ERR_INVALID, "negative F/W/T");
    if (s->total_q_tokens == 0 || s->Hkv == 0) return ok();  // varlen_paged_kernel_v21.cuh:382-383
    dvattn_status st;
    if ((st = check_heads(s)) != DVATTN_OK) return st;
    if ((st = check_rotary(s->rotary_dim, s->E)) != DVATTN_OK) return st;
    if ((st = check_pages(s)) != DVATTN_OK) return st;
    if (!out || !queries) return fail(DVATTN_ERR_INVALID, "null output or query pointer");
    if (s->W > 0 && !cu_seqlens_q) return fail(DVATTN_ERR_INVALID, "null cu_seqlens_q pointer");
    if (s->F > 0 && (!locations || !fragment_lengths || ((!cosines || !sines) && s->rotary_dim > 0)))
        return fail(DVATTN_ERR_INVALID, "null locations / fragment_lengths / cos / sin pointer");
    if (s->num_blocks > 0 && (!k_cache || !v_cache)) return fail(DVATTN_ERR_INVALID, "null k/v cache pointer");
    if (s->max_blocks_per_seq > 0 && !block_tables) return fail(DVATTN_ERR_INVALID, "null block_tables pointer");
    if ((st = check_aligned({{out, "out", 16}, {queries, "queries", 16}, {k_cache, "k_cache", 16},
                             {v_cache, "v_cache", 16}, {workspace, "workspace", 16}, {locations, "locations", 4},
                             {fragment_lengths, "fragment_lengths", 4}, {cosines, "cosines", 4},
                             {sines, "sines", 4}, {block_tables, "block_tables", 4},
                             {cu_seqlens_q, "cu_seqlens_q", 4}})) != DVATTN_OK)
        return st;
    const size_t need = dvattn_varlen_paged_sdpa_workspace_size(dtype, s, -1);
    if (workspace_bytes < need || (need && !workspace))
        return fail(DVATTN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);

    dv::DecodeParams p;
    memset(&p, 0, sizeof(p));
    p.out = out;
    p.loc = locations;
    p.q = queries;
    p.cosv = cosines;
    p.sinv = sines;
    p.fl = fragment_lengths;
    p.kc = k_cache;
    p.vc = v_cache;
    p.bt = block_tables;
    p.cu_q = cu_seqlens_q;
    p.l2scale = scale * 1.4426950408889634f;
    p.F = s->F;
    p.W = s->W;
    p.S = 1;
    p.T = s->total_q_tokens;
    p.Hq = s->Hq;
    p.Hkv = s->Hkv;
    p.R = s->rotary_dim;
    p.bs = s->block_size;
    p.bs_shift = log2_exact(s->block_size);
    p.maxB = s->max_blocks_per_seq;
    p.nblocks = s->num_blocks;
    p.min_keys = dv::kDecodeMinKeys;
    const long long max_keys = (long long)s->max_blocks_per_seq * s->block_size;
    hipError_t e;
    if (dv::use_varlen_chunk(dtype, s->total_q_tokens, s->W)) {
        // two or more packed tokens per sequence on average: each sequence's
        // tokens share one K/V stream (the reference re-reads K/V per token,
        // varlen_paged_kernel_v21.cuh:388)
        p.min_keys = 256;
        e = dv::launch_varlen_chunk(dtype, p, max_keys, workspace, workspace_bytes, (hipStream_t)stream);
    } else {
        e = dv::launch_decode(dtype, dv::kQRotHalf, dv::kKvPaged, dv::kRowVarlen, p, s->total_q_tokens, max_keys,
                              workspace, workspace_bytes, (hipStream_t)stream);
    }
    if (e != hipSuccess) return hip_fail(e, "dvattn_varlen_paged_sdpa launch");
    return ok();
}

// ---------------------------------------------------------------------------
size_t dvattn_sdpa_workspace_size(int dtype, const dvattn_shape* s, int device) {
    if (!s || !valid_dtype(dtype)) return 0;
    if (dv::use_chunk(dtype, s->S))
        return dv::chunk_workspace_bytes(s->W, s->S, s->Hkv, current_device(device)) + contig_table_bytes(s->F);
    return dv::decode_workspace_bytes(s->W * s->S, s->Hkv, current_device(device), dtype) +
           contig_table_bytes(s->F);
}

}  // extern "C"

namespace {

// dvattn_sdpa's argument checks (binding.cu:79-149, plus the shapes the
// reference ignored) and its launch parameters: p, the view table and the
// longest row's key count.  `empty`: nothing to compute.
dvattn_status sdpa_setup(int dtype, void* out, float scale, const int* locations, const void* rotated_queries,
                         const int* fragment_lengths, const void* const* key_fragments,
                         const void* const* value_fragments, const int* fragment_tokens, const int* fragment_batch,
                         const dvattn_shape* s, void* workspace, size_t workspace_bytes, dv::DecodeParams& p,
                         std::vector<dv::FragDesc>& tab, long long& max_keys, bool& empty) {
    empty = true;
    if (!s) return fail(DVATTN_ERR_INVALID, "shape is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (s->F < 0 || s->W < 0 || s->S < 0) return fail(DVATTN_ERR_INVALID, "negative F/W/S");
    if ((long long)s->W * s->S == 0 || s->Hkv == 0) return DVATTN_OK;
    dvattn_status st;
    if ((st = check_heads(s)) != DVATTN_OK) return st;
    if (!out || !rotated_queries) return fail(DVATTN_ERR_INVALID, "null output or query pointer");
    if (s->F > 0 && (!locations || !fragment_lengths || !key_fragments || !value_fragments || !fragment_tokens ||
                     !fragment_batch))
        return fail(DVATTN_ERR_INVALID, "null locations / fragment_lengths / fragment arrays");
    if ((st = check_aligned({{out, "out", 16}, {rotated_queries, "rotated_queries", 16},
                             {workspace, "workspace", 16}, {locations, "locations", 4},
                             {fragment_lengths, "fragment_lengths", 4}})) != DVATTN_OK)
        return st;
    const size_t need = dvattn_sdpa_workspace_size(dtype, s, -1);
    if (workspace_bytes < need || (need && !workspace))
        return fail(DVATTN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);

    memset(&p, 0, sizeof(p));
    tab.assign((size_t)s->F, dv::FragDesc{});
    max_keys = 0;
    for (int f = 0; f < s->F; ++f) {
        const int L = fragment_tokens[f];
        const int B = fragment_batch[f];
        if (L < 0) return fail(DVATTN_ERR_INVALID, "fragment %d: negative token count", f);
        if (B != 1 && B != s->W)
            return fail(DVATTN_ERR_INVALID, "fragment %d: batch %d is neither 1 nor W=%d", f, B, s->W);
        if (L > 0 && (!key_fragments[f] || !value_fragments[f]))
            return fail(DVATTN_ERR_INVALID, "fragment %d: null pointer", f);
        if ((((uintptr_t)key_fragments[f]) | ((uintptr_t)value_fragments[f])) & 15)
            return fail(DVATTN_ERR_INVALID, "fragment %d: pointers must be 16-byte aligned", f);
        dv::FragDesc& d = tab[(size_t)f];
        d.k = key_fragments[f];
        d.v = value_fragments[f];
        d.L = L;
        d.bstride = B == 1 ? 0 : (long long)s->Hkv * L * 128;
        d.pad = 0;
        max_keys += L;
        if (f < dv::kMaxFragArgs) p.frags[f] = d;
    }
    p.out = out;
    p.loc = locations;
    p.q = rotated_queries;
    p.fl = fragment_lengths;
    p.l2scale = scale * 1.4426950408889634f;
    p.F = s->F;
    p.W = s->W;
    p.S = s->S;
    p.Hq = s->Hq;
    p.Hkv = s->Hkv;
    p.R = 0;
    p.bs = 1;
    p.bs_shift = 0;
    p.min_keys = dv::kDecodeMinKeys;
    empty = false;
    return DVATTN_OK;
}

// View descriptors written into the device view table by a kernel whose
// arguments carry them: the values travel with the launch (a captured graph
// keeps its own copy), so no host buffer has to outlive the call, as a
// host-to-device copy from the caller's memory would in a captured graph.
constexpr int kFragFillBatch = 64;  // descriptors per launch: 2 KiB of kernel arguments
struct FragFill {
    dv::FragDesc d[kFragFillBatch];
    int first, n;
};

__global__ __launch_bounds__(kFragFillBatch) void dv_frag_fill(dv::FragDesc* dst, const FragFill b) {
    const int i = threadIdx.x;
    if (i < b.n) dst[b.first + i] = b.d[i];
}

// The general contiguous-view launch: view table (F > kMaxFragArgs) to the
// workspace, then the decode or chunk kernel on already-rotated queries.
dvattn_status sdpa_launch(int dtype, dv::DecodeParams& p, const std::vector<dv::FragDesc>& tab, long long max_keys,
                          void* workspace, size_t workspace_bytes, hipStream_t stream) {
    void* ws = workspace;
    size_t ws_left = workspace_bytes;
    const size_t tab_bytes = contig_table_bytes(p.F);
    if (tab_bytes) {
        dv::FragDesc* dst = reinterpret_cast<dv::FragDesc*>(workspace);
        for (int first = 0; first < p.F; first += kFragFillBatch) {
            FragFill b;
            memset(&b, 0, sizeof(b));
            b.first = first;
            b.n = p.F - first < kFragFillBatch ? p.F - first : kFragFillBatch;
            for (int i = 0; i < b.n; ++i) b.d[i] = tab[(size_t)(first + i)];
            hipLaunchKernelGGL(dv_frag_fill, dim3(1), dim3(kFragFillBatch), 0, stream, dst, b);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return hip_fail(e, "dvattn_sdpa view table");
        }
        p.frag_tab = dst;
        ws = reinterpret_cast<unsigned char*>(workspace) + tab_bytes;
        ws_left -= tab_bytes;
    }
    hipError_t e;
    if (dv::use_chunk(dtype, p.S)) {
        p.min_keys = 256;
        e = dv::launch_chunk(dtype, dv::kQPre, dv::kKvContig, p, max_keys, ws, ws_left, stream);
    } else {
        e = dv::launch_decode(dtype, dv::kQPre, dv::kKvContig, dv::kRowWS, p, p.W * p.S, max_keys, ws, ws_left,
                              stream);
    }
    if (e != hipSuccess) return hip_fail(e, "dvattn_sdpa launch");
    return ok();
}

// Whether the single-launch path takes a validated contiguous-view call (fp32,
// fp16 or bf16): at most kMaxFragArgs views of at most kSmallMaxChunks chunks
// together, and its partials within the documented workspace size of the shape
// (so the choice depends on the shape and the fragment lengths only); rotating
// calls (dvattn_fused) also need rotary_dim % 8 == 0.  Returns the chunk count,
// or -1 for the general path.
// Option small_path (dvattn_set_option; DVATTN_SMALL_PATH at first use): off
// turns the path off; require makes a call it cannot take fail with
// DVATTN_ERR_UNSUPPORTED (*refused); force takes it past the workgroup limit
// below as well (for measuring that limit: bench.py --small-crossover).
int small_path_chunks(int dtype, const dvattn_shape* s, const int* fragment_tokens, bool rotating, bool* refused) {
    *refused = false;
    const int mode = dv::option(dv::kOptSmallPath);
    if (mode == dv::kSmallOff) return -1;
    const bool require = mode == dv::kSmallRequire;
    const bool force = mode == dv::kSmallForce;
    int chunks = -1;
    if (s->F >= 1 && s->F <= dv::kMaxFragArgs && (!rotating || s->rotary_dim % 8 == 0)) {
        chunks = dv::small_chunks(s->F, fragment_tokens);
        const long long items = (long long)s->W * s->S * s->Hkv;
        // Only a single-chunk call (one view of at most kSmallChunk keys) needs
        // no merge.  Any other call (several chunks, from one long view or
        // from several views) merges its chunks in the launch, and every
        // workgroup pays the merge protocol's fences, whose cost grows with the
        // number of workgroups: past items x chunks = small_max_merged() the
        // general path (rotation, decode and merge launches) is faster
        // (measured crossover about 190 workgroups for fp32, about 110 for
        // 16-bit types, whose general path is faster).
        if (chunks > 1 && items * chunks > dv::small_max_merged(dtype) && !force) chunks = -1;
        if (chunks >= 1 && dv::small_workspace_bytes(items, chunks) > dvattn_sdpa_workspace_size(dtype, s, -1))
            chunks = -1;
    }
    if (chunks < 1 && require) {
        fail(DVATTN_ERR_UNSUPPORTED,
             "DVATTN_SMALL_PATH=require: the single-launch path takes calls of 1-%d views with at most %d "
             "chunks of %d keys per row, and at most %d (fp32) or %d (16-bit) workgroups in all when a row "
             "has more than one chunk (one per row, KV head and chunk); rotary_dim %% 8 == 0 when it rotates",
             dv::kMaxFragArgs, dv::kSmallMaxChunks, dv::kSmallChunk, dv::small_max_merged(DVATTN_F32),
             dv::small_max_merged(DVATTN_BF16));
        *refused = true;
    }
    return chunks;
}

dvattn_status small_launch(int dtype, int qmode, const dv::DecodeParams& p, int chunks, const int* fragment_tokens,
                           void* rq_out, void* workspace, hipStream_t stream) {
    dv::SmallParams sp;
    memset(&sp, 0, sizeof(sp));
    sp.d = p;
    sp.rq = rq_out;
    sp.chunks = chunks;
    int c = 0;
    for (int f = 0; f < p.F; ++f) {
        sp.first_chunk[f] = c;
        const int L = fragment_tokens[f];
        c += L > 0 ? (L + dv::kSmallChunk - 1) / dv::kSmallChunk : 1;
    }
    sp.first_chunk[p.F] = c;
    const hipError_t e = dv::launch_small(dtype, qmode, sp, workspace, stream);
    if (e != hipSuccess) return hip_fail(e, "single-launch attention");
    return ok();
}

// dvattn_rope's checks (rope.cuh:54-65) into p; `empty`: nothing to rotate.
dvattn_status rope_setup(int dtype, void* out, const void* queries, const float* cosines, const float* sines,
                         const dvattn_shape* s, dv::RopeParams& p, bool& empty) {
    empty = true;
    if (!s) return fail(DVATTN_ERR_INVALID, "shape is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (s->F < 0 || s->W < 0 || s->Hq < 0 || s->S < 0 || s->E < 0)
        return fail(DVATTN_ERR_INVALID, "negative size");
    dvattn_status st;
    if ((st = check_rotary(s->rotary_dim, s->E)) != DVATTN_OK) return st;
    if ((long long)s->F * s->W * s->Hq * s->S * s->E == 0) return DVATTN_OK;  // rope.cuh:58-60
    if (!out || !queries || (s->rotary_dim > 0 && (!cosines || !sines)))
        return fail(DVATTN_ERR_INVALID, "null pointer");
    if ((st = check_aligned({{out, "out", elem_bytes(dtype)}, {queries, "queries", elem_bytes(dtype)},
                             {cosines, "cosines", 4}, {sines, "sines", 4}})) != DVATTN_OK)
        return st;
    memset(&p, 0, sizeof(p));
    p.out = out;
    p.q = queries;
    p.cosv = cosines;
    p.sinv = sines;
    p.F = s->F;
    p.W = s->W;
    p.Hq = s->Hq;
    p.S = s->S;
    p.E = s->E;
    p.R = s->rotary_dim;
    p.half_width = 0;
    empty = false;
    return DVATTN_OK;
}

}  // namespace

extern "C" {

dvattn_status dvattn_sdpa(int dtype, void* out, float scale, const int* locations, const void* rotated_queries,
                          const int* fragment_lengths, const void* const* key_fragments,
                          const void* const* value_fragments, const int* fragment_tokens,
                          const int* fragment_batch, const dvattn_shape* s, void* workspace,
                          size_t workspace_bytes, void* stream) {
    dv::DecodeParams p;
    std::vector<dv::FragDesc> tab;
    long long max_keys = 0;
    bool empty = true;
    dvattn_status st = sdpa_setup(dtype, out, scale, locations, rotated_queries, fragment_lengths, key_fragments,
                                  value_fragments, fragment_tokens, fragment_batch, s, workspace, workspace_bytes, p,
                                  tab, max_keys, empty);
    if (st != DVATTN_OK) return st;
    if (empty) return ok();
    bool refused = false;
    const int chunks = small_path_chunks(dtype, s, fragment_tokens, false, &refused);
    if (refused) return DVATTN_ERR_UNSUPPORTED;
    if (chunks > 0)
        return small_launch(dtype, dv::kQPre, p, chunks, fragment_tokens, nullptr, workspace, (hipStream_t)stream);
    return sdpa_launch(dtype, p, tab, max_keys, workspace, workspace_bytes, (hipStream_t)stream);
}

// binding.cu:356-372: rotate the queries into rotated_queries, attend on them.
// Both steps' arguments are checked before anything runs; short views take the
// single launch that rotates, attends and merges.
dvattn_status dvattn_fused(int dtype, void* out, void* rotated_queries, float scale, const int* locations,
                           const void* queries, const int* fragment_lengths, const void* const* key_fragments,
                           const void* const* value_fragments, const int* fragment_tokens,
                           const int* fragment_batch, const float* cosines, const float* sines,
                           const dvattn_shape* s, void* workspace, size_t workspace_bytes, void* stream) {
    dv::RopeParams rp;
    bool no_rope = true;
    dvattn_status st = rope_setup(dtype, rotated_queries, queries, cosines, sines, s, rp, no_rope);
    if (st != DVATTN_OK) return st;
    dv::DecodeParams p;
    std::vector<dv::FragDesc> tab;
    long long max_keys = 0;
    bool empty = true;
    st = sdpa_setup(dtype, out, scale, locations, rotated_queries, fragment_lengths, key_fragments, value_fragments,
                    fragment_tokens, fragment_batch, s, workspace, workspace_bytes, p, tab, max_keys, empty);
    if (st != DVATTN_OK) return st;
    // the single launch reads the unrotated queries in vectors as well
    if (!no_rope && (st = check_aligned({{queries, "queries", 16}})) != DVATTN_OK) return st;
    bool refused = false;
    const int chunks = empty || no_rope ? -1 : small_path_chunks(dtype, s, fragment_tokens, true, &refused);
    if (refused) return DVATTN_ERR_UNSUPPORTED;
    if (chunks > 0) {
        p.q = queries;
        p.cosv = cosines;
        p.sinv = sines;
        p.R = s->rotary_dim;
        return small_launch(dtype, dv::kQRotFull, p, chunks, fragment_tokens, rotated_queries, workspace,
                            (hipStream_t)stream);
    }
    if (!no_rope) {
        const hipError_t e = dv::launch_rope(dtype, rp, (hipStream_t)stream);
        if (e != hipSuccess) return hip_fail(e, "dvattn_rope launch");
    }
    if (empty) return ok();
    return sdpa_launch(dtype, p, tab, max_keys, workspace, workspace_bytes, (hipStream_t)stream);
}

// ---------------------------------------------------------------------------
dvattn_status dvattn_rope(int dtype, void* out, const void* queries, const float* cosines, const float* sines,
                          const dvattn_shape* s, void* stream) {
    dv::RopeParams p;
    bool empty = true;
    const dvattn_status st = rope_setup(dtype, out, queries, cosines, sines, s, p, empty);
    if (st != DVATTN_OK) return st;
    if (empty) return ok();
    hipError_t e = dv::launch_rope(dtype, p, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_rope launch");
    return ok();
}

dvattn_status dvattn_varlen_rope(int dtype, void* out, const void* queries, const float* cosines,
                                 const float* sines, const dvattn_shape* s, void* stream) {
    if (!s) return fail(DVATTN_ERR_INVALID, "shape is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (s->F < 0 || s->total_q_tokens < 0 || s->Hq < 0 || s->E < 0) return fail(DVATTN_ERR_INVALID, "negative size");
    dvattn_status st;
    if ((st = check_rotary(s->rotary_dim, s->E)) != DVATTN_OK) return st;
    if ((long long)s->F * s->total_q_tokens * s->Hq * s->E == 0) return ok();  // rope.cuh:106-108
    if (!out || !queries || (s->rotary_dim > 0 && (!cosines || !sines)))
        return fail(DVATTN_ERR_INVALID, "null pointer");
    if ((st = check_aligned({{out, "out", elem_bytes(dtype)}, {queries, "queries", elem_bytes(dtype)},
                             {cosines, "cosines", 4}, {sines, "sines", 4}})) != DVATTN_OK)
        return st;
    dv::RopeParams p;
    memset(&p, 0, sizeof(p));
    p.out = out;
    p.q = queries;
    p.cosv = cosines;
    p.sinv = sines;
    p.F = s->F;
    p.T = s->total_q_tokens;
    p.Hq = s->Hq;
    p.E = s->E;
    p.R = s->rotary_dim;
    p.half_width = 1;
    hipError_t e = dv::launch_rope(dtype, p, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_varlen_rope launch");
    return ok();
}

// ---------------------------------------------------------------------------
dvattn_status dvattn_paged_kv_append(int dtype, int rope_dtype, void* k_cache, void* v_cache,
                                     const int* block_tables, const int* positions, const void* keys,
                                     const void* values, const void* cosines, const void* sines,
                                     const dvattn_shape* s, const dvattn_kv_layout* lay, void* stream) {
    if (!s || !lay) return fail(DVATTN_ERR_INVALID, "shape or layout is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (rope_dtype != DVATTN_F32 && rope_dtype != dtype)
        return fail(DVATTN_ERR_UNSUPPORTED, "cos/sin dtype code %d must be float32 or the storage dtype %d",
                    rope_dtype, dtype);
    if (s->W < 0 || s->S < 0 || s->Hkv < 0 || s->E < 0 || s->Ev < 0)
        return fail(DVATTN_ERR_INVALID, "negative W/S/Hkv/E/Ev");
    if ((long long)s->W * s->S * s->Hkv == 0 || (s->E == 0 && s->Ev == 0)) return ok();
    dvattn_status st;
    if ((st = check_rotary(s->rotary_dim, s->E)) != DVATTN_OK) return st;
    if (s->block_size <= 0) return fail(DVATTN_ERR_INVALID, "block_size must be positive (got %d)", s->block_size);
    if (s->max_blocks_per_seq < 0 || s->num_blocks < 0)
        return fail(DVATTN_ERR_INVALID, "max_blocks_per_seq / num_blocks must be >= 0");
    // the kernel indexes (token, head, element) in 32 bits
    if ((long long)s->W * s->S * s->Hkv * (s->E > s->Ev ? s->E : s->Ev) >= (1ll << 31))
        return fail(DVATTN_ERR_UNSUPPORTED, "%lld key elements in one call exceed 2^31",
                    (long long)s->W * s->S * s->Hkv * (s->E > s->Ev ? s->E : s->Ev));
    if (!k_cache || !v_cache || !keys || !values || !positions || (s->max_blocks_per_seq > 0 && !block_tables) ||
        (s->rotary_dim > 0 && (!cosines || !sines)))
        return fail(DVATTN_ERR_INVALID, "null pointer");
    // element-wise copies where the 16-byte vector form does not apply
    if ((st = check_aligned({{k_cache, "k_cache", elem_bytes(dtype)}, {v_cache, "v_cache", elem_bytes(dtype)},
                             {keys, "keys", elem_bytes(dtype)}, {values, "values", elem_bytes(dtype)},
                             {cosines, "cosines", elem_bytes(rope_dtype)}, {sines, "sines", elem_bytes(rope_dtype)},
                             {positions, "positions", 4}, {block_tables, "block_tables", 4}})) != DVATTN_OK)
        return st;
    dv::AppendParams p;
    memset(&p, 0, sizeof(p));
    p.kc = k_cache;
    p.vc = v_cache;
    p.bt = block_tables;
    p.pos = positions;
    p.k = keys;
    p.v = values;
    p.cosv = cosines;
    p.sinv = sines;
    for (int i = 0; i < 3; ++i) {
        p.kcs[i] = lay->k_cache_strides[i];
        p.vcs[i] = lay->v_cache_strides[i];
        p.ks[i] = lay->key_strides[i];
        p.vs[i] = lay->value_strides[i];
    }
    p.cs[0] = lay->rope_strides[0];
    p.cs[1] = lay->rope_strides[1];
    p.W = s->W;
    p.S = s->S;
    p.Hkv = s->Hkv;
    p.E = s->E;
    p.Ev = s->Ev;
    p.R = s->rotary_dim;
    p.bs = s->block_size;
    p.maxB = s->max_blocks_per_seq;
    p.nblocks = s->num_blocks;
    hipError_t e = dv::launch_kv_append(dtype, rope_dtype, p, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_paged_kv_append launch");
    return ok();
}

dvattn_status dvattn_view_metadata(int* locations, float* cosines, float* sines, const int* fragment_lengths,
                                   const int* order, const float* inv_freq, float attention_scaling,
                                   int round_dtype, int F, int W, int S, int rotary_dim, void* stream) {
    if (F < 0 || W < 0 || S < 0) return fail(DVATTN_ERR_INVALID, "negative F/W/S");
    if (rotary_dim < 0 || (rotary_dim & 1))
        return fail(DVATTN_ERR_UNSUPPORTED, "rotary_dim must be even and >= 0 (got %d)", rotary_dim);
    if (round_dtype != -1 && round_dtype != DVATTN_F32 && round_dtype != DVATTN_F16 && round_dtype != DVATTN_BF16)
        return fail(DVATTN_ERR_UNSUPPORTED, "unsupported round_dtype code %d", round_dtype);
    if ((long long)F * W * S == 0) return ok();
    if (!locations || !fragment_lengths || !order || (rotary_dim > 0 && (!cosines || !sines || !inv_freq)))
        return fail(DVATTN_ERR_INVALID, "null pointer");
    dv::MetaParams p;
    memset(&p, 0, sizeof(p));
    p.loc = locations;
    p.cosv = cosines;
    p.sinv = sines;
    p.fl = fragment_lengths;
    p.order = order;
    p.inv_freq = inv_freq;
    p.scaling = attention_scaling;
    p.round_dt = round_dtype == DVATTN_F32 ? -1 : round_dtype;
    p.F = F;
    p.W = W;
    p.S = S;
    p.R = rotary_dim;
    hipError_t e = dv::launch_view_meta(p, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_view_metadata launch");
    return ok();
}

// ---------------------------------------------------------------------------
dvattn_status dvattn_tree_metadata(int* locations, float* cosines, float* sines, int* tree_views, int* tree_rows,
                                   const int* fragment_lengths, const int* order, const int* parents,
                                   const float* inv_freq, float attention_scaling, int round_dtype, int F, int W,
                                   int S, int rotary_dim, void* stream) {
    return dvattn_tree_metadata_counts(locations, cosines, sines, tree_views, tree_rows, fragment_lengths, order,
                                       parents, nullptr, nullptr, inv_freq, attention_scaling, round_dtype, F, W, S,
                                       rotary_dim, stream);
}

dvattn_status dvattn_tree_metadata_counts(int* locations, float* cosines, float* sines, int* tree_views,
                                          int* tree_rows, const int* fragment_lengths, const int* order,
                                          const int* parents, const int* committed, const int* dropped,
                                          const float* inv_freq, float attention_scaling, int round_dtype, int F,
                                          int W, int S, int rotary_dim, void* stream) {
    if (F < 0 || W < 0 || S < 0) return fail(DVATTN_ERR_INVALID, "negative F/W/S");
    if (rotary_dim < 0 || (rotary_dim & 1))
        return fail(DVATTN_ERR_UNSUPPORTED, "rotary_dim must be even and >= 0 (got %d)", rotary_dim);
    if (round_dtype != -1 && !valid_dtype(round_dtype))
        return fail(DVATTN_ERR_UNSUPPORTED, "unsupported round_dtype code %d", round_dtype);
    if (S > dv::kMaxTreeNodes || F > dv::kMaxTreeViews)
        return fail(DVATTN_ERR_UNSUPPORTED, "at most %d drafted nodes and %d views (S=%d, F=%d)", dv::kMaxTreeNodes,
                    dv::kMaxTreeViews, S, F);
    if (W == 0) return ok();
    // a launch holds 2^24 blocks of 256 threads: one per (view, sequence) and 64 nodes
    if ((long long)(F > 0 ? F : 1) * W * (S > 0 ? (S + 63) / 64 : 1) >= (1ll << 24))
        return fail(DVATTN_ERR_UNSUPPORTED, "%lld (view, sequence) pairs of %d nodes exceed one launch",
                    (long long)F * W, S);
    const bool nodes = F > 0 && S > 0;
    if (!tree_views || !tree_rows || (F > 0 && (!fragment_lengths || !order)) || (S > 0 && !parents) ||
        (nodes && (!locations || (rotary_dim > 0 && (!cosines || !sines || !inv_freq)))))
        return fail(DVATTN_ERR_INVALID, "null pointer");
    const dvattn_status st = check_aligned({{locations, "locations", 4}, {cosines, "cosines", 4}, {sines, "sines", 4},
                                            {tree_views, "tree_views", 4}, {tree_rows, "tree_rows", 4},
                                            {fragment_lengths, "fragment_lengths", 4}, {order, "order", 4},
                                            {parents, "parents", 4}, {committed, "committed", 4},
                                            {dropped, "dropped", 4}, {inv_freq, "inv_freq", 4}});
    if (st != DVATTN_OK) return st;
    dv::TreeMetaParams p;
    memset(&p, 0, sizeof(p));
    p.m.loc = locations;
    p.m.cosv = cosines;
    p.m.sinv = sines;
    p.m.fl = fragment_lengths;
    p.m.order = order;
    p.m.inv_freq = inv_freq;
    p.m.scaling = attention_scaling;
    p.m.round_dt = round_dtype == DVATTN_F32 ? -1 : round_dtype;
    p.m.F = F;
    p.m.W = W;
    p.m.S = S;
    p.m.R = rotary_dim;
    p.parents = parents;
    p.committed = committed;
    p.dropped = dropped;
    p.tree_views = tree_views;
    p.tree_rows = tree_rows;
    const hipError_t e = dv::launch_tree_meta(p, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_tree_metadata launch");
    return ok();
}

// ---------------------------------------------------------------------------
static dv::TreePlan tree_plan_of(int dtype, const dvattn_shape* s) {
    return dv::tree_plan(dtype, s->F, s->W, s->S, s->Hkv, (long long)s->max_blocks_per_seq * s->block_size);
}

size_t dvattn_tree_paged_sdpa_workspace_size(int dtype, const dvattn_shape* s, int device) {
    if (!s || !valid_dtype(dtype)) return 0;
    if (s->F < 0 || s->W < 0 || s->S < 0 || s->Hkv < 0 || s->max_blocks_per_seq < 0 || s->block_size < 0) return 0;
    const dv::TreePlan plan = tree_plan_of(dtype, s);
    return plan.windows > 0 ? dv::tree_workspace_bytes(plan, s->W, s->S, s->Hkv)
                            : dv::chunk_workspace_bytes(s->W, s->S, s->Hkv, current_device(device));
}

dvattn_status dvattn_tree_paged_sdpa(int dtype, void* out, float scale, const int* locations, const void* queries,
                                     const float* cosines, const float* sines, const int* fragment_lengths,
                                     const void* k_cache, const void* v_cache, const int* block_tables,
                                     const int* parents, const int* tree_views, const int* tree_rows,
                                     const dvattn_shape* s, void* workspace, size_t workspace_bytes, void* stream) {
    if (!s) return fail(DVATTN_ERR_INVALID, "shape is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (s->F < 0 || s->W < 0 || s->S < 0) return fail(DVATTN_ERR_INVALID, "negative F/W/S");
    if ((long long)s->W * s->S == 0 || s->Hkv == 0) return ok();
    dvattn_status st;
    if ((st = check_heads(s)) != DVATTN_OK) return st;
    if ((st = check_rotary(s->rotary_dim, s->E)) != DVATTN_OK) return st;
    if ((st = check_pages(s)) != DVATTN_OK) return st;
    if (s->S > dv::kMaxTreeNodes)
        return fail(DVATTN_ERR_UNSUPPORTED, "at most %d drafted nodes per sequence (S=%d)", dv::kMaxTreeNodes, s->S);
    if (!out || !queries || !parents || !tree_views || !tree_rows)
        return fail(DVATTN_ERR_INVALID, "null output, query, parents, tree_views or tree_rows pointer");
    if (s->F > 0 && (!locations || !fragment_lengths || ((!cosines || !sines) && s->rotary_dim > 0)))
        return fail(DVATTN_ERR_INVALID, "null locations / fragment_lengths / cos / sin pointer");
    if (s->num_blocks > 0 && (!k_cache || !v_cache)) return fail(DVATTN_ERR_INVALID, "null k/v cache pointer");
    if (s->max_blocks_per_seq > 0 && !block_tables) return fail(DVATTN_ERR_INVALID, "null block_tables pointer");
    if ((st = check_aligned({{out, "out", 16}, {queries, "queries", 16}, {k_cache, "k_cache", 16},
                             {v_cache, "v_cache", 16}, {workspace, "workspace", 16}, {locations, "locations", 4},
                             {fragment_lengths, "fragment_lengths", 4}, {cosines, "cosines", 4},
                             {sines, "sines", 4}, {block_tables, "block_tables", 4}, {parents, "parents", 4},
                             {tree_views, "tree_views", 4}, {tree_rows, "tree_rows", 4}})) != DVATTN_OK)
        return st;
    const size_t need = dvattn_tree_paged_sdpa_workspace_size(dtype, s, -1);
    if (workspace_bytes < need || (need && !workspace))
        return fail(DVATTN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);

    dv::DecodeParams p;
    memset(&p, 0, sizeof(p));
    p.out = out;
    p.loc = locations;
    p.q = queries;
    p.cosv = cosines;
    p.sinv = sines;
    p.fl = fragment_lengths;
    p.kc = k_cache;
    p.vc = v_cache;
    p.bt = block_tables;
    p.parents = parents;
    p.tree_views = tree_views;
    p.tree_rows = tree_rows;
    p.keep_parts = 1;
    p.l2scale = scale * 1.4426950408889634f;
    p.F = s->F;
    p.W = s->W;
    p.S = s->S;
    p.Hq = s->Hq;
    p.Hkv = s->Hkv;
    p.R = s->rotary_dim;
    p.bs = s->block_size;
    p.bs_shift = log2_exact(s->block_size);
    p.maxB = s->max_blocks_per_seq;
    p.nblocks = s->num_blocks;
    const dv::TreePlan plan = tree_plan_of(dtype, s);
    if (plan.windows > 0) {
        p.part = reinterpret_cast<float*>(workspace);
        const hipError_t e = dv::launch_tree_small(dtype, plan, p, (hipStream_t)stream);
        if (e != hipSuccess) return hip_fail(e, "dvattn_tree_paged_sdpa launch");
        return ok();
    }
    const long long max_keys = (long long)s->max_blocks_per_seq * s->block_size;
    // Smallest key range of a workgroup.  A call too small for the GPU is cut finer: every
    // piece is merged anyway.  bf16, one sequence, 8 KV heads, with 256 / 96 keys: 8 nodes
    // on 1000 keys 29.9 / 25.1 us, 32 on 1000 38.5 / 33.9; 8 on 4000 (more workgroups than
    // that, and more pieces to merge) 30.5 / 33.4.
    const long long segments = (long long)s->W * ((s->S + 15) / 16) * s->Hkv;
    p.min_keys = segments * max_keys <= 192ll * 96 ? 96 : 256;
    const hipError_t e = dv::launch_chunk(dtype, dv::kQRotFull, dv::kKvPaged, p, max_keys, workspace, workspace_bytes,
                                          (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_tree_paged_sdpa launch");
    return ok();
}

// ---------------------------------------------------------------------------
size_t dvattn_paged_key_mass_workspace_size(int dtype, const dvattn_shape* s, long long capacity) {
    if (!s || !valid_dtype(dtype)) return 0;
    return dv::mass_workspace_bytes(dtype, s->F, s->W, s->S, s->Hkv,
                                    (long long)s->max_blocks_per_seq * s->block_size, capacity);
}

dvattn_status dvattn_paged_key_mass(int dtype, float* out, const float* mass, float decay, long long capacity,
                                    float scale, const int* locations, const void* queries, const float* cosines,
                                    const float* sines, const int* fragment_lengths, const void* k_cache,
                                    const int* block_tables, const dvattn_shape* s, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    if (!s) return fail(DVATTN_ERR_INVALID, "shape is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (s->F < 0 || s->W < 0 || s->S < 0) return fail(DVATTN_ERR_INVALID, "negative F/W/S");
    if (capacity < 0) return fail(DVATTN_ERR_INVALID, "negative capacity");
    if (s->W == 0 || s->Hkv == 0 || capacity == 0) return ok();
    dvattn_status st;
    if ((st = check_heads(s)) != DVATTN_OK) return st;
    if ((st = check_rotary(s->rotary_dim, s->E)) != DVATTN_OK) return st;
    if ((st = check_pages(s)) != DVATTN_OK) return st;
    const long long max_rows = (long long)s->max_blocks_per_seq * s->block_size;
    const long long rows = max_rows > capacity ? max_rows : capacity;
    if (max_rows >= (1ll << 32))
        return fail(DVATTN_ERR_UNSUPPORTED, "block tables of %lld rows exceed 2^32", max_rows);
    // a launch holds 2^24 blocks of 256 threads: one per 128 rows and view at least; two per token's
    // query operand and one per sequence.  (Each factor is bounded before a product that it is in.)
    const long long limit = 1ll << 24, wh = (long long)s->W * s->Hkv, sf = (long long)s->S * (s->F > 0 ? s->F : 1);
    if (wh >= limit || rows >= limit * 128 || sf >= limit || wh * (rows / 128 + s->F + 2) >= limit ||
        wh * sf * 2 + s->W > limit)
        return fail(DVATTN_ERR_UNSUPPORTED, "W=%d, Hkv=%d, S=%d, %lld rows: too many blocks for one launch", s->W,
                    s->Hkv, s->S, rows);
    if (!out || (s->S > 0 && !queries) || (decay != 0.0f && !mass))
        return fail(DVATTN_ERR_INVALID, "null out, mass or query pointer");
    if (s->F > 0 && (!fragment_lengths || (s->S > 0 && (!locations || ((!cosines || !sines) && s->rotary_dim > 0)))))
        return fail(DVATTN_ERR_INVALID, "null locations / fragment_lengths / cos / sin pointer");
    if (s->num_blocks > 0 && !k_cache) return fail(DVATTN_ERR_INVALID, "null k cache pointer");
    if (s->max_blocks_per_seq > 0 && !block_tables) return fail(DVATTN_ERR_INVALID, "null block_tables pointer");
    if ((st = check_aligned({{out, "out", 4}, {mass, "mass", 4}, {queries, "queries", 16}, {k_cache, "k_cache", 16},
                             {workspace, "workspace", 16}, {locations, "locations", 4},
                             {fragment_lengths, "fragment_lengths", 4}, {cosines, "cosines", 4},
                             {sines, "sines", 4}, {block_tables, "block_tables", 4}})) != DVATTN_OK)
        return st;
    const size_t need = dvattn_paged_key_mass_workspace_size(dtype, s, capacity);
    if (workspace_bytes < need || (need && !workspace))
        return fail(DVATTN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);

    dv::MassParams p;
    memset(&p, 0, sizeof(p));
    p.out = out;
    p.mass = mass;
    p.decay = decay;
    p.C = capacity;
    p.loc = locations;
    p.q = queries;
    p.cosv = cosines;
    p.sinv = sines;
    p.fl = fragment_lengths;
    p.kc = k_cache;
    p.bt = block_tables;
    p.l2scale = scale * 1.4426950408889634f;
    p.F = s->F;
    p.W = s->W;
    p.S = s->S;
    p.Hq = s->Hq;
    p.Hkv = s->Hkv;
    p.R = s->rotary_dim;
    p.bs = s->block_size;
    p.bs_shift = log2_exact(s->block_size);
    p.maxB = s->max_blocks_per_seq;
    p.nblocks = s->num_blocks;
    const hipError_t e = dv::launch_key_mass(dtype, p, workspace, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_paged_key_mass launch");
    return ok();
}

// ---------------------------------------------------------------------------
dvattn_status dvattn_kv_select(int* rows, const float* mass, const int* first_rows, const int* lengths,
                               long long capacity, int W, int Hkv, int budget, int keep_first, int keep_last,
                               void* stream) {
    if (W < 0 || Hkv < 0 || capacity < 0 || budget < 0 || keep_first < 0 || keep_last < 0)
        return fail(DVATTN_ERR_INVALID, "negative W/Hkv/capacity/budget/keep_first/keep_last");
    if ((long long)keep_first + keep_last > budget)
        return fail(DVATTN_ERR_INVALID, "keep_first %d and keep_last %d exceed the budget %d", keep_first, keep_last,
                    budget);
    if (capacity > (1ll << 30)) return fail(DVATTN_ERR_UNSUPPORTED, "capacity %lld exceeds 2^30 rows", capacity);
    if (budget > (1 << 30)) return fail(DVATTN_ERR_UNSUPPORTED, "budget %d exceeds 2^30 rows", budget);
    if ((long long)W * Hkv >= (1ll << 22))  // blocks of 1024 threads of one launch
        return fail(DVATTN_ERR_UNSUPPORTED, "%lld (sequence, KV head) pairs exceed 2^22", (long long)W * Hkv);
    if ((long long)W * Hkv == 0 || budget == 0) return ok();
    if (!rows || !first_rows || !lengths || (capacity > 0 && !mass)) return fail(DVATTN_ERR_INVALID, "null pointer");
    const dvattn_status st = check_aligned({{rows, "rows", 4}, {mass, "mass", 4}, {first_rows, "first_rows", 4},
                                            {lengths, "lengths", 4}});
    if (st != DVATTN_OK) return st;
    dv::SelectParams p;
    memset(&p, 0, sizeof(p));
    p.rows = rows;
    p.mass = mass;
    p.first = first_rows;
    p.lengths = lengths;
    p.C = capacity;
    p.W = W;
    p.Hkv = Hkv;
    p.budget = budget;
    p.keep_first = keep_first;
    p.keep_last = keep_last;
    const hipError_t e = dv::launch_kv_select(p, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_kv_select launch");
    return ok();
}

dvattn_status dvattn_paged_kv_compact(int dtype, void* k_cache, void* v_cache, const int* block_tables,
                                      const int* rows, int row_heads, int N, const int* first_rows,
                                      const int* lengths, float* mass, long long capacity, const dvattn_shape* s,
                                      const dvattn_kv_layout* lay, void* stream) {
    if (!s || !lay) return fail(DVATTN_ERR_INVALID, "shape or layout is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (s->W < 0 || s->Hkv < 0 || s->E < 0 || s->Ev < 0 || N < 0 || capacity < 0)
        return fail(DVATTN_ERR_INVALID, "negative W/Hkv/E/Ev/N/capacity");
    if ((long long)s->W * s->Hkv == 0) return ok();
    if (row_heads != 1 && row_heads != s->Hkv)
        return fail(DVATTN_ERR_INVALID, "rows must hold 1 or Hkv=%d heads (got %d)", s->Hkv, row_heads);
    if (s->block_size <= 0) return fail(DVATTN_ERR_INVALID, "block_size must be positive (got %d)", s->block_size);
    if (s->max_blocks_per_seq < 0 || s->num_blocks < 0)
        return fail(DVATTN_ERR_INVALID, "max_blocks_per_seq / num_blocks must be >= 0");
    if (s->E > 8192 || s->Ev > 8192)
        return fail(DVATTN_ERR_UNSUPPORTED, "head dims up to 8192 (E=%d, Ev=%d)", s->E, s->Ev);
    // blocks of 512 threads of one launch: fewer than 1024 for the slices of small calls, else up
    // to 33 per (sequence, KV head): 16 slices of 8192 elements, K and V, and mass
    if ((long long)s->W * s->Hkv >= (1ll << 15) || N > (1 << 30))
        return fail(DVATTN_ERR_UNSUPPORTED, "W * Hkv = %lld and N = %d: below 2^15 and at most 2^30",
                    (long long)s->W * s->Hkv, N);
    if (mass && !lengths) return fail(DVATTN_ERR_INVALID, "mass needs lengths");
    if (mass && capacity > (1ll << 30))
        return fail(DVATTN_ERR_UNSUPPORTED, "capacity %lld exceeds 2^30 rows", capacity);
    if (N == 0 && !mass) return ok();
    if (!first_rows || (N > 0 && !rows) || (s->max_blocks_per_seq > 0 && !block_tables) ||
        (s->num_blocks > 0 && ((s->E > 0 && !k_cache) || (s->Ev > 0 && !v_cache))))
        return fail(DVATTN_ERR_INVALID, "null pointer");
    const dvattn_status st = check_aligned({{k_cache, "k_cache", elem_bytes(dtype)},
                                            {v_cache, "v_cache", elem_bytes(dtype)}, {rows, "rows", 4},
                                            {block_tables, "block_tables", 4}, {first_rows, "first_rows", 4},
                                            {lengths, "lengths", 4}, {mass, "mass", 4}});
    if (st != DVATTN_OK) return st;
    // keys and values are moved by blocks of their own, unordered: one array would be moved twice
    if (k_cache == v_cache && s->num_blocks > 0 && s->E > 0 && s->Ev > 0)
        return fail(DVATTN_ERR_INVALID, "k_cache and v_cache are the same array");
    dv::CompactParams p;
    memset(&p, 0, sizeof(p));
    p.kc = k_cache;
    p.vc = v_cache;
    for (int i = 0; i < 3; ++i) {
        p.kcs[i] = lay->k_cache_strides[i];
        p.vcs[i] = lay->v_cache_strides[i];
    }
    p.bt = block_tables;
    p.rows = rows;
    p.first = first_rows;
    p.lengths = lengths;
    p.mass = mass;
    p.C = capacity;
    p.W = s->W;
    p.Hkv = s->Hkv;
    p.heads = row_heads;
    p.N = N;
    p.E = s->E;
    p.Ev = s->Ev;
    p.bs = s->block_size;
    p.bs_shift = log2_exact(s->block_size);
    p.maxB = s->max_blocks_per_seq;
    p.nblocks = s->num_blocks;
    const hipError_t e = dv::launch_kv_compact(dtype, p, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_paged_kv_compact launch");
    return ok();
}

// ---------------------------------------------------------------------------
static_assert(dv::kMaxTableSeqs == DVATTN_MAX_TABLE_SEQS, "header and kernels agree");

dvattn_status dvattn_block_tables(int* cu_seqlens, int* starts, int* positions, long long* slots, int* new_lengths,
                                  int* new_free_count, int* block_tables, int* free_pages, const int* lengths,
                                  const int* new_tokens, const int* free_count, int max_tokens, const dvattn_shape* s,
                                  void* stream) {
    if (!s) return fail(DVATTN_ERR_INVALID, "shape is null");
    if (s->W < 0 || max_tokens < 0) return fail(DVATTN_ERR_INVALID, "negative W / max_tokens");
    if (s->W > DVATTN_MAX_TABLE_SEQS)
        return fail(DVATTN_ERR_UNSUPPORTED, "%d sequences in one call exceed %d", s->W, DVATTN_MAX_TABLE_SEQS);
    if (s->block_size <= 0) return fail(DVATTN_ERR_INVALID, "block_size must be positive (got %d)", s->block_size);
    if (s->max_blocks_per_seq < 0 || s->num_blocks < 0)
        return fail(DVATTN_ERR_INVALID, "max_blocks_per_seq / num_blocks must be >= 0");
    if (!cu_seqlens || !new_free_count || !free_count || (max_tokens > 0 && (!positions || !slots)) ||
        (s->W > 0 && (!starts || !new_lengths || !lengths || !new_tokens)) || (s->num_blocks > 0 && !free_pages) ||
        ((long long)s->W * s->max_blocks_per_seq > 0 && !block_tables))
        return fail(DVATTN_ERR_INVALID, "null pointer");
    dvattn_status st;
    if ((st = check_aligned({{cu_seqlens, "cu_seqlens", 4}, {starts, "starts", 4}, {positions, "positions", 4},
                             {slots, "slots", 8}, {new_lengths, "new_lengths", 4},
                             {new_free_count, "new_free_count", 4}, {block_tables, "block_tables", 4},
                             {free_pages, "free_pages", 4}, {lengths, "lengths", 4}, {new_tokens, "new_tokens", 4},
                             {free_count, "free_count", 4}})) != DVATTN_OK)
        return st;
    dv::TablesParams p;
    memset(&p, 0, sizeof(p));
    p.cu = cu_seqlens;
    p.starts = starts;
    p.positions = positions;
    p.slots = slots;
    p.lengths_out = new_lengths;
    p.count_out = new_free_count;
    p.bt = block_tables;
    p.stack = free_pages;
    p.lengths = lengths;
    p.new_tokens = new_tokens;
    p.count = free_count;
    p.W = s->W;
    p.maxB = s->max_blocks_per_seq;
    p.nblocks = s->num_blocks;
    p.bs = s->block_size;
    p.T = max_tokens;
    const hipError_t e = dv::launch_block_tables(p, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_block_tables launch");
    return ok();
}

// ---------------------------------------------------------------------------
dvattn_status dvattn_paged_kv_append_q8(int dtype, int rope_dtype, void* k_cache, void* v_cache,
                                        unsigned char* k_scales, unsigned char* v_scales, const long long* slots,
                                        const void* keys, const void* values, const void* cosines, const void* sines,
                                        const dvattn_shape* s, const dvattn_kv_layout* lay, void* stream) {
    if (!s || !lay) return fail(DVATTN_ERR_INVALID, "shape or layout is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (rope_dtype != DVATTN_F32 && rope_dtype != dtype)
        return fail(DVATTN_ERR_UNSUPPORTED, "cos/sin dtype code %d must be float32 or the storage dtype %d",
                    rope_dtype, dtype);
    if (s->W < 0 || s->S < 0 || s->Hkv < 0) return fail(DVATTN_ERR_INVALID, "negative W/S/Hkv");
    dvattn_status st;
    if (s->E != 128 || s->Ev != 128)
        return fail(DVATTN_ERR_UNSUPPORTED, "only head dims E == Ev == 128 are implemented (E=%d, Ev=%d)", s->E,
                    s->Ev);
    if ((st = check_rotary(s->rotary_dim, s->E)) != DVATTN_OK) return st;
    if ((st = check_pages(s)) != DVATTN_OK) return st;
    if ((long long)s->W * s->S * s->Hkv == 0) return ok();
    if ((long long)s->W * s->S >= (1ll << 30) || s->Hkv >= (1 << 16))
        return fail(DVATTN_ERR_UNSUPPORTED, "%lld tokens / %d KV heads in one call", (long long)s->W * s->S, s->Hkv);
    if (!slots || !keys || !values || (s->num_blocks > 0 && (!k_cache || !v_cache || !k_scales || !v_scales)) ||
        (s->rotary_dim > 0 && (!cosines || !sines)))
        return fail(DVATTN_ERR_INVALID, "null pointer");
    if (s->num_blocks > 0 && (k_cache == v_cache || k_scales == v_scales))
        return fail(DVATTN_ERR_INVALID, "one array as both caches (or both scales)");
    if ((st = check_aligned({{k_cache, "k_cache", 16}, {v_cache, "v_cache", 16}, {slots, "slots", 8},
                             {keys, "keys", elem_bytes(dtype)}, {values, "values", elem_bytes(dtype)},
                             {cosines, "cosines", elem_bytes(rope_dtype)},
                             {sines, "sines", elem_bytes(rope_dtype)}})) != DVATTN_OK)
        return st;
    dv::Append8Params p;
    memset(&p, 0, sizeof(p));
    p.kc = (unsigned char*)k_cache;
    p.vc = (unsigned char*)v_cache;
    p.ks = k_scales;
    p.vs = v_scales;
    p.slots = slots;
    p.k = keys;
    p.v = values;
    for (int i = 0; i < 3; ++i) {
        p.kst[i] = lay->key_strides[i];
        p.vst[i] = lay->value_strides[i];
    }
    p.cosv = cosines;
    p.sinv = sines;
    p.cs[0] = lay->rope_strides[0];
    p.cs[1] = lay->rope_strides[1];
    p.W = s->W;
    p.S = s->S;
    p.Hkv = s->Hkv;
    p.R = s->rotary_dim;
    p.bs = s->block_size;
    p.nblocks = s->num_blocks;
    const hipError_t e = dv::launch_kv_append8(dtype, rope_dtype, p, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "dvattn_paged_kv_append_q8 launch");
    return ok();
}

// ---------------------------------------------------------------------------
size_t dvattn_paged_sdpa_q8_workspace_size(int dtype, const dvattn_shape* s, int device) {
    if (!s || !valid_dtype(dtype)) return 0;
    return dv::sdpa8_workspace_bytes(dtype, false, s->W, s->S, s->Hkv, current_device(device));
}

size_t dvattn_varlen_paged_sdpa_q8_workspace_size(int dtype, const dvattn_shape* s, int device) {
    if (!s || !valid_dtype(dtype)) return 0;
    return dv::sdpa8_workspace_bytes(dtype, true, s->W, s->total_q_tokens, s->Hkv, current_device(device));
}

}  // extern "C"

namespace {

// Checks and launch of both attentions over 8-bit caches.
dvattn_status sdpa_q8(bool varlen, int dtype, void* out, float scale, const int* locations, const void* queries,
                      const float* cosines, const float* sines, const int* fragment_lengths, const void* k_cache,
                      const void* v_cache, const unsigned char* k_scales, const unsigned char* v_scales,
                      const int* block_tables, const int* cu_seqlens_q, const dvattn_shape* s, void* workspace,
                      size_t workspace_bytes, void* stream) {
    const char* op = varlen ? "dvattn_varlen_paged_sdpa_q8 launch" : "dvattn_paged_sdpa_q8 launch";
    if (!s) return fail(DVATTN_ERR_INVALID, "shape is null");
    if (!valid_dtype(dtype)) return fail(DVATTN_ERR_UNSUPPORTED, "unsupported dtype code %d", dtype);
    if (s->F < 0 || s->W < 0 || (varlen ? s->total_q_tokens : s->S) < 0)
        return fail(DVATTN_ERR_INVALID, "negative F / W / number of tokens");
    const long long rows = varlen ? s->total_q_tokens : (long long)s->W * s->S;
    if (rows == 0 || s->Hkv == 0) return ok();
    if (rows >= (1ll << 31)) return fail(DVATTN_ERR_UNSUPPORTED, "%lld query rows exceed 2^31", rows);
    dvattn_status st;
    if ((st = check_heads(s)) != DVATTN_OK) return st;
    if ((st = check_rotary(s->rotary_dim, s->E)) != DVATTN_OK) return st;
    if ((st = check_pages(s)) != DVATTN_OK) return st;
    if (!out || !queries) return fail(DVATTN_ERR_INVALID, "null output or query pointer");
    if (varlen && s->W > 0 && !cu_seqlens_q) return fail(DVATTN_ERR_INVALID, "null cu_seqlens_q pointer");
    if (varlen && s->W == 0) return fail(DVATTN_ERR_INVALID, "tokens without any sequence");
    if (s->F > 0 && (!locations || !fragment_lengths || ((!cosines || !sines) && s->rotary_dim > 0)))
        return fail(DVATTN_ERR_INVALID, "null locations / fragment_lengths / cos / sin pointer");
    if (s->num_blocks > 0 && (!k_cache || !v_cache || !k_scales || !v_scales))
        return fail(DVATTN_ERR_INVALID, "null k/v cache or scales pointer");
    if (s->max_blocks_per_seq > 0 && !block_tables) return fail(DVATTN_ERR_INVALID, "null block_tables pointer");
    if ((st = check_aligned({{out, "out", 16}, {queries, "queries", 16}, {k_cache, "k_cache", 16},
                             {v_cache, "v_cache", 16}, {workspace, "workspace", 16}, {locations, "locations", 4},
                             {fragment_lengths, "fragment_lengths", 4}, {cosines, "cosines", 4},
                             {sines, "sines", 4}, {block_tables, "block_tables", 4},
                             {cu_seqlens_q, "cu_seqlens_q", 4}})) != DVATTN_OK)
        return st;
    const size_t need = varlen ? dvattn_varlen_paged_sdpa_q8_workspace_size(dtype, s, -1)
                               : dvattn_paged_sdpa_q8_workspace_size(dtype, s, -1);
    if (workspace_bytes < need || (need && !workspace))
        return fail(DVATTN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);
    dv::DecodeParams p;
    memset(&p, 0, sizeof(p));
    p.out = out;
    p.loc = locations;
    p.q = queries;
    p.cosv = cosines;
    p.sinv = sines;
    p.fl = fragment_lengths;
    p.kc = k_cache;
    p.vc = v_cache;
    p.ks = k_scales;
    p.vs = v_scales;
    p.bt = block_tables;
    p.cu_q = cu_seqlens_q;
    p.l2scale = scale * 1.4426950408889634f;  // scale / ln 2
    p.F = s->F;
    p.W = s->W;
    p.S = varlen ? 1 : s->S;
    p.T = varlen ? s->total_q_tokens : 0;
    p.Hq = s->Hq;
    p.Hkv = s->Hkv;
    p.R = s->rotary_dim;
    p.bs = s->block_size;
    p.bs_shift = log2_exact(s->block_size);
    p.maxB = s->max_blocks_per_seq;
    p.nblocks = s->num_blocks;
    const long long max_keys = (long long)s->max_blocks_per_seq * s->block_size;
    const hipError_t e =
        dv::launch_sdpa8(dtype, varlen, p, max_keys, workspace, workspace_bytes, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, op);
    return ok();
}

}  // namespace

extern "C" {

dvattn_status dvattn_paged_sdpa_q8(int dtype, void* out, float scale, const int* locations, const void* queries,
                                   const float* cosines, const float* sines, const int* fragment_lengths,
                                   const void* k_cache, const void* v_cache, const unsigned char* k_scales,
                                   const unsigned char* v_scales, const int* block_tables, const dvattn_shape* s,
                                   void* workspace, size_t workspace_bytes, void* stream) {
    return sdpa_q8(false, dtype, out, scale, locations, queries, cosines, sines, fragment_lengths, k_cache, v_cache,
                   k_scales, v_scales, block_tables, nullptr, s, workspace, workspace_bytes, stream);
}

dvattn_status dvattn_varlen_paged_sdpa_q8(int dtype, void* out, float scale, const int* locations,
                                          const void* queries, const float* cosines, const float* sines,
                                          const int* fragment_lengths, const void* k_cache, const void* v_cache,
                                          const unsigned char* k_scales, const unsigned char* v_scales,
                                          const int* block_tables, const int* cu_seqlens_q, const dvattn_shape* s,
                                          void* workspace, size_t workspace_bytes, void* stream) {
    return sdpa_q8(true, dtype, out, scale, locations, queries, cosines, sines, fragment_lengths, k_cache, v_cache,
                   k_scales, v_scales, block_tables, cu_seqlens_q, s, workspace, workspace_bytes, stream);
}

}  // extern "C"
