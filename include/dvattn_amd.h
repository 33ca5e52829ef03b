/*
 * dvattn_amd.h -- C ABI of the MI355X (gfx950) DVAttn library, libdvattn_amd.so.
 *
 * Drop-in replacement for the compute entry points behind the reference's
 * `libdvatt` torch operators.  Every function here is plain C: raw device
 * pointers, int sizes, a caller-owned device workspace and a HIP stream passed
 * as `void*`.  Nothing throws across this boundary; each call returns a
 * dvattn_status and, on failure, leaves a message for dvattn_last_error().
 *
 * Reference interfaces replaced (paths in the reference repository):
 *   dvattn_paged_sdpa        <- op `dvattn_paged_sdpa`, src/binding.cu:412-413,151-203
 *                               (+ rope_gpu src/rope.cuh:54-65 and
 *                               paged_v21::dvattn_paged_attention_gpu
 *                               src/kernels/paged_kernel_v21.cuh:377-431)
 *   dvattn_varlen_paged_sdpa <- op `dvattn_varlen_paged_sdpa`, src/binding.cu:418-420,249-296
 *                               (+ rope_varlen_gpu src/rope.cuh:102-114 and
 *                               src/kernels/varlen_paged_kernel_v21.cuh:373-428)
 *   dvattn_sdpa              <- op `dvattn_sdpa`, src/binding.cu:410-411,79-149
 *                               (+ v21::dvattn_attention_gpu src/kernels/kernel_v21.cuh:369-414)
 *   dvattn_fused             <- op `dvattn_fused`, src/binding.cu:415-416,356-372
 *   dvattn_rope              <- op `dvattn_rope`, src/binding.cu:414,41-77 (rope_gpu)
 *   dvattn_varlen_rope       <- op `dvattn_varlen_rope`, src/binding.cu:417,205-247
 *   dvattn_shape             <- struct Shape, src/common.h:5-20
 * and, around the path (the reference does these in Python):
 *   dvattn_paged_kv_append   <- python/dvattn/attention.py:304 + 141-152 (key rotation and
 *                               cache append of a decode step), 245-251 (merge_caches)
 *   dvattn_view_metadata     <- python/dvattn/attention.py:158-186 (per-view locations,
 *                               cos/sin)
 * and, with no counterpart there, for drafted token trees and bounded caches:
 *   dvattn_tree_metadata, dvattn_tree_paged_sdpa, dvattn_paged_key_mass,
 *   dvattn_kv_select, dvattn_paged_kv_compact;
 * and for caches held in 8 bits:
 *   dvattn_block_tables, dvattn_paged_kv_append_q8, dvattn_paged_sdpa_q8,
 *   dvattn_varlen_paged_sdpa_q8.
 *
 * Semantics (identical to the reference operators):
 *   - GQA factor 16 (Hq == 16*Hkv) and head dims E == Ev == 128 only; other
 *     shapes are rejected with DVATTN_ERR_UNSUPPORTED (the reference printed a
 *     message and returned/no-op'd, paged_kernel_v21.cuh:426-429, kernel_v21.cuh:410-413).
 *   - Query rotation: dims e < R use x*cos - rotate_half(x)*sin with the first
 *     R/2 entries of each cos/sin row (full width [.., R] for paged/contiguous,
 *     half width [.., R/2] for varlen); dims >= R are copied.  fp32 math,
 *     rotated query rounded to the storage type before the dot products.
 *   - Key l of view f is visible to a query iff 0 <= l <= locations[f, row]
 *     and l < fragment_lengths[f]; one softmax over all visible keys of all
 *     views; fp32 accumulation; a query row with no visible key outputs zeros.
 *     scale may be negative, or zero (all visible keys weigh the same).
 *   - Paged views are laid out back to back in each sequence's logical token
 *     stream: view f starts at sum_{g<f} fragment_lengths[g]; logical position
 *     p lives in page block_tables[w, p / block_size], row p % block_size of a
 *     [num_blocks, block_size, Hkv, E] cache.
 *   - Keys whose logical page is beyond the block_tables row, or whose page id
 *     is outside [0, num_blocks), are treated as not visible (the reference
 *     reads out of bounds there).
 *
 * Alignment (checked; the reference's kernels assumed 16-byte vectors,
 * paged_kernel_v21.cuh:58-62, without checking): the attention entry points
 * (dvattn_paged_sdpa[_noalloc], dvattn_varlen_paged_sdpa, dvattn_sdpa,
 * dvattn_fused, dvattn_tree_paged_sdpa, dvattn_paged_key_mass, dvattn_paged_sdpa_q8,
 * dvattn_varlen_paged_sdpa_q8) need out, queries, rotated_queries, k_cache, v_cache, every
 * key/value fragment and the workspace 16-byte aligned and the int32 / fp32
 * arrays 4-byte aligned; dvattn_rope, dvattn_varlen_rope,
 * dvattn_paged_kv_append, the metadata entries, dvattn_kv_select,
 * dvattn_paged_kv_compact and dvattn_block_tables need each array aligned to its element
 * size, and so does dvattn_paged_kv_append_q8, but for its caches (16 bytes).  A
 * pointer off its alignment returns DVATTN_ERR_INVALID, naming the argument.
 * Tensors from a device allocator, and views of them that start on a row of
 * the last dimension, always qualify.
 */
#ifndef DVATTN_AMD_H
#define DVATTN_AMD_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DVATTN_ABI_VERSION 1

#if defined(__GNUC__) || defined(__clang__)
#define DVATTN_API __attribute__((visibility("default")))
#else
#define DVATTN_API
#endif

/* Storage type of queries / keys / values / outputs (cos/sin are always fp32,
 * index tensors int32), binding.cu:14-38. */
typedef enum dvattn_dtype {
    DVATTN_F32 = 0,
    DVATTN_F16 = 1,
    DVATTN_BF16 = 2
} dvattn_dtype;

typedef enum dvattn_status {
    DVATTN_OK = 0,
    DVATTN_ERR_INVALID = 1,     /* bad argument (null pointer, inconsistent sizes) */
    DVATTN_ERR_UNSUPPORTED = 2, /* shape/dtype outside what the kernels implement */
    DVATTN_ERR_WORKSPACE = 3,   /* workspace smaller than the *_workspace_size query */
    DVATTN_ERR_HIP = 4          /* a HIP runtime call failed */
} dvattn_status;

/* Launch descriptor, mirrors Shape (src/common.h:5-20).  Fields an entry point
 * does not use are ignored. */
typedef struct dvattn_shape {
    int F;                  /* views ("fragments") */
    int W;                  /* sequences ("workers") */
    int Hq;                 /* query heads (16 * Hkv) */
    int Hkv;                /* key/value heads */
    int E;                  /* q/k head dim (128) */
    int Ev;                 /* v head dim (128) */
    int S;                  /* query tokens per sequence (paged / contiguous) */
    int block_size;         /* page size in tokens (paged, varlen) */
    int max_blocks_per_seq; /* block_tables row length (paged, varlen) */
    int total_q_tokens;     /* T (varlen) */
    int num_blocks;         /* pages in k_cache / v_cache (paged, varlen) */
    int rotary_dim;         /* R (even, <= E; 0 = no rotation) */
} dvattn_shape;

/* Last error message of the calling thread ("" if none). */
DVATTN_API const char* dvattn_last_error(void);
DVATTN_API int dvattn_abi_version(void);

/* Process-wide switches.  No counterpart in the reference (its kernels have no
 * such choices).  Each starts from an environment variable, read once at first
 * use; dvattn_set_option replaces the value for all later calls (set it while
 * no other thread is inside a call, or those calls may see either value).
 *   "small_path"  (DVATTN_SMALL_PATH: 0/"0" off, 1 auto = default, 2/"require",
 *                  3/"force"): the single-launch path of dvattn_sdpa /
 *                  dvattn_fused; require fails a call it cannot take with
 *                  DVATTN_ERR_UNSUPPORTED, force takes it past its workgroup limit.
 * dvattn_get_option returns the current value, -1 for an unknown name. */
DVATTN_API dvattn_status dvattn_set_option(const char* name, int value);
DVATTN_API int dvattn_get_option(const char* name);

/* ---- paged decode attention with fused query RoPE --------------------------
 * out [W,Hq,S,Ev] T; locations [F,W,S] i32; queries [W,Hq,S,E] T;
 * cosines/sines [F,W,S,R] f32; fragment_lengths [F] i32 (device);
 * k_cache [num_blocks,block_size,Hkv,E] T; v_cache [num_blocks,block_size,Hkv,Ev] T;
 * block_tables [W,max_blocks_per_seq] i32.  All contiguous, on one device.
 * Replaces binding.cu:151-203 / paged_kernel_v21.cuh:377-431. */
DVATTN_API size_t dvattn_paged_sdpa_workspace_size(int dtype, const dvattn_shape* shape, int device);
DVATTN_API dvattn_status dvattn_paged_sdpa(int dtype, void* out, float scale, const int* locations,
                                const void* queries, const float* cosines, const float* sines,
                                const int* fragment_lengths, const void* k_cache, const void* v_cache,
                                const int* block_tables, const dvattn_shape* shape,
                                void* workspace, size_t workspace_bytes, void* stream);

/* ---- paged decode attention without allocation -----------------------------
 * No counterpart in the reference.  For callers that cannot allocate device
 * memory: code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc.  Same arguments, checks and results as dvattn_paged_sdpa,
 * minus the workspace: the partial results and merge directory live in a static
 * device array of DVATTN_NOALLOC_SCRATCH_BYTES that each GPU the library runs on
 * holds until the process ends.  A shape whose dvattn_paged_sdpa_workspace_size
 * exceeds it is rejected with DVATTN_ERR_WORKSPACE.  The call allocates nothing
 * (no hipMalloc, no allocating library routine).  Every call on a GPU uses that
 * GPU's one array: calls that overlap on one GPU (two streams or threads at
 * once) race and must be serialised by the caller. */
#define DVATTN_NOALLOC_SCRATCH_BYTES (64u << 20)
DVATTN_API dvattn_status dvattn_paged_sdpa_noalloc(int dtype, void* out, float scale, const int* locations,
                                        const void* queries, const float* cosines, const float* sines,
                                        const int* fragment_lengths, const void* k_cache,
                                        const void* v_cache, const int* block_tables,
                                        const dvattn_shape* shape, void* stream);

/* ---- varlen paged decode attention with fused query RoPE -------------------
 * out [T,Hq,Ev] T; locations [F,T] i32 (a view with locations < 0 is skipped);
 * queries [T,Hq,E] T; cosines/sines [F,T,R/2] f32 (half width);
 * cu_seqlens_q [W+1] i32: token t belongs to the first sequence i with
 * t < cu_seqlens_q[i+1] (sequence 0 if none); cu_seqlens_k is accepted and,
 * as in the reference (binding.cu:279,290), not read.  16-bit calls with
 * T >= 2W (and W <= 4096) read each sequence's K/V once per group of up to 16
 * of its tokens (the workspace size follows the same rule); other calls once
 * per token, as the reference does.
 * Replaces binding.cu:249-296 / varlen_paged_kernel_v21.cuh:373-428. */
DVATTN_API size_t dvattn_varlen_paged_sdpa_workspace_size(int dtype, const dvattn_shape* shape, int device);
DVATTN_API dvattn_status dvattn_varlen_paged_sdpa(int dtype, void* out, float scale, const int* locations,
                                       const void* queries, const float* cosines, const float* sines,
                                       const int* fragment_lengths, const void* k_cache,
                                       const void* v_cache, const int* block_tables,
                                       const int* cu_seqlens_q, const int* cu_seqlens_k,
                                       const dvattn_shape* shape, void* workspace,
                                       size_t workspace_bytes, void* stream);

/* ---- contiguous-view attention on already-rotated queries ------------------
 * out [W,Hq,S,Ev] T; locations [F,W,S]; rotated_queries [F,W,Hq,S,E] T;
 * fragment_lengths [F] i32 (device).  key_fragments[f] / value_fragments[f]
 * (host arrays of F device pointers) point at [B_f,Hkv,L_f,E|Ev] T tensors;
 * fragment_tokens[f] = L_f and fragment_batch[f] = B_f (host arrays).  B_f is
 * W, or 1 for a fragment shared by every sequence (the PyTorch reference
 * broadcasts it, attention.py:45,53).  Visible keys are also bounded by L_f.
 * Replaces binding.cu:79-149 / kernel_v21.cuh:369-414. */
DVATTN_API size_t dvattn_sdpa_workspace_size(int dtype, const dvattn_shape* shape, int device);
DVATTN_API dvattn_status dvattn_sdpa(int dtype, void* out, float scale, const int* locations,
                          const void* rotated_queries, const int* fragment_lengths,
                          const void* const* key_fragments, const void* const* value_fragments,
                          const int* fragment_tokens, const int* fragment_batch,
                          const dvattn_shape* shape, void* workspace, size_t workspace_bytes,
                          void* stream);

/* ---- rope + contiguous attention (dvattn_fused) -----------------------------
 * Writes rotated_queries [F,W,Hq,S,E] (from queries [W,Hq,S,E] and full-width
 * cos/sin [F,W,S,R]) and then runs dvattn_sdpa on it.
 * Replaces binding.cu:356-372.  Same workspace size as dvattn_sdpa. */
DVATTN_API dvattn_status dvattn_fused(int dtype, void* out, void* rotated_queries, float scale,
                           const int* locations, const void* queries, const int* fragment_lengths,
                           const void* const* key_fragments, const void* const* value_fragments,
                           const int* fragment_tokens, const int* fragment_batch,
                           const float* cosines, const float* sines, const dvattn_shape* shape,
                           void* workspace, size_t workspace_bytes, void* stream);

/* ---- standalone query rotation ---------------------------------------------
 * dvattn_rope: out [F,W,Hq,S,E] from queries [W,Hq,S,E], cos/sin [F,W,S,R].
 * Replaces binding.cu:41-77 + rope.cuh:54-65.
 * dvattn_varlen_rope: out [F,T,Hq,E] from queries [T,Hq,E], cos/sin [F,T,R/2].
 * Replaces binding.cu:205-247 + rope.cuh:102-114. */
DVATTN_API dvattn_status dvattn_rope(int dtype, void* out, const void* queries, const float* cosines,
                          const float* sines, const dvattn_shape* shape, void* stream);
DVATTN_API dvattn_status dvattn_varlen_rope(int dtype, void* out, const void* queries, const float* cosines,
                                 const float* sines, const dvattn_shape* shape, void* stream);

/* ---- K side of a decode step: rotate new keys, append K/V into pages --------
 * For every new token (w, s) with positions[w,s] = p >= 0, page
 * block_tables[w, p / block_size], row p % block_size:
 *   k_cache[page, row, h, :] = rope(keys[w, h, s, :], cosines[w, s, :], sines[w, s, :])
 *   v_cache[page, row, h, :] = values[w, h, s, :]
 * rope is the reference's apply_rotary_pos_emb (attention.py:82-88): dims e < R
 * take x*cos + rotate_half(x)*sin reading all R entries of the cos/sin row,
 * dims >= R are copied; each product and the sum are rounded to the promoted
 * dtype of (keys, cos) and the result to the storage type, exactly as PyTorch
 * evaluates it.  rope_dtype is DVATTN_F32 or dtype (the model dtype the
 * transformers rotary embedding returns).  Tokens whose position is negative
 * (masked), past the block_tables row or on a page outside [0, num_blocks) are
 * not written.  Uses shape fields W, Hkv, S, E, Ev, block_size,
 * max_blocks_per_seq, num_blocks, rotary_dim; positions [W,S] and block_tables
 * [W,max_blocks_per_seq] are contiguous int32; the other tensors are described
 * by element strides (last dim contiguous; cos/sin strides may be 0 to
 * broadcast one row, which makes this merge_caches' constant-offset
 * re-rotation, attention.py:245-251).  Keys/values must not overlap the cache
 * rows this call writes (they may live elsewhere in the cache allocations).
 * Replaces attention.py:304 (key rotation) + attention.py:141-152 (append to the
 * sequence's cache, transformers Cache.update). */
typedef struct dvattn_kv_layout {
    long long key_strides[3];     /* keys [W,Hkv,S,E]: strides of w, h, s */
    long long value_strides[3];   /* values [W,Hkv,S,Ev] */
    long long rope_strides[2];    /* cosines / sines [W,S,R]: strides of w, s */
    long long k_cache_strides[3]; /* k_cache [num_blocks,block_size,Hkv,E]: page, row, head */
    long long v_cache_strides[3]; /* v_cache [num_blocks,block_size,Hkv,Ev] */
} dvattn_kv_layout;

DVATTN_API dvattn_status dvattn_paged_kv_append(int dtype, int rope_dtype, void* k_cache, void* v_cache,
                                     const int* block_tables, const int* positions, const void* keys,
                                     const void* values, const void* cosines, const void* sines,
                                     const dvattn_shape* shape, const dvattn_kv_layout* layout, void* stream);

/* ---- per-view locations and rotary cos/sin on the device ---------------------
 * locations [F,W,S] i32, cosines/sines [F,W,S,R] f32 (R = rotary_dim, full
 * width, both halves equal) from fragment_lengths [F] i32 (device; lengths
 * already including the S new tokens), order [W,F] i32 (order[w, j]: the view
 * index of sequence w's j-th segment, its own segment last) and inv_freq
 * [R/2] f32 (the model's rotary inverse frequencies):
 *   locations[f,w,s] = (sum of the lengths of w's segments from f's place in
 *                       its order to the end) - S + s
 *   cos/sin[f,w,s,i] = cos/sin(float(locations[f,w,s]) * inv_freq[i % (R/2)])
 *                      * attention_scaling
 * A view missing from a sequence's order gets location -1 and cos 1, sin 0.
 * round_dtype (-1, DVATTN_F16 or DVATTN_BF16) rounds cos/sin through that type,
 * as the reference does when the model runs in it (rotary output in the model
 * dtype, then .to(float)).
 * Replaces attention.py:158-186 (DVAttnCache.update's host loops and the
 * transformers rotary embedding call). */
DVATTN_API dvattn_status dvattn_view_metadata(int* locations, float* cosines, float* sines,
                                   const int* fragment_lengths, const int* order, const float* inv_freq,
                                   float attention_scaling, int round_dtype, int F, int W, int S,
                                   int rotary_dim, void* stream);

/* ---- a step that drafts a token tree per sequence: metadata --------------------
 * Each of W sequences drafts a tree of up to S nodes.  parents [W,S] i32:
 * parents[w,s] = -1 for a child of the committed tokens, or the index of an
 * earlier node (0 .. s-1); any other entry makes the node absent (padding of a
 * smaller tree), and with it every node below it.  The S drafted rows are the
 * last S of each sequence's own view (its last in order): fragment_lengths
 * count them, and c(g), the committed tokens of view g, is fragment_lengths[g] -
 * S where g is the own view of some sequence, else fragment_lengths[g] (at least
 * 0).  With d(s) the depth of node s (0 for a child of the committed tokens):
 *   position(f,w,s)    = (sum of c over w's segments from f's place in its order
 *                        to the end) + d(s)
 *   locations[f,w,s]   = c(f) - 1          (the committed keys of the view)
 *   cos/sin[f,w,s,i]   = cos/sin(float(position) * inv_freq[i % (R/2)])
 *                        * attention_scaling, rounded as round_dtype says
 *   tree_views[w]      = w's own view (-1: none)
 *   tree_rows[w]       = the stream row of node 0: c(own) after the sum of the
 *                        fragment_lengths before the view; node s is written to
 *                        tree_rows[w] + s (dvattn_paged_kv_append's positions)
 * Absent nodes and views missing from a sequence's order get location -1, cos 1,
 * sin 0.  Without views (F = 0) or nodes (S = 0) tree_views and tree_rows (0 for no
 * view) are still written.  The other sequences' drafted nodes are neither seen nor counted.  For
 * one sequence and a chain (parents -1, 0, 1, ...) cos/sin are
 * dvattn_view_metadata's.  S <= 4096, F <= 4096.
 *
 * fragment_lengths are every sequence's alike, and a view's rows are the tokens it has
 * seen.  dvattn_tree_metadata_counts lifts both, each by an array [W,F] i32 or null:
 *   committed[w,g] -- c(g) of sequence w (below 0: 0), in place of what the length gives.
 *     Of sequences that share a view's length and hold different numbers of rows in it:
 *     fragment_lengths are then at least the most committed rows and S, and a node's
 *     row tree_rows[w] + s lies behind its own sequence's.
 *   dropped[w,g] -- tokens of the view that sequence w no longer holds, counted by
 *     position(f,w,s) beside c(g) and by nothing else.  A cache that was cut
 *     (dvattn_kv_select, dvattn_paged_kv_compact) holds fewer rows than its sequence has
 *     seen tokens, and its keys keep the rotation of their own positions. */
#define DVATTN_MAX_TREE_NODES 4096
DVATTN_API dvattn_status dvattn_tree_metadata(int* locations, float* cosines, float* sines, int* tree_views,
                                   int* tree_rows, const int* fragment_lengths, const int* order,
                                   const int* parents, const float* inv_freq, float attention_scaling,
                                   int round_dtype, int F, int W, int S, int rotary_dim, void* stream);
DVATTN_API dvattn_status dvattn_tree_metadata_counts(int* locations, float* cosines, float* sines, int* tree_views,
                                   int* tree_rows, const int* fragment_lengths, const int* order,
                                   const int* parents, const int* committed, const int* dropped,
                                   const float* inv_freq, float attention_scaling, int round_dtype, int F, int W,
                                   int S, int rotary_dim, void* stream);

/* ---- attention of drafted token trees over a paged cache -------------------------
 * dvattn_paged_sdpa's arguments, with S drafted nodes per sequence, and parents
 * [W,S], tree_views [W], tree_rows [W] as above.  Node s of sequence w sees
 *   - key l of view f iff l <= locations[f,w,s] and l < fragment_lengths[f], as in
 *     dvattn_paged_sdpa, and
 *   - of view tree_views[w], the keys in stream rows tree_rows[w] + j for j = s and
 *     every ancestor j of s, if the row lies inside the view,
 * each key once.  An absent node's output is zeros.  A drafted row that a node
 * does not see is not read for it, whatever it holds; a committed key past a
 * node's location but within that of another node of its sequence takes part with
 * weight 0 and must be finite, as in dvattn_paged_sdpa.  S <= 4096.
 * Weights of bf16 calls are rounded to bf16 for the product with V, as in
 * dvattn_paged_sdpa, where the block tables are wide; under narrow ones (and in the other
 * types) they are not: the same keys may round differently under another table. */
DVATTN_API size_t dvattn_tree_paged_sdpa_workspace_size(int dtype, const dvattn_shape* shape, int device);
DVATTN_API dvattn_status dvattn_tree_paged_sdpa(int dtype, void* out, float scale, const int* locations,
                                     const void* queries, const float* cosines, const float* sines,
                                     const int* fragment_lengths, const void* k_cache, const void* v_cache,
                                     const int* block_tables, const int* parents, const int* tree_views,
                                     const int* tree_rows, const dvattn_shape* shape, void* workspace,
                                     size_t workspace_bytes, void* stream);

/* ---- attention weight that every cached key receives ------------------------------
 * out, mass [W,Hkv,capacity] f32 by stream row (view f's key l is row l + the sum of
 * the fragment_lengths before f; negative lengths count as 0):
 *   out[w,h,c] = decay * mass[w,h,c] + the softmax weights that the S queries and 16
 *                query heads of KV head h give to the key in row c
 * with the weights of dvattn_paged_sdpa (same queries, locations, cos/sin, scale), in
 * fp32.  Rows no query sees only decay; rows from capacity on take part in the
 * softmax and are not stored.  All S queries take part and see what their locations say:
 * those of a drafted tree (dvattn_tree_metadata) leave out its own rows, so a tree's
 * accepted tokens are passed as the causal chain they are once they are kept.  out may be
 * mass (accumulation in place), else they
 * must not overlap; with decay 0 mass is not read and may be null.  Every key is
 * summed in a fixed order: the same call gives the same bits.  Workspace of a single
 * token: about a quarter of a 16-bit K cache of W * max_blocks_per_seq pages, at most
 * 1 GiB of scores; of several: the rotated queries of all of them, [F,W,Hq,S,E] in dtype,
 * and 128 bytes per KV head, part of the keys (32 to 256 rows) and token, of at most 64
 * tokens at a time. */
DVATTN_API size_t dvattn_paged_key_mass_workspace_size(int dtype, const dvattn_shape* shape, long long capacity);
DVATTN_API dvattn_status dvattn_paged_key_mass(int dtype, float* out, const float* mass, float decay,
                                    long long capacity, float scale, const int* locations, const void* queries,
                                    const float* cosines, const float* sines, const int* fragment_lengths,
                                    const void* k_cache, const int* block_tables, const dvattn_shape* shape,
                                    void* workspace, size_t workspace_bytes, void* stream);

/* ---- which rows of a cache to keep --------------------------------------------------
 * rows [W,Hkv,budget] i32 from mass [W,Hkv,capacity] f32: of the n = lengths[w] rows
 * from stream row first_rows[w] on (n at least 0 and at most capacity -
 * first_rows[w]; none for a negative first row), relative to it and ascending: all
 * of them if n <= budget, followed by -1; else the first keep_first, the last
 * keep_last and the budget - keep_first - keep_last of greatest mass among the
 * others (ties to the lowest row; NaN weighs least).  keep_first + keep_last <=
 * budget; capacity <= 2^30. */
DVATTN_API dvattn_status dvattn_kv_select(int* rows, const float* mass, const int* first_rows, const int* lengths,
                               long long capacity, int W, int Hkv, int budget, int keep_first, int keep_last,
                               void* stream);

/* ---- moving kept rows together --------------------------------------------------------
 * In place, for every sequence, KV head and i < N with rows[w,h,i] >= i (and <
 * lengths[w] where lengths is given):
 *   cache row (stream row first_rows[w] + i) = what row first_rows[w] + rows[w,h,i] held
 * in K and V; other rows are left as they are.  rows [W,row_heads,N] i32, row_heads
 * Hkv or 1 (the same rows for every KV head: a tree's accepted path, with first_rows =
 * tree_rows).  Entries may come in any order and more than once; one below its place,
 * past the range, or whose source or destination lies on no valid page moves nothing.
 * With mass [W,Hkv,capacity] f32 (needs lengths) its entries move by the rows and the
 * range alone (row first_rows[w] + i takes the entry of rows[w,h,i], whatever the pages), and
 * those of the rows first_rows[w] + i, i < lengths[w], that nothing moves into become 0
 * (capacity <= 2^30).  Uses
 * shape fields W, Hkv, E, Ev, block_size, max_blocks_per_seq, num_blocks and the
 * layout's cache strides.  The queries that follow keep counting positions with the rows
 * that went (dropped above).  The pages of the rows moved must each be named once in
 * block_tables (pages shared by sequences or segments lie before first_rows), and k_cache
 * and v_cache may not share rows (the same array is refused). */
DVATTN_API dvattn_status dvattn_paged_kv_compact(int dtype, void* k_cache, void* v_cache, const int* block_tables,
                                      const int* rows, int row_heads, int N, const int* first_rows,
                                      const int* lengths, float* mass, long long capacity,
                                      const dvattn_shape* shape, const dvattn_kv_layout* layout, void* stream);

/* ---- block tables, positions and slots of a step ---------------------------------------
 * From the tokens each sequence holds, lengths [W] i32, and those it adds in this step,
 * new_tokens [W] i32 (0: none; below 0: the sequence has ended):
 *   - an ended sequence's pages, block_tables[w, 0 .. ceil(lengths[w] / block_size)), are
 *     pushed on the stack free_pages [num_blocks] i32, whose first *free_count entries are
 *     free pages, in order of w and page; its length becomes 0 (its row is left as it is);
 *   - every other sequence takes the pages that lengths[w] + new_tokens[w] tokens need
 *     beyond those it holds, from the top of that stack down, in order of w, and they are
 *     written to its row.  A sequence is refused if its row or the max_tokens packed
 *     tokens have no room for it, or if the stack does not hold the pages that it and all
 *     sequences before it that were not refused for room need: it takes no page and its
 *     length stays;
 *   - the step's tokens are packed in order of w: cu_seqlens [W+1] i32 are the sums of the
 *     new tokens (refused sequences keep their places), starts [W] i32 the position of
 *     each sequence's first new token (-1: refused or ended), positions [max_tokens] i32
 *     and slots [max_tokens] i64 those of each packed token: position p lies in slot
 *     block_tables[w, p / block_size] * block_size + p % block_size (-1 for both: a
 *     token of a refused sequence, or behind the last; slot -1 too where the table names
 *     no page);
 *   - new_lengths [W] and new_free_count [1] hold the state after the step; they may be
 *     lengths and free_count.  The same call on the same lengths and count gives the same.
 * A page must be held by one sequence when it ends (pages that sequences share would be
 * pushed twice).  Lengths outside [0, max_blocks_per_seq * block_size] and counts outside
 * [0, num_blocks] are brought into the range.  Uses W, max_blocks_per_seq, num_blocks and
 * block_size; W <= DVATTN_MAX_TABLE_SEQS.  One launch, two from 4097 tokens on. */
#define DVATTN_MAX_TABLE_SEQS 8192
DVATTN_API dvattn_status dvattn_block_tables(int* cu_seqlens, int* starts, int* positions, long long* slots,
                                  int* new_lengths, int* new_free_count, int* block_tables, int* free_pages,
                                  const int* lengths, const int* new_tokens, const int* free_count, int max_tokens,
                                  const dvattn_shape* shape, void* stream);

/* ---- caches held in 8 bits --------------------------------------------------------------
 * k_cache [num_blocks,block_size,Hkv,E], v_cache [num_blocks,block_size,Hkv,Ev] hold OCP E4M3
 * bytes and k_scales, v_scales [num_blocks,Hkv] an exponent byte b (E8M0) for each page
 * and KV head: an element is byte * 2^(b - 127).  b = 0 is an empty page (its elements count
 * as zeros, whatever its bytes are), so scales cleared to zero make a valid cache; b = 255 is
 * no number: the elements are NaN to the tokens that see them.
 *
 * dvattn_paged_kv_append_q8 rounds new tokens to that form.  Token (w, s) is written to
 * slots[w,s] i64 (slot = page * block_size + row; negative or past the cache: not
 * written): the key rotated as dvattn_paged_kv_append rotates it and rounded to the storage type, and
 * the value, as that cache would hold them.  For each page, KV head, and keys and
 * values apart, with amax the largest finite magnitude written to the page:
 *   - the exponent that amax asks for is the smallest b >= 1 with amax <= 448 * 2^(b - 127);
 *   - if row 0 of the page is written (or b was 255), the page starts anew: it takes
 *     that exponent, and its rows that are not written hold nothing any more;
 *   - else it takes the larger of that and its own, and if its own was smaller, all
 *     rows that are not written are rounded again under the new one (exact but for elements
 *     that become less than 2^-6 of the new unit);
 *   - elements are rounded to E4M3, ties to even.  NaN and infinities become NaN; finite fp16
 *     magnitudes above 61440 are held as 61440.
 * A sequence that fills its pages in order thus never reads what a page held before.  Slots
 * may come in any order and more than once (the last token of a slot is the one that is
 * held); tokens in consecutive slots are the fast case.  Keys and values must not overlap
 * the caches.  Strides as in dvattn_kv_layout (its cache strides are not read: caches and
 * scales are contiguous).  Uses W, Hkv, S, E = Ev = 128, block_size, num_blocks, rotary_dim. */
DVATTN_API dvattn_status dvattn_paged_kv_append_q8(int dtype, int rope_dtype, void* k_cache, void* v_cache,
                                        unsigned char* k_scales, unsigned char* v_scales, const long long* slots,
                                        const void* keys, const void* values, const void* cosines,
                                        const void* sines, const dvattn_shape* shape, const dvattn_kv_layout* layout,
                                        void* stream);

/* dvattn_paged_sdpa and dvattn_varlen_paged_sdpa over such caches: the same arguments, the
 * caches' bytes and their scales.  dtype is that of queries and out; every element of a
 * cache is exact in the products, queries are rounded to dtype after their rotation,
 * and weights to bf16 in bf16 calls (fp16 calls carry 16 bits of them, fp32 calls
 * 24).  bf16 calls hold a split row's partial results as fp16 under a power of two per
 * row, within 2^-11 of its largest element.  But fp16 calls of more than eight tokens per
 * sequence, and packed sequences of more than four, take keys as fp16 numbers, whose
 * magnitudes end at 65504 and whose spacing at 2^-24: caches that an fp16 append wrote hold no
 * larger ones. */
DVATTN_API size_t dvattn_paged_sdpa_q8_workspace_size(int dtype, const dvattn_shape* shape, int device);
DVATTN_API dvattn_status dvattn_paged_sdpa_q8(int dtype, void* out, float scale, const int* locations,
                                   const void* queries, const float* cosines, const float* sines,
                                   const int* fragment_lengths, const void* k_cache, const void* v_cache,
                                   const unsigned char* k_scales, const unsigned char* v_scales,
                                   const int* block_tables, const dvattn_shape* shape, void* workspace,
                                   size_t workspace_bytes, void* stream);
DVATTN_API size_t dvattn_varlen_paged_sdpa_q8_workspace_size(int dtype, const dvattn_shape* shape, int device);
DVATTN_API dvattn_status dvattn_varlen_paged_sdpa_q8(int dtype, void* out, float scale, const int* locations,
                                          const void* queries, const float* cosines, const float* sines,
                                          const int* fragment_lengths, const void* k_cache, const void* v_cache,
                                          const unsigned char* k_scales, const unsigned char* v_scales,
                                          const int* block_tables, const int* cu_seqlens_q, const dvattn_shape* shape,
                                          void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DVATTN_AMD_H */
