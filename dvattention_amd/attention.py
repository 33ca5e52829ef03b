"""Python operator API, mirroring python/dvattn/attention.py:17-88 of the reference.

Every ``dvattn_*`` wrapper calls ``torch.ops.libdvatt.<op>`` (registered by
``_libdvatt.so`` over the HIP kernels); there is no eager fallback.  The
function names, argument order and defaults are the reference's; the paged /
varlen operators, which the reference exposes only through ``torch.ops``, get
thin wrappers as well.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch


def dvattn_fused(queries: torch.Tensor, locations: torch.Tensor, keys: list, values: list,
                 scale: float, fragment_lengths, cosines: torch.Tensor, sines: torch.Tensor, *,
                 rotated_queries, out):
    """Rope + attention over contiguous views (attention.py:17-21).

    queries ``[W,Hq,S,E]``, cosines/sines ``[F,W,S,R]`` fp32; writes the rotated
    queries ``[F,W,Hq,S,E]`` into ``rotated_queries`` and the result into ``out``.
    """
    torch.ops.libdvatt.dvattn_fused(out, rotated_queries, scale, locations, queries.contiguous(),
                                    fragment_lengths, keys, values, cosines, sines)
    return out


def dvattn_sdpa(queries: torch.Tensor, locations: torch.Tensor, keys: list, values: list,
                scale: float, fragment_lengths=None, out=None) -> torch.Tensor:
    """Attention of already-rotated queries ``[F,W,Hq,S,E]`` over contiguous views
    (attention.py:24-33)."""
    if out is None:
        out = torch.empty((queries.size(1), queries.size(2), queries.size(3), values[0].size(-1)),
                          dtype=queries.dtype, device=queries.device)
    if fragment_lengths is None:
        fragment_lengths = torch.tensor([k.size(-2) for k in keys], dtype=torch.int32, device=queries.device)
    keys = [k.contiguous() for k in keys]
    values = [v.contiguous() for v in values]
    torch.ops.libdvatt.dvattn_sdpa(out, scale, locations, queries.contiguous(), fragment_lengths, keys, values)
    return out


def dvattn_rope(queries: torch.Tensor, cosines: torch.Tensor, sines: torch.Tensor, out=None):
    """Rotate ``[W,Hq,S,E]`` queries once per view -> ``[F,W,Hq,S,E]`` (attention.py:68-72)."""
    if out is None:
        out = torch.empty((cosines.size(0), queries.size(0), queries.size(1), queries.size(2), queries.size(3)),
                          dtype=queries.dtype, device=queries.device)
    torch.ops.libdvatt.dvattn_rope(out, queries, cosines, sines)
    return out


def dvattn_varlen_rope(queries: torch.Tensor, cosines: torch.Tensor, sines: torch.Tensor, out=None):
    """Rotate packed ``[T,H,E]`` queries with half-width cos/sin ``[F,T,R/2]`` -> ``[F,T,H,E]``
    (op ``dvattn_varlen_rope``, binding.cu:205-247)."""
    if out is None:
        out = torch.empty((cosines.size(0),) + tuple(queries.shape), dtype=queries.dtype, device=queries.device)
    torch.ops.libdvatt.dvattn_varlen_rope(out, queries, cosines, sines)
    return out


def dvattn_paged_sdpa(queries: torch.Tensor, locations: torch.Tensor, cosines: torch.Tensor, sines: torch.Tensor,
                      fragment_lengths: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      block_tables: torch.Tensor, scale: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Paged multi-view decode attention with fused query rotation (op
    ``dvattn_paged_sdpa``, binding.cu:151-203).  queries ``[W,Hq,S,E]`` ->
    out ``[W,Hq,S,Ev]``."""
    if out is None:
        out = torch.empty(tuple(queries.shape[:3]) + (v_cache.size(-1),), dtype=queries.dtype,
                          device=queries.device)
    torch.ops.libdvatt.dvattn_paged_sdpa(out, scale, locations, queries, cosines, sines, fragment_lengths,
                                         k_cache, v_cache, block_tables)
    return out


def dvattn_varlen_paged_sdpa(queries: torch.Tensor, locations: torch.Tensor, cosines: torch.Tensor,
                             sines: torch.Tensor, fragment_lengths: torch.Tensor, k_cache: torch.Tensor,
                             v_cache: torch.Tensor, block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor,
                             cu_seqlens_k: torch.Tensor, scale: float,
                             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Varlen (packed tokens) paged multi-view attention (op
    ``dvattn_varlen_paged_sdpa``, binding.cu:249-296).  queries ``[T,Hq,E]`` ->
    out ``[T,Hq,Ev]``."""
    if out is None:
        out = torch.empty(tuple(queries.shape[:2]) + (v_cache.size(-1),), dtype=queries.dtype,
                          device=queries.device)
    torch.ops.libdvatt.dvattn_varlen_paged_sdpa(out, scale, locations, queries, cosines, sines, fragment_lengths,
                                                k_cache, v_cache, block_tables, cu_seqlens_q, cu_seqlens_k)
    return out


def dvattn_paged_kv_append(keys: torch.Tensor, values: torch.Tensor, positions: torch.Tensor,
                           cosines: torch.Tensor, sines: torch.Tensor, k_cache: torch.Tensor,
                           v_cache: torch.Tensor, block_tables: torch.Tensor):
    """The K side of a decode step on a paged cache: rotate the new keys with the
    model's (cos, sin) and write keys and values into their pages (the reference
    rotates ``key_states`` at attention.py:304 and appends them to the sequence's
    own cache at attention.py:141-152).

    keys/values ``[W,Hkv,S,E]`` (strided views such as k_proj's output
    transposed are fine), positions ``[W,S]`` int32 logical positions in each
    sequence's token stream (negative: masked, not written), cosines/sines
    ``[W,S,R]`` / ``[S,R]`` / ``[R]`` in float32 or the model dtype, read in full
    (``apply_rotary_pos_emb``, attention.py:82-88, evaluated with PyTorch's
    rounding).  Caches ``[num_blocks, block_size, Hkv, E]`` are updated in place.
    """
    W, _, S, _ = keys.shape
    R = cosines.size(-1)
    cos = cosines.reshape((1,) * (3 - cosines.dim()) + tuple(cosines.shape)) if cosines.dim() < 3 else cosines
    sin = sines.reshape((1,) * (3 - sines.dim()) + tuple(sines.shape)) if sines.dim() < 3 else sines
    cos = cos.expand(W, S, R)
    sin = sin.expand(W, S, R)
    torch.ops.libdvatt.dvattn_paged_kv_append(k_cache, v_cache, block_tables, positions, keys, values, cos, sin)
    return k_cache, v_cache


def merge_caches_paged(source_keys: torch.Tensor, source_values: torch.Tensor, offset_cos: torch.Tensor,
                       offset_sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       block_tables: torch.Tensor, positions: torch.Tensor):
    """``merge_caches`` (attention.py:245-251) into a paged target: the source
    keys ``[1,Hkv,L,E]`` are re-rotated by the target's length (one cos/sin row,
    ``offset_cos``/``offset_sin`` ``[R]``: the rotary embedding at that length)
    and written with the source values at ``positions`` ``[1,L]`` (the target's
    next L logical positions)."""
    return dvattn_paged_kv_append(source_keys, source_values, positions, offset_cos.reshape(-1),
                                  offset_sin.reshape(-1), k_cache, v_cache, block_tables)


def dvattn_view_metadata(fragment_lengths: torch.Tensor, order: torch.Tensor, num_new_tokens: int,
                         inv_freq: torch.Tensor, attention_scaling: float = 1.0,
                         round_to: Optional[torch.dtype] = None):
    """Per-view locations and query cos/sin for a decode step, on the device
    (attention.py:158-186).

    fragment_lengths ``[F]`` int32: segment lengths including the new tokens;
    order ``[W,F]`` int32: sequence w's segments in its own order (view indices,
    its own segment last); inv_freq ``[R/2]`` float32: the model's rotary inverse
    frequencies (``model.rotary_emb.inv_freq``).  Returns ``(locations [F,W,S]
    int32, cosines [F,W,S,R], sines [F,W,S,R])`` float32, ready for
    ``dvattn_paged_sdpa`` / ``dvattn_fused``.  ``round_to`` rounds cos/sin through
    the model dtype, as the reference's rotary call does.

    Positions are sums of the lengths: the tables are for caches that hold every row.
    Of a cache that was cut, ``dvattn_tree_metadata`` on a chain (parents -1, 0, 1, ...)
    gives them with ``dropped``; token s then sees ``locations + 1 + s`` of its own view.
    """
    F = fragment_lengths.numel()
    W = order.size(0)
    R = 2 * inv_freq.numel()
    dev = fragment_lengths.device
    loc = torch.empty((F, W, num_new_tokens), dtype=torch.int32, device=dev)
    cos = torch.empty((F, W, num_new_tokens, R), dtype=torch.float32, device=dev)
    sin = torch.empty_like(cos)
    torch.ops.libdvatt.dvattn_view_metadata(loc, cos, sin, fragment_lengths, order, inv_freq,
                                            float(attention_scaling), round_to)
    return loc, cos, sin


def dvattn_tree_metadata(fragment_lengths: torch.Tensor, order: torch.Tensor, parents: torch.Tensor,
                         inv_freq: torch.Tensor, attention_scaling: float = 1.0,
                         round_to: Optional[torch.dtype] = None, dropped: Optional[torch.Tensor] = None,
                         committed: Optional[torch.Tensor] = None):
    """Metadata of a step in which every sequence drafts a tree of up to S tokens:
    ``dvattn_view_metadata`` with positions that follow the nodes' depths.

    parents ``[W,S]`` int32: -1 for a child of the committed tokens, the index of
    an earlier node (``0 .. s-1``), or anything else (-2, say) for an absent node:
    the padding of a smaller tree; nodes below an absent one are absent too.  The
    drafted rows are the last S of each sequence's own view (the last of its
    ``order [W,F]``): fragment_lengths ``[F]`` count them.  Returns

    * ``locations [F,W,S]``: the committed keys of each view, -1 for absent nodes;
    * ``cosines``, ``sines`` ``[F,W,S,R]`` at the position (committed tokens from the
      view to the end of the sequence's order) + (the node's depth);
    * ``tree_views [W]``, ``tree_rows [W]``: each sequence's own view, and the row of
      its page stream that holds node 0 (node s is appended at ``tree_rows + s``).

    The last four and the first are ``dvattn_tree_paged_sdpa``'s arguments.  Another
    sequence's drafted nodes are neither seen nor counted.  S and F are at most 4096.

    A cache that was cut (``dvattn_kv_select``, ``dvattn_paged_kv_compact``) holds
    fewer rows than its sequence has seen tokens, and kept keys keep the rotation of
    their own positions: ``dropped [W,F]`` int32 are the tokens of each view that the
    sequence no longer holds.  They count for the positions and for nothing else.
    Without them the tables are for caches that hold every row.

    Sequences that share a view index share its length, but after their first accepted
    paths they hold different numbers of rows: ``committed [W,F]`` int32 are then the
    committed rows of each view (0 and up) in place of those its length gives, and
    fragment_lengths are at least the most of them and S.
    """
    return torch.ops.libdvatt.dvattn_tree_metadata(fragment_lengths, order, parents, inv_freq,
                                                   float(attention_scaling), round_to, dropped, committed)


def dvattn_tree_paged_sdpa(queries: torch.Tensor, locations: torch.Tensor, cosines: torch.Tensor,
                           sines: torch.Tensor, fragment_lengths: torch.Tensor, k_cache: torch.Tensor,
                           v_cache: torch.Tensor, block_tables: torch.Tensor, parents: torch.Tensor,
                           tree_views: torch.Tensor, tree_rows: torch.Tensor, scale: float,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dvattn_paged_sdpa`` for the nodes of drafted token trees.  Node s of sequence
    w (queries ``[W,Hq,S,E]``) sees the keys its ``locations`` allow and, in view
    ``tree_views[w]``, the rows ``tree_rows[w] + j`` of the page stream for j = s and
    its ancestors by ``parents [W,S]`` (see ``dvattn_tree_metadata``).  Absent nodes
    give zeros.  Out ``[W,Hq,S,Ev]``."""
    if out is None:
        out = torch.empty(tuple(queries.shape[:3]) + (v_cache.size(-1),), dtype=queries.dtype,
                          device=queries.device)
    torch.ops.libdvatt.dvattn_tree_paged_sdpa(out, scale, locations, queries, cosines, sines, fragment_lengths,
                                              k_cache, v_cache, block_tables, parents, tree_views, tree_rows)
    return out


def dvattn_paged_key_mass(mass: Optional[torch.Tensor], queries: torch.Tensor, locations: torch.Tensor,
                          cosines: torch.Tensor, sines: torch.Tensor, fragment_lengths: torch.Tensor,
                          k_cache: torch.Tensor, block_tables: torch.Tensor, scale: float, decay: float = 1.0,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention weight that every cached key receives: ``out = decay * mass +`` the
    softmax weights of ``dvattn_paged_sdpa`` on the same arguments, summed over the
    tokens and the 16 query heads of each KV head.

    mass ``[W,Hkv,capacity]`` float32, by row of each sequence's page stream (views
    one after the other); ``out`` defaults to ``mass`` itself (accumulation in place).
    With ``decay=0`` mass is not read and may be None if ``out`` is given.  Rows at or
    past the capacity take part in the softmax and are not stored.  Lengths below zero
    count as 0.

    Every query votes, and its locations say all that it sees: the tables of a tree step
    would leave out the drafted rows.  The weights of its accepted tokens are those of
    the causal chain that they are once ``dvattn_paged_kv_compact`` has kept them."""
    if out is None:
        out = mass
    if out is None:
        raise ValueError("dvattn_paged_key_mass: mass or out must be given")
    torch.ops.libdvatt.dvattn_paged_key_mass(out, mass, float(decay), scale, locations, queries, cosines, sines,
                                             fragment_lengths, k_cache, block_tables)
    return out


def dvattn_kv_select(mass: torch.Tensor, first_rows: torch.Tensor, lengths: torch.Tensor, budget: int,
                     keep_first: int = 0, keep_last: int = 0, rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The rows of a cache worth keeping, ``[W,Hkv,budget]`` int32, ascending and
    relative to ``first_rows [W]``: of the ``lengths[w]`` rows from there on all if
    they fit the budget (then -1), else the first ``keep_first``, the last
    ``keep_last`` and the heaviest others by ``mass [W,Hkv,capacity]`` (ties to the
    lowest row, NaN lightest).  ``dvattn_paged_kv_compact`` moves them together."""
    if rows is None:
        rows = torch.empty(tuple(mass.shape[:2]) + (budget,), dtype=torch.int32, device=mass.device)
    elif rows.size(-1) != budget:
        raise ValueError(f"dvattn_kv_select: rows hold {rows.size(-1)} entries, budget {budget}")
    torch.ops.libdvatt.dvattn_kv_select(rows, mass, first_rows, lengths, keep_first, keep_last)
    return rows


def dvattn_paged_kv_compact(rows: torch.Tensor, first_rows: torch.Tensor, k_cache: torch.Tensor,
                            v_cache: torch.Tensor, block_tables: torch.Tensor, mass: Optional[torch.Tensor] = None,
                            lengths: Optional[torch.Tensor] = None):
    """Move kept rows of a paged cache together, in place: row ``first_rows[w] + i``
    takes the keys and values of row ``first_rows[w] + rows[w,h,i]`` wherever
    ``rows[w,h,i] >= i`` (and ``< lengths[w]`` if given); other rows stay.

    rows ``[W,Hkv,N]`` int32 (``dvattn_kv_select``), or ``[W,1,N]`` for all KV heads
    alike: the accepted path of a drafted tree, with ``first_rows = tree_rows``.
    ``mass [W,Hkv,capacity]`` moves along (needs lengths); entries of the range's
    rows that nothing moves into become 0.  The caches may be strided views as in
    ``dvattn_paged_kv_append``, and may not share rows.  The moved rows' pages must not be named twice in
    ``block_tables``: pages that sequences or segments share lie before first_rows.
    Positions of the kept keys do not change (their rotation stays valid); the
    caller's locations and lengths count rows from here on, and the queries' positions
    have to count the rows that went (``dropped`` of ``dvattn_tree_metadata``)."""
    torch.ops.libdvatt.dvattn_paged_kv_compact(k_cache, v_cache, block_tables, rows, first_rows, lengths, mass)
    return k_cache, v_cache


def dvattn_block_tables(lengths: torch.Tensor, new_tokens: torch.Tensor, block_tables: torch.Tensor,
                        free_pages: torch.Tensor, free_count: torch.Tensor, block_size: int, max_tokens: int,
                        in_place: bool = False):
    """Where a step's tokens go in a paged cache, on the device, from request lengths.

    lengths ``[W]`` int32: tokens that each sequence holds; new_tokens ``[W]`` int32:
    tokens it adds in this step (0: none; negative: the sequence has ended and gives its
    pages back).  block_tables ``[W,max_blocks]`` int32 are extended in place by the
    pages that the new tokens need, taken from free_pages ``[num_blocks]`` int32, a stack
    whose first ``free_count [1]`` int32 entries are the free pages.  Returns

    * ``cu_seqlens [W+1]``: the packed tokens' bounds, sequence after sequence;
    * ``starts [W]``: the position of each sequence's first new token; -1 for one that has
      ended, or was refused: the stack, its table row or the ``max_tokens`` packed tokens
      have no room for it.  A refused sequence takes no page and its length stays;
    * ``positions [max_tokens]`` int32 and ``slots [max_tokens]`` int64 of the packed
      tokens (slot = page * block_size + row), -1 for tokens of refused sequences and
      behind the last;
    * ``lengths [W]`` and ``free_count [1]`` after the step: new tensors, or with
      ``in_place`` the ones given (a captured step then carries its state on).

    ``slots`` are ``dvattn_paged_kv_append_q8``'s; ``positions[None]`` are locations of
    the varlen operators with one view.  Pages that an ending sequence holds may not be
    shared.  At most 8192 sequences."""
    lengths_out = lengths if in_place else torch.empty_like(lengths)
    count_out = free_count if in_place else torch.empty_like(free_count)
    cu, starts, positions, slots = torch.ops.libdvatt.dvattn_block_tables(
        block_tables, free_pages, lengths_out, count_out, lengths, new_tokens, free_count, block_size, max_tokens)
    return cu, starts, positions, slots, lengths_out, count_out


def dvattn_paged_kv_append_q8(keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor, cosines: torch.Tensor,
                              sines: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                              k_scales: torch.Tensor, v_scales: torch.Tensor):
    """``dvattn_paged_kv_append`` into a cache held in 8 bits: rotated keys and values are
    rounded to E4M3 under a power of two for each page and KV head.

    keys/values ``[T,Hkv,E]`` (packed tokens) or ``[W,Hkv,S,E]``, strided views alike;
    slots ``[T]`` or ``[W,S]`` int64: page * block_size + row (negative: not written), as
    ``dvattn_block_tables`` gives them; cosines/sines ``[T,R]`` / ``[R]`` or ``[W,S,R]`` /
    ``[S,R]`` / ``[R]`` in float32 or the model dtype.  Caches
    ``[num_blocks,block_size,Hkv,E]`` float8_e4m3fn (or uint8) and scales
    ``[num_blocks,Hkv]`` float8_e8m0fnu (or uint8 exponents) are updated in place; all
    cleared to zero they are an empty cache.

    A page takes the smallest power of two that holds the largest element written, or
    keeps its own if that is larger; rows that it holds under a smaller one are
    rounded again.  Writing row 0 of a page starts it anew: what its other rows held
    before is gone.  A slot given more than once holds its last token."""
    if keys.dim() == 3:
        keys, values, slots = keys.transpose(0, 1)[None], values.transpose(0, 1)[None], slots[None]
    W, _, S, _ = keys.shape
    R = cosines.size(-1)
    cos = cosines.reshape((1,) * (3 - cosines.dim()) + tuple(cosines.shape)) if cosines.dim() < 3 else cosines
    sin = sines.reshape((1,) * (3 - sines.dim()) + tuple(sines.shape)) if sines.dim() < 3 else sines
    torch.ops.libdvatt.dvattn_paged_kv_append_q8(k_cache, v_cache, k_scales, v_scales, slots, keys, values,
                                                 cos.expand(W, S, R), sin.expand(W, S, R))
    return k_cache, v_cache, k_scales, v_scales


def dvattn_paged_sdpa_q8(queries: torch.Tensor, locations: torch.Tensor, cosines: torch.Tensor, sines: torch.Tensor,
                         fragment_lengths: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         k_scales: torch.Tensor, v_scales: torch.Tensor, block_tables: torch.Tensor, scale: float,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dvattn_paged_sdpa`` over a cache held in 8 bits (``dvattn_paged_kv_append_q8``):
    the same queries, views and tables, in float32, float16 or bfloat16, with the caches'
    scales.  queries ``[W,Hq,S,E]`` -> out ``[W,Hq,S,Ev]``."""
    if out is None:
        out = torch.empty(tuple(queries.shape[:3]) + (v_cache.size(-1),), dtype=queries.dtype,
                          device=queries.device)
    torch.ops.libdvatt.dvattn_paged_sdpa_q8(out, scale, locations, queries, cosines, sines, fragment_lengths,
                                            k_cache, v_cache, k_scales, v_scales, block_tables)
    return out


def dvattn_varlen_paged_sdpa_q8(queries: torch.Tensor, locations: torch.Tensor, cosines: torch.Tensor,
                                sines: torch.Tensor, fragment_lengths: torch.Tensor, k_cache: torch.Tensor,
                                v_cache: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
                                block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor,
                                scale: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dvattn_varlen_paged_sdpa`` over a cache held in 8 bits.  queries ``[T,Hq,E]`` ->
    out ``[T,Hq,Ev]``; cu_seqlens_k is not read."""
    if out is None:
        out = torch.empty(tuple(queries.shape[:2]) + (v_cache.size(-1),), dtype=queries.dtype,
                          device=queries.device)
    torch.ops.libdvatt.dvattn_varlen_paged_sdpa_q8(out, scale, locations, queries, cosines, sines, fragment_lengths,
                                                   k_cache, v_cache, k_scales, v_scales, block_tables, cu_seqlens_q,
                                                   cu_seqlens_k)
    return out


def dvattn_sdpa_pt(queries: torch.Tensor, locations: torch.Tensor, keys: list, values: list,
                   scale: float, return_intermediate_results: bool = False):
    """Pure-PyTorch attention over already-rotated queries and contiguous views,
    for testing and debugging; the reference's helper of the same name and
    contract (attention.py:36-65).  No operator of this package calls it.

    queries ``[F,W,Hq,S,E]`` (rotated per view), locations ``[F,W,S]``,
    keys[f] / values[f] ``[B,Hkv,L_f,E|Ev]`` or ``[Hkv,L_f,E|Ev]`` (B = 1
    broadcasts over the W sequences).  Key ``l`` of view ``f`` is visible to
    query ``(w, s)`` iff ``l <= locations[f, w, s]``; one fp32 softmax of
    ``scale * q.k`` runs over the keys of all views.  Returns the output in
    ``queries.dtype``; with ``return_intermediate_results``, the fp32 output
    ``[W,Hq,S,Ev]``, the masked unscaled scores and the softmax weights
    ``[W,Hq,S,sum_f L_f]``.  A query that sees no key gets NaN here (the HIP
    operators write zeros, as the reference's kernels do).

    GQA without replicating K/V: the 16 query heads of a KV head are viewed as
    16*S query rows of that head.  The views' scores fill one preallocated
    key axis, and visibility is one comparison of every key's in-view position
    against the query's location in that key's view.
    """
    F, W, Hq, S, E = queries.shape
    Hkv = keys[0].shape[-3]
    G = Hq // Hkv
    Ev = values[0].shape[-1]
    dev = queries.device
    lens = [int(k.shape[-2]) for k in keys]
    total = sum(lens)
    view_of = torch.repeat_interleave(torch.arange(F, device=dev), torch.tensor(lens, device=dev))
    pos_in_view = torch.cat([torch.arange(n, device=dev) for n in lens]) if total else \
        torch.zeros(0, dtype=torch.long, device=dev)

    scores = torch.empty((W, Hkv, G * S, total), dtype=torch.float32, device=dev)
    v_all = torch.empty((W, Hkv, total, Ev), dtype=torch.float32, device=dev)
    start = 0
    for f, n in enumerate(lens):
        q_rows = queries[f].to(torch.float32).reshape(W, Hkv, G * S, E)
        scores[..., start:start + n] = q_rows @ keys[f].to(torch.float32).transpose(-1, -2)
        v_all[:, :, start:start + n] = values[f].to(torch.float32)
        start += n
    scores = scores.view(W, Hq, S, total)
    hidden = pos_in_view > locations.to(device=dev, dtype=torch.long)[view_of].permute(1, 2, 0)  # [W,S,total]
    scores.masked_fill_(hidden[:, None], float("-inf"))
    weights = torch.softmax(scores * scale, dim=-1)
    result = (weights.view(W, Hkv, G * S, total) @ v_all).view(W, Hq, S, Ev)
    if return_intermediate_results:
        return result, scores, weights
    return result.to(queries.dtype)


def rotate_half(x):
    """Rotates half the hidden dims of the input (attention.py:75-79)."""
    x1 = x[..., : x.shape[-1] // 2]
    x2 = x[..., x.shape[-1] // 2:]
    return torch.cat((-x2, x1), dim=-1)


def apply_rotary_pos_emb(x, cos, sin, unsqueeze_dim=1):
    """Partial RoPE on the first ``cos.shape[-1]`` dims (attention.py:82-88)."""
    cos = cos.unsqueeze(unsqueeze_dim)
    sin = sin.unsqueeze(unsqueeze_dim)
    rotary_dim = cos.shape[-1]
    x_rot, x_pass = x[..., :rotary_dim], x[..., rotary_dim:]
    x_rot_emb = (x_rot * cos) + (rotate_half(x_rot) * sin)
    return torch.cat((x_rot_emb, x_pass), dim=-1).to(x.dtype)


__all__ = [
    "dvattn_fused", "dvattn_sdpa", "dvattn_rope", "dvattn_varlen_rope", "dvattn_paged_sdpa",
    "dvattn_varlen_paged_sdpa", "dvattn_sdpa_pt", "rotate_half", "apply_rotary_pos_emb",
    "dvattn_paged_kv_append", "merge_caches_paged", "dvattn_view_metadata", "dvattn_tree_metadata",
    "dvattn_tree_paged_sdpa", "dvattn_paged_key_mass", "dvattn_kv_select", "dvattn_paged_kv_compact",
    "dvattn_block_tables", "dvattn_paged_kv_append_q8", "dvattn_paged_sdpa_q8", "dvattn_varlen_paged_sdpa_q8",
]
