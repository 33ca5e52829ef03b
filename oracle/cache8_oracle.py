"""64-bit CPU restatements of the operators around 8-bit caches
(dvattn_block_tables, dvattn_paged_kv_append_q8, dvattn_paged_sdpa_q8,
dvattn_varlen_paged_sdpa_q8), written from their definitions, sequence by
sequence and slot by slot.  Test infrastructure only.

The rotated key (rounded to its type as PyTorch evaluates it) and the rotated
query are part of the definitions; everything after them is float64.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from oracle import tree_cache_oracle as TO

GQA = 16
F64 = torch.float64


def tables(lengths, new_tokens, block_tables, free_pages, free_count, bs, max_tokens):
    """(cu, starts, positions, slots, lengths, count, block_tables, free_pages) as lists and arrays."""
    bt, pages = np.asarray(block_tables).astype(np.int64), [int(x) for x in free_pages]
    W, width = bt.shape
    P = len(pages)
    room = min(width * bs, 2 ** 31 - 1)
    count = min(max(int(free_count), 0), P)
    held = [min(max(int(x), 0), room) for x in lengths]
    new = [int(x) for x in new_tokens]
    for w in range(W):
        if new[w] < 0:
            for b in range(-(-held[w] // bs)):
                if count < P:
                    pages[count] = int(bt[w, b])
                    count += 1
            held[w] = 0
    left, stopped = count, False
    cu, starts, after = [0], [], []
    positions, slots = [-1] * max_tokens, [-1] * max_tokens
    for w in range(W):
        n = max(new[w], 0)
        need = -(-(held[w] + n) // bs) - -(-held[w] // bs)
        ok = held[w] + n <= room and cu[-1] + n <= max_tokens
        if ok and need:
            stopped = stopped or need > left
            ok = not stopped
        if ok:
            for j in range(need):
                left -= 1
                bt[w, -(-held[w] // bs) + j] = pages[left]
            for j in range(n):
                p = held[w] + j
                page = int(bt[w, p // bs])
                positions[cu[-1] + j] = p
                slots[cu[-1] + j] = page * bs + p % bs if 0 <= page < P else -1
        starts.append(held[w] if ok and new[w] >= 0 else -1)
        after.append(held[w] + n if ok else held[w])
        cu.append(min(cu[-1] + n, 2 ** 31 - 1))
    return cu, starts, positions, slots, after, left, bt, pages


def e4m3(x):
    """float64 numbers of at most 448 rounded to E4M3, ties to even; NaN stays."""
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(np.nan_to_num(x)), 1e-300))), -6) - 3)
    return np.rint(x / step) * step


def bytes_of(values):
    """E4M3 bytes of E4M3 numbers (NaN: 0x7f)."""
    b = torch.from_numpy(np.nan_to_num(values, nan=0.0)).float().to(torch.float8_e4m3fn).view(torch.uint8)
    b[torch.from_numpy(np.isnan(values))] = 0x7f
    return b


def values_of(cache):
    return cache.view(torch.uint8).view(torch.float8_e4m3fn).float().double()


def rotated_keys(keys, cos, sin):
    """keys [W,Hkv,S,E] rotated by cos/sin [W,S,R] as apply_rotary_pos_emb evaluates it, in keys' type."""
    from dvattention_amd.attention import apply_rotary_pos_emb
    return apply_rotary_pos_emb(keys, cos, sin)


def exponent(amax):
    """The smallest b >= 1 with amax <= 448 * 2^(b - 127)."""
    b = 1
    if amax > 0:
        b = max(1, math.frexp(amax)[1] - 9 + 127)
        while amax > 448.0 * 2.0 ** (b - 127):
            b += 1
        while b > 1 and amax <= 448.0 * 2.0 ** (b - 128):
            b -= 1
    return b


def append(k_cache, v_cache, k_scales, v_scales, slots, keys, values, cos, sin):
    """New (k_cache, v_cache, k_scales, v_scales): bytes (uint8)."""
    P, bs, Hkv, _ = k_cache.shape
    held = {}  # page -> {row: (w, s)}, the last token of a slot
    for w in range(slots.shape[0]):
        for s in range(slots.shape[1]):
            at = int(slots[w, s])
            if 0 <= at < P * bs:
                held.setdefault(at // bs, {})[at % bs] = (w, s)
    out = []
    for x, cache, scales in ((rotated_keys(keys, cos, sin), k_cache, k_scales), (values, v_cache, v_scales)):
        x = x.double()
        if keys.dtype == torch.float16:
            x = torch.where(x.isinf(), x, x.clamp(-61440.0, 61440.0))
        x = torch.where(x.isinf(), math.nan, x)
        new, b8 = cache.view(torch.uint8).clone(), scales.view(torch.uint8).clone()
        for page, rows in held.items():
            for h in range(Hkv):
                mine = torch.stack([x[w, h, s] for w, s in rows.values()])
                b = exponent(float(mine.nan_to_num(0.0).abs().max()))
                old = int(b8[page, h])
                if 0 not in rows and old != 255:
                    if b > old:
                        rest = [r for r in range(bs) if r not in rows]
                        v = values_of(new[page, rest, h]).numpy()
                        v = v * 2.0 ** (old - b) if old else np.zeros_like(v)
                        new[page, rest, h] = bytes_of(e4m3(v))
                    b = max(b, old)
                b8[page, h] = b
                new[page, list(rows), h] = bytes_of(e4m3(mine.numpy() * 2.0 ** (127 - b)))
        out += [new, b8]
    return out[0], out[2], out[1], out[3]


def dequantised(cache, scales):
    """float64 [P,bs,Hkv,E]; the elements of an empty page (0) are zeros whatever its bytes are."""
    b = scales.view(torch.uint8).double()[:, None, :, None]
    f = torch.where(b == 255, math.nan, torch.exp2(b - 127))
    return torch.where(b == 0, 0.0, values_of(cache) * f)


def sdpa(scale, locations, queries, cosines, sines, fragment_lengths, k_cache, v_cache, k_scales, v_scales,
         block_tables):
    """(out, sum of weight * |v|, spread): float64 [W,Hq,S,Ev] twice, and [W,Hq,S,1]."""
    k, v = dequantised(k_cache, k_scales), dequantised(v_cache, v_scales)
    W, Hq, S, _ = queries.shape
    out = torch.zeros(W, Hq, S, v.shape[3], dtype=F64)
    size, spread = torch.zeros_like(out), torch.zeros(W, Hq, S, 1, dtype=F64)
    for w, h, s, keys, p, sp in TO.attention_rows(scale, locations, queries, cosines, sines, fragment_lengths, k,
                                                  block_tables):
        if keys:
            rows = v[[x[2] for x in keys], [x[3] for x in keys], h]
            out[w, GQA * h:GQA * (h + 1), s] = p @ rows
            size[w, GQA * h:GQA * (h + 1), s] = p @ rows.abs()
            spread[w, GQA * h:GQA * (h + 1), s] = sp
    return out, size, spread


def varlen_sdpa(scale, locations, queries, cosines, sines, fragment_lengths, k_cache, v_cache, k_scales, v_scales,
                block_tables, cu_seqlens_q):
    """The same for packed tokens: [T,Hq,Ev] twice, and [T,Hq,1].  Token t is of the first
    sequence i with t < cu_seqlens_q[i + 1], of sequence 0 if there is none."""
    T = queries.shape[0]
    parts = []
    for t in range(T):
        w = next((i for i in range(len(cu_seqlens_q) - 1) if t < int(cu_seqlens_q[i + 1])), 0)
        full = [torch.cat([x[:, t], x[:, t]], dim=-1)[:, None, None] for x in (cosines, sines)]
        parts.append([x[0, :, 0] for x in sdpa(scale, locations[:, t, None, None], queries[t][None, :, None], *full,
                                               fragment_lengths, k_cache, v_cache, k_scales, v_scales,
                                               block_tables[w:w + 1])])
    return tuple(torch.stack([p[i] for p in parts]) for i in range(3))
