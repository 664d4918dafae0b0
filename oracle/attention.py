"""The attention half of the decoder layer in 64 bits, one row at a time.

Restates transformers models/gpt_oss/modeling_gpt_oss.py (apply_rotary_pos_emb;
eager_attention_forward with its sinks and sliding window) over a paged cache,
and the cache's upkeep, from the formulas alone.  CPU, for tests.
"""

from __future__ import annotations

import math

import torch

NEG = -math.inf


def rotary(x, table, positions, interleaved=False, inverse=False):
    """x [..., heads, D] f64 turned; positions x.shape[:-2]; rows of a position outside the table are zero."""
    x, table = x.double(), table.double()
    rot = 2 * table.shape[1]
    out = x.clone()
    flat, fpos = out.view(-1, *x.shape[-2:]), positions.reshape(-1).tolist()
    for n, p in enumerate(fpos):
        if not 0 <= p < table.shape[0]:
            flat[n] = 0
            continue
        for i in range(rot // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
            c, s = table[p, i, 0], table[p, i, 1] * (-1 if inverse else 1)
            u, v = flat[n, :, a].clone(), flat[n, :, b].clone()
            flat[n, :, a], flat[n, :, b] = u * c - v * s, v * c + u * s
    return out


def slot(cache, page_table, b, j):
    """Row of slot j of sequence b: [heads, D]."""
    page = cache.shape[1]
    return cache[int(page_table[b, j // page]), j % page]


def sees(n, T, pos, mask, window, t):
    """Slots that drafted token t of a sequence with n committed slots attends."""
    if pos[t] < 0:
        return []
    floor = max(pos[t], n) - window if window else -math.inf
    seen = [j for j in range(n) if j > floor]
    for u in range(T):
        on = u <= t if mask is None else bool(mask[t][u])
        if on and pos[u] >= 0 and pos[u] > floor:
            seen.append(n + u)
    return seen


def tree_attention(q, k_cache, v_cache, page_table, lens, positions, mask=None, sinks=None, window=0, scale=None):
    """(out, lse, spread) in f64; spread = sum of weight * |v|, which bounds the rounding of the weights."""
    B, T, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    spread = torch.zeros_like(out)
    lse = torch.full((B, T, Hq), NEG, dtype=torch.float64)
    for b in range(B):
        n, pos = int(lens[b]), positions[b].tolist()
        m = None if mask is None else (mask if mask.dim() == 2 else mask[b]).tolist()
        for t in range(T):
            if pos[t] < 0:
                continue
            seen = sees(n, T, pos, m, window, t)
            if seen:
                k = torch.stack([slot(k_cache, page_table, b, j) for j in seen]).double()
                v = torch.stack([slot(v_cache, page_table, b, j) for j in seen]).double()
            for h in range(Hq):
                x = k[:, h // G] @ q[b, t, h].double() * scale if seen else torch.zeros(0, dtype=torch.float64)
                if sinks is not None:
                    x = torch.cat([x, sinks[h].double().reshape(1)])
                if x.numel() == 0 or bool((x == NEG).all()):
                    continue
                z = x.logsumexp(0)
                lse[b, t, h] = z
                if seen:
                    w = (x - z).exp()[: len(seen)]
                    out[b, t, h] = w @ v[:, h // G]
                    spread[b, t, h] = w @ v[:, h // G].abs()
    return out, lse, spread


def kv_scores(scores, q, lse, k_cache, page_table, lens, accepted=None, scale=None):
    B, T, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = scores.double().clone()
    for b in range(B):
        path = range(T) if accepted is None else accepted[b].tolist()
        for i, u in enumerate(path):
            if not 0 <= u < T:
                continue
            for h in range(Hq):
                if lse[b, u, h] == NEG:
                    continue
                for j in range(min(int(lens[b]) + i + 1, scores.shape[2])):
                    x = slot(k_cache, page_table, b, j)[h // (Hq // Hkv)].double() @ q[b, u, h].double() * scale
                    out[b, h // (Hq // Hkv), j] += math.exp(x - lse[b, u, h].double())
    return out


def evict(scores, lens, budget, first, last):
    """Kept slots of every (sequence, head), ascending; NaN below every number, ties to the lowest slot."""
    kept = []
    for b in range(scores.shape[0]):
        n = int(lens[b])
        row = []
        for h in range(scores.shape[1]):
            s = scores[b, h].tolist()

            def rank(j):
                safe = j < first or j >= n - last
                value = NEG if s[j] != s[j] else s[j]
                return (0 if safe else 1, 1 if s[j] != s[j] and not safe else 0, 0.0 if safe else -value, j)

            row.append(sorted(sorted(range(n), key=rank)[:budget]))
        kept.append(row)
    return kept
