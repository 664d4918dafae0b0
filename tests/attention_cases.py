"""Small paged caches and drafted trees for the attention tests."""

import torch


def pages_for(n, page):
    return max(1, -(-n // page))


def make_cache(lens, T, Hkv, D, page, seed, head_major=False, spare=2, dtype=torch.bfloat16, fill=None):
    """CPU cache of randomly ordered pages; slots of no sequence hold `fill` (NaN by default)."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    P = pages_for(max(lens) + T, page)
    total = B * P + spare
    table = torch.randperm(total, generator=g)[: B * P].reshape(B, P).to(torch.int32)
    fill = float("nan") if fill is None else fill
    shape = (total, Hkv, page, D) if head_major else (total, page, Hkv, D)
    out = []
    for _ in range(2):
        c = torch.full(shape, fill, dtype=dtype)
        c = c.transpose(1, 2) if head_major else c
        for b, n in enumerate(lens):
            for j in range(n + T):
                c[int(table[b, j // page]), j % page] = torch.randn(Hkv, D, generator=g).to(dtype)
        out.append(c)
    return out[0], out[1], table, torch.tensor(lens, dtype=torch.int32), g


def make_tree(B, T, lens, g, unused=0):
    """Random trees: mask [B, T, T] and positions [B, T] (the last `unused` drafts of odd sequences off)."""
    mask = torch.zeros(B, T, T, dtype=torch.bool)
    pos = torch.zeros(B, T, dtype=torch.int32)
    for b in range(B):
        for t in range(T):
            p = int(torch.randint(-1, t, (1,), generator=g)) if t else -1
            depth = 0
            if p >= 0:
                mask[b, t] = mask[b, p]
                depth = int(pos[b, p]) - lens[b] + 1
            mask[b, t, t] = True
            pos[b, t] = lens[b] + depth
        if b % 2 and unused:
            pos[b, T - unused:] = -1
    return mask, pos


def poison_unused(cache, table, lens, pos):
    """The slots of drafts not in use hold NaN: nothing may read them."""
    page = cache.shape[1]
    for b in range(pos.shape[0]):
        for t in range(pos.shape[1]):
            if pos[b, t] < 0:
                j = int(lens[b]) + t
                cache[int(table[b, j // page]), j % page] = float("nan")
