"""The attention half of a decoder layer around the MoE layer, as cases to measure.

Four operators, each with a plain form in elementary torch operations (32 bits,
one rounding at the end) and the call that a user makes of the framework:

``rotary``  rotary positions of queries and keys from a cos/sin table, both
            layouts, forward with its gradient (training), and the serving form
            that also writes the new keys and values into a paged cache;
``tree``    attention of a tree of drafted tokens over a paged key/value cache
            (one drafted token is ordinary decoding), with sinks and a window;
``mass``    the attention weight each cached key received, added to its score;
``evict``   the keys of highest score, with protected first and last ones, kept
            and compacted into other pages of the cache.

Layouts: q [B, T, Hq, D]; cache [pages, page, Hkv, D] (any strides with the last
dimension contiguous); page_table [B, P] int32; slot j of a sequence is row
j % page of page page_table[b, j // page]; the drafted tokens of a sequence sit
at slots cache_lens[b] + t.  A position below zero marks a draft slot not in use.
"""

import math

import torch

own = False


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one training step's rotation of 8192 tokens, forward and backward
        dict(name="rotary_train", op="rotary", dtype="bf16", tokens=8192, Hq=64, Hkv=8, D=64, rot=64,
             interleaved=False, max_pos=131072),
        # 32-bit heads rotated in their first half only, interleaved pairs, an odd number of tokens
        dict(name="rotary_partial_f32", op="rotary", dtype="f32", tokens=1531, Hq=12, Hkv=3, D=96, rot=48,
             interleaved=True, max_pos=40000),
        # a decoding step of many sequences: rotate, and append the new key and value to the cache
        dict(name="append_decode", op="append", B=128, T=1, Hq=64, Hkv=8, D=64, rot=64, interleaved=False,
             page=16, length=1000, head_major=False, unused=0, max_pos=8192),
        # one sequence, one token, a short cache: latency
        dict(name="decode_one", op="tree", B=1, T=1, Hq=64, Hkv=8, D=64, page=16, length=500, ragged=False,
             head_major=False, window=0, sinks=True, tree="chain", unused=0),
        # ordinary batched decoding over ragged lengths
        dict(name="decode_batch", op="tree", B=64, T=1, Hq=64, Hkv=8, D=64, page=64, length=8192, ragged=True,
             head_major=True, window=0, sinks=True, tree="chain", unused=0),
        # a windowed layer: small trees, odd heads and pages, empty and one-key caches, unused draft slots
        dict(name="window_odd", op="tree", B=7, T=13, Hq=20, Hkv=4, D=80, page=24, length=4001, ragged=True,
             head_major=False, window=128, sinks=True, tree="each", unused=4),
        # small trees over a long context
        dict(name="tree_long", op="tree", B=2, T=16, Hq=64, Hkv=8, D=64, page=64, length=131072, ragged=False,
             head_major=False, window=0, sinks=False, tree="shared", unused=0),
        # wide trees: many drafted rows to each key
        dict(name="tree_wide", op="tree", B=8, T=64, Hq=32, Hkv=8, D=128, page=64, length=16384, ragged=True,
             head_major=False, window=0, sinks=False, tree="each", unused=9),
        # scores of the cached keys after a decoding step of a batch
        dict(name="mass_decode", op="mass", B=32, T=1, A=1, Hq=64, Hkv=8, D=64, page=16, length=8192,
             ragged=True, head_major=False),
        # after a verification step: the accepted path of each tree
        dict(name="mass_accepted", op="mass", B=3, T=24, A=7, Hq=32, Hkv=4, D=128, page=128, length=30011,
             ragged=True, head_major=True),
        # long caches cut to a quarter
        dict(name="evict_long", op="evict", B=8, Hkv=8, D=64, page=64, length=32768, ragged=False,
             head_major=False, budget=8192, first=4, last=1024),
        # short, odd caches, some of them within the budget already
        dict(name="evict_odd", op="evict", B=3, Hkv=4, D=80, page=24, length=1500, ragged=True,
             head_major=True, budget=511, first=3, last=100),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "tree", "tree", "tree", "mass", "evict"])
    hkv = rng.choice([1, 2, 4, 8])
    d = rng.choice([32, 64, 64, 80, 96, 128, 128])
    page = rng.choice([8, 16, 24, 32, 64, 128])
    common = dict(Hkv=hkv, D=d, page=page, head_major=rng.random() < 0.5)
    if op == "rotary":
        c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), tokens=_log_int(rng, 1, 8192), Hkv=hkv,
                 Hq=hkv * rng.choice([1, 4, 5, 8]), D=d, rot=rng.choice([d, d // 2]),
                 interleaved=rng.random() < 0.5, max_pos=_log_int(rng, 2048, 131072))
    elif op == "append":
        c = dict(op=op, B=_log_int(rng, 1, 128), T=rng.choice([1, 1, 5, 16]), Hq=hkv * rng.choice([1, 4, 5, 8]),
                 rot=rng.choice([d, d // 2]), interleaved=rng.random() < 0.5, length=_log_int(rng, 1, 2000),
                 max_pos=8192, **common)
        c["unused"] = rng.randrange(c["T"])
    elif op == "tree":
        t = rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 2, 64)])
        c = dict(op=op, B=_log_int(rng, 1, 64), T=t, Hq=hkv * rng.choice([1, 4, 5, 8]), length=_log_int(rng, 1, 131072),
                 ragged=rng.random() < 0.5, window=rng.choice([0, 0, 128, 1000]), sinks=rng.random() < 0.5,
                 tree=rng.choice(["chain", "shared", "each"]), unused=rng.randrange(t), **common)
    elif op == "mass":
        a = rng.choice([1, 1, _log_int(rng, 2, 12)])
        c = dict(op=op, B=_log_int(rng, 1, 32), T=rng.choice([a, 2 * a + 3]), A=a, Hq=hkv * rng.choice([1, 4, 5, 8]),
                 length=_log_int(rng, 1, 32768), ragged=rng.random() < 0.5, **common)
    else:
        n = _log_int(rng, 16, 32768)
        b = max(4, int(n * rng.uniform(0.1, 1.1)))
        c = dict(op=op, B=_log_int(rng, 1, 16), length=n, ragged=rng.random() < 0.5, budget=b,
                 first=rng.randrange(min(b // 4, 8) + 1), last=rng.randrange(b // 2 + 1), **common)
    # no more work or memory than the largest listed cases: bytes, products, a full cache, a full score matrix
    while "length" in c and _heavy(c):
        if c["B"] > 1:
            c["B"] //= 2
        else:
            c["length"] //= 2
    return c


def _heavy(c):
    w, rows = work(c), c.get("Hq", 0) * c.get("A", c.get("T", 0))
    n = c["B"] * c["length"]
    return w["bytes"] > 5e8 or w["flops"] > 6e10 or n * c["Hkv"] * c["D"] > 2.6e8 or n * rows > 2.6e8


def _lens(case):
    """Cached lengths of the sequences, from the case alone: all full, or spread from 0 and 1 up."""
    B, n = case["B"], case["length"]
    if not case.get("ragged"):
        return [n] * B
    lens = [int(n * ((b * 0.6180339887) % 1.0)) for b in range(B)]
    if B > 2:
        lens[0], lens[1], lens[2] = n, 0, min(1, n)
    else:
        lens[0] = n
    return lens


def work(case):
    op = case["op"]
    D = case["D"]
    if op in ("rotary", "append"):
        e = 4 if case.get("dtype") == "f32" else 2
        n = case["tokens"] if op == "rotary" else case["B"] * case["T"]
        rows = n * (case["Hq"] + case["Hkv"])
        if op == "rotary":  # forward and backward, each input read and each output written once
            return {"bytes": 4 * rows * D * e + 2 * n * case["rot"] * 4, "flops": 2 * 3 * rows * case["rot"]}
        return {"bytes": 2 * (rows + n * case["Hkv"]) * D * e + n * case["rot"] * 4, "flops": 3 * rows * case["rot"]}
    lens = _lens(case)
    Hkv = case["Hkv"]
    if op == "tree":
        T, W = case["T"], case["window"]
        keys = [(min(n, W - 1) if W else n) + T for n in lens]
        qo = case["B"] * T * case["Hq"] * (4 * D + 4)
        return {"bytes": sum(keys) * Hkv * D * 4 + qo, "flops": 4 * D * case["Hq"] * T * sum(keys)}
    if op == "mass":
        A, cap = case["A"], _capacity(case)
        keys = [n + A for n in lens]
        return {"bytes": sum(keys) * Hkv * D * 2 + 2 * case["B"] * Hkv * cap * 4 + case["B"] * A * case["Hq"] * (2 * D + 4),
                "flops": 2 * D * case["Hq"] * A * sum(keys)}
    kept = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": sum(lens) * Hkv * 4 + kept * Hkv * (8 * D + 4) + case["B"] * Hkv * 4 * (case["budget"] + _out_capacity(case)),
            "flops": 0}


# ------------------------------------------------------------------ inputs
def _pages(n, page):
    return -(-n // page)


def _capacity(case):
    return _pages(case["length"] + case.get("T", 0), case["page"]) * case["page"]


def _out_capacity(case):
    return _pages(min(case["budget"], max(case["length"], 1)), case["page"]) * case["page"]


def _cache(case, pages, gen, dev):
    shape = (pages, case["page"], case["Hkv"], case["D"])
    if case["head_major"]:
        return torch.randn(pages, case["Hkv"], case["page"], case["D"], generator=gen, device=dev,
                           dtype=torch.bfloat16).transpose(1, 2)
    return torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16)


def _table(max_pos, rot, dev):
    """cos and sin of position * frequency [max_pos, rot/2, 2], frequencies stretched for long contexts
    (interpolated below one turn in 4096 positions, kept above 32 turns, blended between), made in 64 bits."""
    i = torch.arange(rot // 2, device=dev, dtype=torch.float64)
    f = 150000.0 ** (-2 * i / rot)
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns.log() - math.log(1.0)) / math.log(32.0)).clamp(0, 1)
    f = f * keep + f / 32 * (1 - keep)
    a = torch.arange(max_pos, device=dev, dtype=torch.float64)[:, None] * f
    m = 0.1 * math.log(32.0) + 1.0
    return (torch.stack([a.cos(), a.sin()], -1) * m).float()


def _parents(T, gen):
    return [-1] + [int(torch.randint(-1, t, (1,), generator=gen)) for t in range(1, T)]


def _closure(parents):
    T = len(parents)
    mask, depth = torch.zeros(T, T, dtype=torch.bool), torch.zeros(T, dtype=torch.int32)
    for t, p in enumerate(parents):
        if p >= 0:
            mask[t] = mask[p]
            depth[t] = depth[p] + 1
        mask[t, t] = True
    return mask, depth


def _sequences(case, seed, dev):
    """Lengths in the seed's order, and a page table whose pages are in the seed's order."""
    g = torch.Generator().manual_seed(seed)
    B = case["B"]
    order = torch.randperm(B, generator=g)
    lens = torch.tensor(_lens(case), dtype=torch.int32)[order].to(dev)
    P = _pages(case["length"] + case.get("T", 0), case["page"])
    table = torch.randperm(B * P, generator=g).reshape(B, P).to(torch.int32).to(dev)
    return g, lens, table, B * P


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "rotary":
        dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        n, Hq, Hkv, D = case["tokens"], case["Hq"], case["Hkv"], case["D"]
        # the fused projection's output, of which queries and keys are strided views
        qkv = torch.randn(n, Hq + 2 * Hkv, D, generator=gen, device=dev, dtype=dt)
        s["q"] = qkv[:, :Hq].requires_grad_()
        s["k"] = qkv[:, Hq:Hq + Hkv].requires_grad_()
        s["dq"] = torch.randn(n, Hq, D, generator=gen, device=dev, dtype=dt)
        s["dk"] = torch.randn(n, Hkv, D, generator=gen, device=dev, dtype=dt)
        start = torch.randint(0, max(1, case["max_pos"] - n), (1,), generator=gen, device=dev)
        s["positions"] = (torch.arange(n, device=dev) + start).clamp(max=case["max_pos"] - 1).to(torch.int32)
        s["table"] = _table(case["max_pos"], case["rot"], dev)
        return s
    g, lens, table, pages = _sequences(case, seed, dev)
    s["lens"], s["page_table"] = lens, table
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    if case["op"] == "append":
        T, Hq = case["T"], case["Hq"]
        s["kc"], s["vc"] = _cache(case, pages, gen, dev), _cache(case, pages, gen, dev)
        qkv = torch.randn(B, T, Hq + 2 * Hkv, D, generator=gen, device=dev, dtype=torch.bfloat16)
        s["q"], s["k"], s["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
        t = torch.arange(T, device=dev, dtype=torch.int32)
        pos = (lens[:, None] + t).clamp(max=case["max_pos"] - 1)
        off = torch.arange(B, device=dev) % 2 == 1
        s["positions"] = torch.where(off[:, None] & (t >= T - case["unused"]), -1, pos)
        s["table"] = _table(case["max_pos"], case["rot"], dev)
    elif case["op"] == "tree":
        T, Hq = case["T"], case["Hq"]
        s["kc"], s["vc"] = _cache(case, pages, gen, dev), _cache(case, pages, gen, dev)
        s["q"] = (torch.randn(B, T, Hq, D, generator=gen, device=dev) * 1.5).bfloat16()
        s["sinks"] = torch.randn(Hq, generator=gen, device=dev) if case["sinks"] else None
        if case["tree"] == "chain":
            mask, depth = None, torch.arange(T, dtype=torch.int32).expand(B, T)
        elif case["tree"] == "shared":
            mask, depth = _closure(_parents(T, g))
            depth = depth.expand(B, T)
        else:
            both = [_closure(_parents(T, g)) for _ in range(B)]
            mask, depth = torch.stack([m for m, _ in both]), torch.stack([d for _, d in both])
        s["mask"] = None if mask is None else mask.to(dev)
        t = torch.arange(T, device=dev)
        off = torch.arange(B, device=dev) % 2 == 1
        s["positions"] = torch.where(off[:, None] & (t >= T - case["unused"]), -1, lens[:, None] + depth.to(dev)).to(torch.int32)
    elif case["op"] == "mass":
        T, A, Hq = case["T"], case["A"], case["Hq"]
        s["kc"] = _cache(case, pages, gen, dev)
        s["q"] = (torch.randn(B, T, Hq, D, generator=gen, device=dev) * 1.5).bfloat16()
        # an ascending path of 1 to A accepted drafts, or None where every token is accepted
        if A < T:
            acc = torch.full((B, A), -1, dtype=torch.int32)
            for b in range(B):
                n = int(torch.randint(1, A + 1, (1,), generator=g))
                acc[b, :n] = torch.randperm(T, generator=g)[:n].sort().values.to(torch.int32)
            s["accepted"] = acc.to(dev)
        else:
            s["accepted"] = None
        cap = _capacity(case)
        j = torch.arange(cap, device=dev)
        s["scores"] = torch.where(j < lens[:, None, None], torch.rand(B, Hkv, cap, generator=gen, device=dev) * 0.1, 0.0)
        # what attention said of the same tokens: the logarithm of each row's sum
        order = torch.arange(T, device=dev).expand(B, T) if A == T else s["accepted"].long()
        rank = torch.full((B, T + 1), -1, device=dev).scatter_(1, torch.where(order < 0, T, order), torch.arange(A, device=dev).expand(B, A))[:, :T]
        seen = j <= (lens[:, None] + rank.clamp(min=0))[:, :, None]
        x = _scores(s["q"], _gather(s["kc"], table, cap))
        x = x.masked_fill(~seen[:, None, :, None], -math.inf)
        s["lse"] = x.logsumexp(-1).permute(0, 2, 1, 3).reshape(B, T, Hq).contiguous()
    else:
        P, Q = table.shape[1], _out_capacity(case) // case["page"]
        pages += B * Q
        order = torch.randperm(pages, generator=g).to(torch.int32).to(dev)
        s["page_table"], s["out_table"] = order[:B * P].reshape(B, P), order[B * P:].reshape(B, Q)
        s["kc"], s["vc"] = _cache(case, pages, gen, dev), _cache(case, pages, gen, dev)
        cap = P * case["page"]
        j = torch.arange(cap, device=dev)
        x = torch.randn(B, Hkv, cap, generator=gen, device=dev)
        x = torch.where(x < -1, 0.0, (2 * x).exp())  # a few keys hold most of the weight, some have none
        s["scores"] = torch.where(j < lens[:, None, None], x, 0.0)
    return s


# ------------------------------------------------------------------ the plain forms
def _rotate(x, cs, interleaved, inverse):
    """Pairs of the first rot values turned by the angle whose (cos, sin) is cs [..., rot/2, 2]."""
    r = 2 * cs.shape[-2]
    c, s = cs[..., 0].unsqueeze(-2), cs[..., 1].unsqueeze(-2)
    s = -s if inverse else s
    y = x[..., :r]
    if interleaved:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = y[..., : r // 2], y[..., r // 2:]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, x[..., r:]], -1)


def _gather(cache, table, n):
    """Slots 0..n-1 of every sequence: [B, n, Hkv, D]."""
    page = cache.shape[1]
    j = torch.arange(n, device=cache.device)
    return cache[table[:, j // page].long(), j % page]


def _scores(q, k):
    """q . k / sqrt(D): [B, Hkv, T, Hq/Hkv, n]."""
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    x = q.float().view(B, T, Hkv, -1, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    x = torch.matmul(x, k.float().permute(0, 2, 3, 1)) * D ** -0.5
    return x.view(B, Hkv, T, Hq // Hkv, -1)


def _visible(lens, pos, mask, window, n):
    """Which of the slots 0..n-1 each drafted token attends: [B, T, n]."""
    B, T = pos.shape
    dev = pos.device
    j = torch.arange(n, device=dev)
    lens, used = lens[:, None, None].long(), pos >= 0
    if mask is None:
        mask = torch.ones(T, T, dtype=torch.bool, device=dev).tril()
    mask = mask.expand(B, T, T) & used[:, None, :]
    u = (j - lens).expand(B, T, n)
    at = u.clamp(0, T - 1)
    drafted = (u >= 0) & (u < T) & mask.gather(2, at)
    keypos = torch.where(u < 0, j, pos.long()[:, None, :].expand(B, T, T).gather(2, at))
    see = (u < 0) | drafted
    if window:
        see = see & (keypos > torch.maximum(pos.long()[:, :, None], lens) - window)
    return see & used[:, :, None]


def _attend(q, k, v, see, sinks, used):
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    x = _scores(q, k).masked_fill(~see[:, None, :, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    if sinks is not None:
        sink = sinks.float().view(1, Hkv, 1, -1, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m.isinf(), 0.0, m)
    p = (x - m).exp()
    z = p.sum(-1, keepdim=True)
    if sinks is not None:
        z = z + (sink - m).exp()
    o = torch.matmul(p.view(B, Hkv, -1, p.shape[-1]), v.float().permute(0, 2, 1, 3)).view(B, Hkv, T, -1, D)
    on = used[:, None, :, None, None]
    o = torch.where(on & (z > 0), o / z, 0.0)
    lse = torch.where(on, m + z.log(), -math.inf)[..., 0]
    return (o.permute(0, 2, 1, 3, 4).reshape(B, T, Hq, D).to(q.dtype), lse.permute(0, 2, 1, 3).reshape(B, T, Hq))


def _mass(q, k, lse, scores, lens, accepted):
    B, T, Hq, D = q.shape
    if accepted is None:
        accepted = torch.arange(T, device=q.device).expand(B, T)
    at = accepted.clamp(min=0).long()
    Hkv, cap = scores.shape[1], scores.shape[2]
    x = _scores(q.gather(1, at[:, :, None, None].expand(-1, -1, Hq, D)), k)
    y = lse.gather(1, at[:, :, None].expand(-1, -1, Hq)).view(B, -1, Hkv, Hq // Hkv).permute(0, 2, 1, 3)
    i = torch.arange(accepted.shape[1], device=q.device)
    see = (torch.arange(cap, device=q.device) <= (lens[:, None] + i)[:, :, None]) & (accepted >= 0)[:, :, None]
    p = torch.where(see[:, None, :, None], (x - y[..., None]).exp(), 0.0)
    return scores + p.sum((2, 3))


def _evict(s, c):
    lens, scores, budget = s["lens"].long()[:, None, None], s["scores"], c["budget"]
    B, Hkv, cap = scores.shape
    page, dev = c["page"], scores.device
    j = torch.arange(cap, device=dev)
    safe = (j < c["first"]) | (j >= lens - c["last"])
    key = torch.where(j < lens, torch.where(safe, math.inf, scores), -math.inf)
    n = min(budget, cap)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :n]
    lens_out = lens.clamp(max=budget)
    i = torch.arange(n, device=dev)
    kept = torch.where(i < lens_out, best, cap).sort(-1).values
    ok = (i < lens_out).expand(B, Hkv, n)
    at = kept.clamp(max=cap - 1)
    out_cap = s["out_table"].shape[1] * page
    src = s["page_table"].long().unsqueeze(1).expand(B, Hkv, -1).gather(2, at // page), at % page
    b, h, x = torch.nonzero(ok, as_tuple=True)
    dst = s["out_table"].long()[b, x // page], x % page
    s["kc"][dst[0], dst[1], h] = s["kc"][src[0][b, h, x], src[1][b, h, x], h]
    s["vc"][dst[0], dst[1], h] = s["vc"][src[0][b, h, x], src[1][b, h, x], h]
    new = torch.zeros(B, Hkv, out_cap, device=dev)
    new[..., :n] = torch.where(ok, scores.gather(2, at), 0.0)
    full = torch.full((B, Hkv, budget), -1, dtype=torch.int32, device=dev)
    full[..., :n] = torch.where(ok, kept, -1).to(torch.int32)
    return full, lens_out[:, 0, 0].to(torch.int32), new


def _plain(s):
    c = s["case"]
    if c["op"] == "rotary":
        cs = s["table"][s["positions"].long()]
        turn = lambda x, inv: _rotate(x.detach().float(), cs, c["interleaved"], inv).to(x.dtype)  # noqa: E731
        return turn(s["q"], False), turn(s["k"], False), turn(s["dq"], True), turn(s["dk"], True)
    if c["op"] == "append":
        pos, lens, kc, vc = s["positions"], s["lens"], s["kc"], s["vc"]
        used = (pos >= 0)[:, :, None, None]
        cs = s["table"][pos.clamp(min=0).long()]
        q = torch.where(used, _rotate(s["q"].float(), cs, c["interleaved"], False).to(s["q"].dtype), 0)
        k = _rotate(s["k"].float(), cs, c["interleaved"], False).to(kc.dtype)
        j = (lens[:, None] + torch.arange(c["T"], device=pos.device)).long()
        at = s["page_table"].gather(1, j // c["page"]).long(), j % c["page"]
        kc[at] = torch.where(used, k, kc[at])
        vc[at] = torch.where(used, s["v"], vc[at])
        return q, kc, vc
    if c["op"] == "tree":
        n = c["length"] + c["T"]
        see = _visible(s["lens"], s["positions"], s["mask"], c["window"], n)
        return _attend(s["q"], _gather(s["kc"], s["page_table"], n), _gather(s["vc"], s["page_table"], n), see,
                       s["sinks"], s["positions"] >= 0)
    if c["op"] == "mass":
        k = _gather(s["kc"], s["page_table"], s["scores"].shape[2])
        return _mass(s["q"], k, s["lse"], s["scores"], s["lens"], s["accepted"])
    return *_evict(s, c), s["kc"], s["vc"]


def run(state):
    s, c = state, state["case"]
    if not own:
        return _plain(s)
    from blockstreamer_b200 import attention, kernels
    if c["op"] == "rotary":
        q, k = attention.apply_rotary(s["q"], s["k"], s["table"], s["positions"], interleaved=c["interleaved"])
        return q, k, *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    if c["op"] == "append":
        q = kernels.rope_append(s["q"], s["k"], s["v"], s["table"], s["positions"], s["kc"], s["vc"], s["page_table"],
                                s["lens"], interleaved=c["interleaved"])
        return q, s["kc"], s["vc"]
    if c["op"] == "tree":
        return kernels.tree_attention(s["q"], s["kc"], s["vc"], s["page_table"], s["lens"], s["positions"],
                                      tree_mask=s["mask"], sinks=s["sinks"], window=c["window"])
    if c["op"] == "mass":
        return kernels.kv_scores_add(s["scores"], s["q"], s["lse"], s["kc"], s["page_table"], s["lens"],
                                     accepted=s["accepted"])
    kept, lens, scores = kernels.kv_evict(s["kc"], s["vc"], s["page_table"], s["lens"], s["scores"], c["budget"],
                                          s["out_table"], keep_first=c["first"], keep_last=c["last"])
    return kept, lens, scores, s["kc"], s["vc"]


# ------------------------------------------------------------------ the definitions in 64 bits
def _turn64(x, table, positions, interleaved, sign):
    """Complex multiplication by cos + i sin of the first rot values, as pairs."""
    used = positions >= 0
    w = torch.view_as_complex(table.double().contiguous())[positions.clamp(min=0).long()].unsqueeze(-2)
    w = w if sign > 0 else w.conj()
    r = 2 * w.shape[-1]
    y = x.double().clone()
    pair = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(y[..., pair[0]].contiguous(), y[..., pair[1]].contiguous()) * w
    y[..., pair[0]], y[..., pair[1]] = z.real, z.imag
    return y * used[..., None, None]


def _rows64(cache, table, b, n):
    page = cache.shape[1]
    pages = table[b, : _pages(max(n, 1), page)].long()
    return cache[pages].reshape(-1, *cache.shape[2:])[:n].double()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        t, p, i = s["table"], s["positions"], case["interleaved"]
        with torch.no_grad():
            return (_turn64(s["q"], t, p, i, 1), _turn64(s["k"], t, p, i, 1), _turn64(s["dq"], t, p, i, -1),
                    _turn64(s["dk"], t, p, i, -1))
    if op == "append":
        k = _turn64(s["k"], s["table"], s["positions"], case["interleaved"], 1)
        kc = s["kc"].double()
        for b, n in enumerate(s["lens"].tolist()):
            for t in range(case["T"]):
                if int(s["positions"][b, t]) >= 0:
                    kc[int(s["page_table"][b, (n + t) // case["page"]]), (n + t) % case["page"]] = k[b, t]
        return _turn64(s["q"], s["table"], s["positions"], case["interleaved"], 1), kc, None
    lens = s["lens"].tolist()
    if op == "evict":
        out = torch.zeros(case["B"], case["Hkv"], _out_capacity(case), dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            score = s["scores"][b, :, :n].double()
            rank = score.clone()
            rank[:, : case["first"]] = math.inf
            rank[:, max(0, n - case["last"]):] = math.inf
            keep = rank.sort(dim=-1, descending=True, stable=True).indices[:, : case["budget"]].sort(-1).values
            out[b, :, : keep.shape[1]] = score.gather(1, keep)
        return None, None, out, None, None
    Hkv, D, T = case["Hkv"], case["D"], case["T"]
    G = case["Hq"] // Hkv
    if op == "mass":
        out = s["scores"].double()
        for b, n in enumerate(lens):
            path = list(range(T)) if s["accepted"] is None else [u for u in s["accepted"][b].tolist() if u >= 0]
            k = _rows64(s["kc"], s["page_table"], b, n + len(path))
            for i, u in enumerate(path):
                q = s["q"][b, u].double().view(Hkv, G, D)
                x = torch.einsum("hgd,nhd->hgn", q, k[: n + i + 1]) / math.sqrt(D)
                out[b, :, : n + i + 1] += (x - s["lse"][b, u].double().view(Hkv, G, 1)).exp().sum(1)
        return out
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    pos = s["positions"]
    sink = None if s["sinks"] is None else s["sinks"].double().view(1, Hkv, G, 1)
    for b, n in enumerate(lens):
        k, v = _rows64(s["kc"], s["page_table"], b, n + T), _rows64(s["vc"], s["page_table"], b, n + T)
        p = pos[b].long()
        m = torch.ones(T, T, device="cuda").tril().bool() if s["mask"] is None else s["mask"] if s["mask"].dim() == 2 else s["mask"][b]
        see = torch.cat([torch.ones(T, n, dtype=torch.bool, device="cuda"), m & (p >= 0)], 1)
        if case["window"]:
            at = torch.cat([torch.arange(n, device="cuda"), p])
            see &= at[None] > p.clamp(min=n)[:, None] - case["window"]
        x = torch.einsum("thgd,nhd->thgn", s["q"][b].double().view(T, Hkv, G, D), k) / math.sqrt(D)
        x = x.masked_fill(~see[:, None, None], -math.inf)
        if sink is not None:
            x = torch.cat([x, sink.expand(T, -1, -1, -1)], -1)
        z = x.logsumexp(-1)
        w = torch.nan_to_num((x - z[..., None]).exp(), nan=0.0)[..., : n + T]
        on = p >= 0
        o[b] = torch.einsum("thgn,nhd->thgd", w, v).reshape(T, -1, D) * on[:, None, None]
        lse[b] = torch.where(on[:, None], z.reshape(T, -1), -math.inf)
    return o, lse
