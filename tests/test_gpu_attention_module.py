"""The attention layer and its paged cache, used as a decoding loop uses them:
against transformers' own GptOssAttention over the whole sequence, and through
the example.

Tolerance against transformers in fp32 on the same (bf16) weights and inputs: ours
rounds to bf16 q, k and v (once after the projection, q and k once more after the
turn), the weights P, the heads' output and the projected output; seven roundings
of relative 2^-9 rms each that are independent, 2^-9 sqrt(7) = 5e-3, doubled.
"""

import os
import subprocess
import sys
import types

import pytest
import torch

from conftest import REPO
from blockstreamer_b200 import B200GptOssAttention, PagedKVCache, attention, kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(hidden=128, heads=8, kv_heads=2, head_dim=64, window=0, seed=0):
    cfg = types.SimpleNamespace(hidden_size=hidden, num_attention_heads=heads, num_key_value_heads=kv_heads,
                                head_dim=head_dim, sliding_window=window, attention_bias=True,
                                layer_types=["sliding_attention" if window else "full_attention"])
    m = B200GptOssAttention(cfg)
    g = torch.Generator().manual_seed(seed)
    state = {n: (torch.randn(p.shape, generator=g) * (hidden ** -0.5 if p.dim() == 2 else 0.5)).to(torch.bfloat16)
             for n, p in m.named_parameters()}
    m.load_state_dict(state, assign=True)
    return m.to(DEV).requires_grad_(False), state, g


def transformers_layer(state, hidden, heads, kv_heads, head_dim, window):
    hf = pytest.importorskip("transformers.models.gpt_oss.modeling_gpt_oss")
    cfg = pytest.importorskip("transformers").GptOssConfig(
        hidden_size=hidden, num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=head_dim,
        num_hidden_layers=1, sliding_window=window or 128, num_local_experts=2, num_experts_per_tok=1,
        intermediate_size=32, vocab_size=16,
        layer_types=["sliding_attention" if window else "full_attention"])
    cfg._attn_implementation = "eager"
    layer = hf.GptOssAttention(cfg, 0).float()
    layer.load_state_dict({n: t.float() for n, t in state.items()})
    return layer, hf.GptOssRotaryEmbedding(cfg), cfg


@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("chunks", [[1] * 9, [40, 1, 1, 7, 30, 2]])
def test_layer_matches_transformers(window, chunks):
    hidden, heads, kv_heads, D = 128, 8, 2, 64
    m, state, g = make(hidden, heads, kv_heads, D, window)
    layer, rotary, cfg = transformers_layer(state, hidden, heads, kv_heads, D, window)
    n, B = sum(chunks), 2
    x = torch.randn(B, n, hidden, generator=g).to(torch.bfloat16)
    pos = torch.arange(n)[None].expand(B, n)
    i = torch.arange(n)
    see = i[None] <= i[:, None]
    if window:
        see = see & (i[None] > i[:, None] - window)
    bias = torch.where(see, 0.0, torch.finfo(torch.float32).min)[None, None].expand(B, 1, n, n)
    with torch.no_grad():
        want = layer(x.float(), position_embeddings=rotary(x.float(), pos), attention_mask=bias)[0]
    scaling = {k: v for k, v in (getattr(cfg, "rope_parameters", None) or cfg.rope_scaling).items()}
    base = scaling.get("rope_theta", getattr(cfg, "rope_theta", 150000.0))
    table = attention.rotary_table(256, D, base, scaling, device=DEV)
    cache = PagedKVCache(B, 32, 16, kv_heads, D, 128, DEV)
    got, at = [], 0
    for c in chunks:
        p = (at + torch.arange(c, dtype=torch.int32))[None].repeat(B, 1).to(DEV)
        out, _, _ = m(x[:, at:at + c].to(DEV), p, cache, table)
        cache.commit([list(range(c))] * B, c)
        got.append(out.float().cpu())
        at += c
    got = torch.cat(got, 1)
    assert cache.lengths == [n, n] and cache.lens.tolist() == [n, n]
    rel = ((got - want).norm() / want.norm()).item()
    print(f"window {window}: rel-L2 {rel:.2e}")
    assert rel <= 1e-2
    assert kernels.device_status(clear=True) == 0


def test_a_tree_gives_each_path_what_the_path_alone_gives():
    """Drafted siblings do not see each other: every root-to-leaf path of a tree gives
    the outputs of a chain of its tokens, and after commit the cache is that chain's."""
    m, _, g = make()
    table = attention.rotary_table(64, 64, device=DEV)
    x0 = torch.randn(1, 5, 128, generator=g).to(torch.bfloat16).to(DEV)
    x = torch.randn(1, 6, 128, generator=g).to(torch.bfloat16).to(DEV)
    parents = [-1, 0, 0, 1, 2, 2]
    mask = torch.zeros(6, 6, dtype=torch.bool)
    for t, p in enumerate(parents):
        if p >= 0:
            mask[t] = mask[p]
        mask[t, t] = True
    depth = mask.sum(-1) - 1

    def fresh():
        c = PagedKVCache(1, 8, 4, 2, 64, 32, DEV)
        p = torch.arange(5, dtype=torch.int32, device=DEV)[None]
        m(x0, p, c, table)
        c.commit([list(range(5))], 5)
        return c

    tree = fresh()
    out, _, _ = m(x, (5 + depth).to(torch.int32)[None].to(DEV), tree, table, mask.to(DEV))
    for leaf in (3, 4, 5):
        path = mask[leaf].nonzero().flatten().tolist()
        chain = fresh()
        p = (5 + torch.arange(len(path), dtype=torch.int32))[None].to(DEV)
        alone, _, _ = m(x[:, path], p, chain, table)
        err = (alone.float() - out[:, path].float()).norm() / alone.float().norm()
        assert err <= 1e-2     # the same keys in another order of slots
        if leaf == 4:
            keep, want = path, chain
    tree.commit([keep], 6)
    want.commit([list(range(len(keep)))], len(keep))
    n = 5 + len(keep)
    for c, d in ((tree.k, want.k), (tree.v, want.v)):
        rows = [c[tree.page_table[0].long()].reshape(-1, 2, 64)[:n], d[want.page_table[0].long()].reshape(-1, 2, 64)[:n]]
        # K and V of a token come from the same product and turn in both
        assert torch.equal(rows[0], rows[1])


def test_cache_hands_out_pages_and_evicts():
    cache = PagedKVCache(2, 12, 4, 1, 32, 24, DEV, track_scores=True)
    table = attention.rotary_table(64, 32, device=DEV)
    g = torch.Generator().manual_seed(3)
    with pytest.raises(ValueError, match="max_len"):
        cache.reserve(25)
    for step in range(5):
        q, k, v = (torch.randn(2, 2, h, 32, generator=g).to(torch.bfloat16).to(DEV) for h in (4, 1, 1))
        pos = cache.lens[:, None] + torch.arange(2, dtype=torch.int32, device=DEV)
        qt = cache.append(q, k, v, table, pos)
        _, lse = cache.attend(qt, pos)
        cache.commit([[0, 1], [1]], 2, qt, lse)
    assert cache.lengths == [10, 5]
    total = cache.scores.double().sum(-1).flatten().tolist()
    # five steps of two tokens, four heads: 40; of one token that saw one draft more than it kept: below 20
    assert total[0] == pytest.approx(40, abs=1e-3) and 0 < total[1] < 20
    before = [cache.k[cache.page_table[b].long()].reshape(-1, 32)[:n].clone() for b, n in enumerate(cache.lengths)]
    scores = cache.scores.clone()
    kept = cache.evict(6, keep_first=1, keep_last=2)
    assert cache.lengths == [6, 5] and len(cache._free) == 12 - 2 - 2
    for b in range(2):
        rows = kept[b, 0][: cache.lengths[b]].long()
        assert rows.tolist() == sorted(rows.tolist()) and rows[0] == 0
        now = cache.k[cache.page_table[b].long()].reshape(-1, 32)[: cache.lengths[b]]
        assert torch.equal(now, before[b][rows])
        assert torch.equal(cache.scores[b, 0, : cache.lengths[b]], scores[b, 0][rows])
        assert bool((cache.scores[b, 0, cache.lengths[b]:] == 0).all())
    with pytest.raises(RuntimeError, match="free"):
        cache.max_len = 10 ** 6
        cache.reserve(400)
    assert kernels.device_status(clear=True) == 0


def test_example_runs():
    res = subprocess.run([sys.executable, os.path.join(REPO, "examples", "tree_decode.py"), "--steps", "6", "--batch",
                          "3", "--drafts", "10", "--budget", "16"], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
    assert "(cut)" in res.stdout and "step 5" in res.stdout and "nan" not in res.stdout
