"""Speculative decoding steps of one gpt-oss decoder layer on synthetic weights.

Each step drafts a small tree of tokens per sequence, runs the layer on all of
them at once (attention half: ``B200GptOssAttention`` over a ``PagedKVCache``;
MoE half: ``B200GptOssMoEBlock``), accepts one path of every tree, keeps its keys
and values, adds the attention they gave to the cached keys' scores, and cuts the
cache to its budget when it has grown past it.

    python examples/tree_decode.py [--steps 12] [--batch 4] [--drafts 12] [--budget 24]
"""

import argparse
import os
import sys
import types

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from blockstreamer_b200 import B200GptOssAttention, B200GptOssMoEBlock, PagedKVCache, kernels, rotary_table  # noqa: E402
from blockstreamer_b200.synthetic import LayerShape, make_layer  # noqa: E402


def build_layer(hidden=256, heads=16, kv_heads=2, head_dim=64, seed=7, device="cuda"):
    """A small decoder layer with seeded weights: (attention, input norm weight, MoE block, config)."""
    shape = LayerShape(hidden, hidden, 8, 2)
    cfg = types.SimpleNamespace(hidden_size=hidden, intermediate_size=hidden, num_local_experts=8,
                                num_experts_per_tok=2, swiglu_limit=7.0, num_attention_heads=heads,
                                num_key_value_heads=kv_heads, head_dim=head_dim, sliding_window=0,
                                layer_types=["full_attention"], attention_bias=True, rms_norm_eps=1e-5)
    g = torch.Generator().manual_seed(seed)
    attn = B200GptOssAttention(cfg)
    state = {n: (torch.randn(p.shape, generator=g) * (hidden ** -0.5 if p.dim() == 2 else 0.1)).to(torch.bfloat16)
             for n, p in attn.named_parameters()}
    attn.load_state_dict(state, assign=True)
    block = B200GptOssMoEBlock(cfg)
    moe = {f"mlp.{n}": t for n, t in make_layer(shape, seed).items()}
    moe["post_attention_layernorm.weight"] = torch.ones(hidden)
    block.load_state_dict(moe, assign=True)
    return attn.to(device).requires_grad_(False), torch.ones(hidden, device=device), block.to(device), cfg


def draft_tree(drafts, lens, generator):
    """A random tree for every sequence: mask [B, T, T] and positions [B, T]."""
    mask = torch.zeros(len(lens), drafts, drafts, dtype=torch.bool)
    pos = torch.zeros(len(lens), drafts, dtype=torch.int32)
    for b, n in enumerate(lens):
        for t in range(drafts):
            parent = int(torch.randint(-1, t, (1,), generator=generator)) if t else -1
            if parent >= 0:
                mask[b, t] = mask[b, parent]
            mask[b, t, t] = True
            pos[b, t] = n + int(mask[b, t].sum()) - 1
    return mask, pos


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=12)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--drafts", type=int, default=12)
    ap.add_argument("--budget", type=int, default=24)
    a = ap.parse_args()
    attn, norm, block, cfg = build_layer()
    g = torch.Generator().manual_seed(1)
    page = 16
    cache = PagedKVCache(a.batch, 16 * a.batch * (1 + (a.budget + 2 * a.drafts) // page), page, cfg.num_key_value_heads,
                         cfg.head_dim, max_len=a.budget + 4 * a.drafts, track_scores=True)
    table = rotary_table(4096, cfg.head_dim, 150000.0,
                         dict(rope_type="yarn", factor=32.0, original_max_position_embeddings=4096, truncate=False))
    tokens = [0] * a.batch   # positions of the sequences; the cache may hold fewer keys
    with torch.no_grad():
        for step in range(a.steps):
            mask, pos = draft_tree(a.drafts, tokens, g)
            x = torch.randn(a.batch, a.drafts, cfg.hidden_size, generator=g).to(torch.bfloat16).cuda()
            flat = kernels.rmsnorm(x.view(-1, cfg.hidden_size), norm, cfg.rms_norm_eps).view_as(x)
            h, q, lse = attn(flat, pos.cuda(), cache, table, mask.cuda())
            y = block(x + h)
            # accept the path to one leaf (a model would compare tokens here)
            accepted = [mask[b, int(torch.randint(0, a.drafts, (1,), generator=g))].nonzero().flatten().tolist()
                        for b in range(a.batch)]
            cache.commit(accepted, a.drafts, q, lse)
            tokens = [n + len(p) for n, p in zip(tokens, accepted)]
            cut = max(cache.lengths) > a.budget
            if cut:
                first = min(2, a.budget)
                cache.evict(a.budget, keep_first=first, keep_last=min(4, a.budget - first))
            print(f"step {step}: accepted {[len(p) for p in accepted]}, positions {tokens}, "
                  f"cached {cache.lengths}{' (cut)' if cut else ''}, output rms {y.float().pow(2).mean().sqrt():.3f}")
    status = kernels.device_status()
    if status:
        raise SystemExit(f"device status {status}")


if __name__ == "__main__":
    main()
