"""The attention half of a gpt-oss decoder layer at decode sizes.

``rotary_frequencies`` / ``rotary_table`` make the cos/sin table that the rotary
kernels read, with transformers' scalings for long contexts (yarn, linear);
``apply_rotary`` is the differentiable form for training.  The kernels
themselves are in ``kernels``.

Mirrors transformers models/gpt_oss/modeling_gpt_oss.py (GptOssRotaryEmbedding,
apply_rotary_pos_emb, GptOssAttention), which the reference runs unchanged.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from . import kernels


def rotary_frequencies(rot: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[Tensor, float]:
    """Angle per position of each of the rot/2 pairs (f64), and the factor on cos and sin.

    ``scaling`` follows transformers' ``rope_scaling``: ``{"rope_type":
    "linear", "factor": f}`` stretches every frequency; ``{"rope_type": "yarn",
    "factor": f, "original_max_position_embeddings": n, "beta_fast": 32,
    "beta_slow": 1, "truncate": bool, "attention_factor": optional}`` keeps the
    pairs that turn more than beta_fast times in n positions, stretches those
    that turn less than beta_slow times and blends linearly between."""
    if rot <= 0 or rot % 2:
        raise ValueError(f"rot must be even and positive, got {rot}")
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return freq, 1.0
    factor = float(scaling["factor"])
    if kind == "linear":
        return freq / factor, 1.0
    if kind != "yarn":
        raise ValueError(f"unknown rope_type {kind!r} (default, linear or yarn)")
    n = scaling["original_max_position_embeddings"]

    def pair_of(turns: float) -> float:
        # index of the pair that turns `turns` times in n positions
        return rot * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = pair_of(scaling.get("beta_fast") or 32.0), pair_of(scaling.get("beta_slow") or 1.0)
    if scaling.get("truncate", True):
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, rot - 1)
    if low == high:
        high += 0.001
    stretch = ((torch.arange(rot // 2, dtype=torch.float64) - low) / (high - low)).clamp(0, 1)
    factor_out = scaling.get("attention_factor")
    if factor_out is None:
        factor_out = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return freq * (1 - stretch) + freq / factor * stretch, float(factor_out)


def rotary_table(max_pos: int, rot: int, base: float = 10000.0, scaling: dict | None = None,
                 device="cuda") -> Tensor:
    """cos and sin of every position and pair, [max_pos, rot/2, 2] f32, made in
    64 bits (a 32-bit product of position and frequency is off by up to 4e-3 rad
    at position 131072)."""
    freq, factor = rotary_frequencies(rot, base, scaling)
    angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return (torch.stack([angle.cos(), angle.sin()], dim=-1) * factor).float()


class _Rotary(torch.autograd.Function):
    """bs_rope forward; the gradient is the turn by the opposite angle."""

    @staticmethod
    def forward(ctx, q: Tensor, k: Tensor | None, table: Tensor, positions: Tensor, interleaved: bool):
        ctx.save_for_backward(table, positions)
        ctx.interleaved = interleaved
        return kernels.rope(q, k, table, positions, interleaved)

    @staticmethod
    def backward(ctx, dq: Tensor | None, dk: Tensor | None):
        table, positions = ctx.saved_tensors
        if dq is None or dk is None:
            one = dq if dq is not None else dk
            if one is None:
                return None, None, None, None, None
            g, _ = kernels.rope(_last_contiguous(one), None, table, positions, ctx.interleaved, inverse=True)
            return (g if dq is not None else None), (g if dk is not None else None), None, None, None
        gq, gk = kernels.rope(_last_contiguous(dq), _last_contiguous(dk), table, positions, ctx.interleaved,
                              inverse=True)
        return gq, gk, None, None, None


def _last_contiguous(t: Tensor) -> Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def apply_rotary(q: Tensor, k: Tensor | None, table: Tensor, positions: Tensor, interleaved: bool = False):
    """Rotary positions of q and k with gradients (``kernels.rope`` both ways).
    No gradient flows to the table."""
    return _Rotary.apply(q, k, table, positions, interleaved)
