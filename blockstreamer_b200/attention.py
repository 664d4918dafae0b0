"""The attention half of a gpt-oss decoder layer at decode sizes.

``rotary_frequencies`` / ``rotary_table`` make the cos/sin table that the rotary
kernels read, with transformers' scalings for long contexts (yarn, linear);
``apply_rotary`` is the differentiable form for training.  ``PagedKVCache``
holds a batch of sequences and runs the steps of speculative decoding on them
(append, tree attention, commit, scores, eviction); ``B200GptOssAttention`` is
the layer around it, with transformers' parameter names.  The kernels themselves
are in ``kernels``.

Mirrors transformers models/gpt_oss/modeling_gpt_oss.py (GptOssRotaryEmbedding,
apply_rotary_pos_emb, GptOssAttention), which the reference runs unchanged.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor, nn

from . import kernels


def rotary_frequencies(rot: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[Tensor, float]:
    """Angle per position of each of the rot/2 pairs (f64), and the factor on cos and sin.

    ``scaling`` follows transformers' ``rope_scaling``: ``{"rope_type":
    "linear", "factor": f}`` stretches every frequency; ``{"rope_type": "yarn",
    "factor": f, "original_max_position_embeddings": n, "beta_fast": 32,
    "beta_slow": 1, "truncate": bool, "attention_factor": optional}`` keeps the
    pairs that turn more than beta_fast times in n positions, stretches those
    that turn less than beta_slow times and blends linearly between.  The factor
    is ``attention_factor``, or 0.1 m ln f + 1 with m = 1, or, where both are
    given, that of m = ``mscale`` over that of m = ``mscale_all_dim``."""
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
        def grown(m: float) -> float:
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

        m, all_dim = scaling.get("mscale"), scaling.get("mscale_all_dim")
        factor_out = grown(m) / grown(all_dim) if m and all_dim else grown(1.0)
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
    def forward(ctx, q: Tensor, k: Tensor | None, table: Tensor, positions: Tensor, interleaved: bool,
                inverse: bool = False):
        ctx.save_for_backward(table, positions)
        ctx.turn = interleaved, inverse
        return kernels.rope(q, k, table, positions, interleaved, inverse)

    @staticmethod
    def backward(ctx, dq: Tensor, dk: Tensor | None):
        # gradients that did not arrive are zeros here (autograd makes them); dk is None without k
        table, positions = ctx.saved_tensors
        interleaved, inverse = ctx.turn
        dq = dq if dq.stride(-1) == 1 else dq.contiguous()
        if dk is not None and dk.stride(-1) != 1:
            dk = dk.contiguous()
        if torch.is_grad_enabled():  # create_graph: the turn back has a gradient of its own
            gq, gk = _Rotary.apply(dq, dk, table, positions, interleaved, not inverse)
        else:
            gq, gk = kernels._rope(dq.get_device(), dq, dk, table, positions, interleaved, not inverse)
        return gq, gk, None, None, None, None


def apply_rotary(q: Tensor, k: Tensor | None, table: Tensor, positions: Tensor, interleaved: bool = False):
    """Rotary positions of q and k with gradients of any order (``kernels.rope`` both
    ways).  No gradient flows to the table."""
    return _Rotary.apply(q, k, table, positions, interleaved)


class PagedKVCache:
    """Keys and values of ``batch`` sequences in ``pages`` pages of ``page_size`` slots.

    Pages are [page, head, slot, dim] in memory, so that a head's slots of a page
    lie together.  The host keeps the lengths and hands out the pages; what the
    kernels read (``page_table``, ``lens``) is on the device.  ``scores`` (with
    ``track_scores``) accumulates the attention weight of every cached key; scores and
    eviction are for layers without a window."""

    def __init__(self, batch: int, pages: int, page_size: int, heads: int, dim: int, max_len: int, device="cuda",
                 track_scores: bool = False) -> None:
        shape = (pages, heads, page_size, dim)
        self.k = torch.zeros(shape, dtype=torch.bfloat16, device=device).transpose(1, 2)
        self.v = torch.zeros(shape, dtype=torch.bfloat16, device=device).transpose(1, 2)
        self.page_size, self.max_len = page_size, max_len
        self.width = -(-max_len // page_size)
        self.page_table = torch.zeros(batch, self.width, dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.scores = None
        if track_scores:
            self.scores = torch.zeros(batch, heads, self.width * page_size, dtype=torch.float32, device=device)
        self.lengths = [0] * batch                      # the host's copy of lens
        self._free = list(range(pages - 1, -1, -1))
        self._held: list[list[int]] = [[] for _ in range(batch)]
        self._windowed = False                          # a window has left keys out
        self._cut = False                               # slots are no longer positions

    def _upload(self) -> None:
        rows = [h + [0] * (self.width - len(h)) for h in self._held]
        self.page_table.copy_(torch.tensor(rows, dtype=torch.int32))
        self.lens.copy_(torch.tensor(self.lengths, dtype=torch.int32))

    def reserve(self, tokens: int) -> None:
        """Pages for ``tokens`` more slots of every sequence."""
        need = [-(-(n + tokens) // self.page_size) - len(h) for n, h in zip(self.lengths, self._held)]
        if any(n + tokens > self.max_len for n in self.lengths):
            raise ValueError(f"a sequence would pass max_len = {self.max_len}")
        if sum(max(0, x) for x in need) > len(self._free):
            raise RuntimeError(f"{sum(max(0, x) for x in need)} pages wanted, {len(self._free)} free")
        if max(need, default=0) > 0:
            for held, x in zip(self._held, need):
                held.extend(self._free.pop() for _ in range(max(0, x)))
            self._upload()

    def append(self, q: Tensor, k: Tensor, v: Tensor, table: Tensor, positions: Tensor,
               interleaved: bool = False) -> Tensor:
        """Turns q and k, writes k and v behind the committed keys; returns the turned q."""
        self.reserve(q.shape[1])
        return kernels.rope_append(q, k, v, table, positions, self.k, self.v, self.page_table, self.lens, interleaved)

    def attend(self, q: Tensor, positions: Tensor, tree_mask: Tensor | None = None, sinks: Tensor | None = None,
               window: int = 0):
        """(out, lse) of the drafted tokens whose keys ``append`` wrote."""
        if window:
            if self._cut:
                raise ValueError("attend: after evict slots are no longer positions, by which a window goes")
            self._windowed = self._windowed or max(self.lengths, default=0) + q.shape[1] > window
        return kernels.tree_attention(q, self.k, self.v, self.page_table, self.lens, positions, tree_mask, sinks,
                                      window)

    def commit(self, accepted: list[list[int]], drafted: int, q: Tensor | None = None, lse: Tensor | None = None) -> None:
        """Keeps the accepted drafts (ascending indices per sequence) and, given the
        step's turned ``q`` and its ``lse``, adds their attention to the scores."""
        scored = self.scores is not None and q is not None and lse is not None
        if scored and self._windowed:
            raise ValueError("commit: keys outside a window got no weight that could be added to their scores")
        if len(accepted) != len(self.lengths):
            raise ValueError(f"commit takes {len(self.lengths)} lists of accepted drafts, got {len(accepted)}")
        page = self.page_size
        for x, n, held in zip(accepted, self.lengths, self._held):
            # the device would leave such a sequence as it is, but not know its new length
            if not x:
                continue
            if x[0] < 0 or x[-1] >= drafted or (len(x) > 1 and sorted(set(x)) != x):
                raise ValueError(f"accepted drafts must ascend from 0 to below {drafted}, got {x}")
            if n + x[-1] >= len(held) * page:
                raise ValueError(f"draft {x[-1]} behind {n} keys lies outside the {len(held)} reserved pages")
        most = max((len(x) for x in accepted), default=0)
        if most:
            rows = [x + [-1] * (most - len(x)) for x in accepted]
            acc = torch.tensor(rows, dtype=torch.int32, device=self.k.device)
            kernels.tree_commit(self.k, self.v, self.page_table, self.lens, acc, drafted)
            if scored:
                kernels.kv_scores_add(self.scores, q, lse, self.k, self.page_table, self.lens, acc, out=self.scores)
        self.lengths = [n + len(x) for n, x in zip(self.lengths, accepted)]
        self.lens.copy_(torch.tensor(self.lengths, dtype=torch.int32))

    def evict(self, budget: int, keep_first: int | None = None, keep_last: int = 0) -> Tensor:
        """Cuts every sequence to its ``budget`` best keys per head, the first
        ``keep_first`` (by default four, or what ``keep_last`` leaves of the budget for
        them) and the last ``keep_last`` among them; returns the kept slots.  Only for
        layers without a window: slots are no longer positions."""
        if self.scores is None:
            raise ValueError("PagedKVCache.evict needs track_scores=True")
        if self._windowed:
            raise ValueError("evict is for layers without a window")
        if keep_first is None:
            keep_first = min(4, max(0, budget - keep_last))
        if keep_first < 0 or keep_last < 0 or keep_first + keep_last > budget:
            raise ValueError(f"keep_first {keep_first} + keep_last {keep_last} must not exceed the budget {budget}")
        # a sequence within the budget keeps the pages of its slots; the others' new ones
        # leave the free list when the call has been accepted
        new = [-(-min(n, budget) // self.page_size) for n in self.lengths]
        need = sum(x for x, n in zip(new, self.lengths) if n > budget)
        if need > len(self._free):
            raise RuntimeError(f"eviction needs {need} free pages, {len(self._free)} are")
        pages = reversed(self._free)
        taken = [[next(pages) for _ in range(x)] if n > budget else held[:x]
                 for x, n, held in zip(new, self.lengths, self._held)]
        width = max(1, max(new, default=0))
        out = torch.tensor([t + [0] * (width - len(t)) for t in taken], dtype=torch.int32, device=self.k.device)
        # a budget that no sequence reaches cuts nothing, whatever is protected
        budget = min(budget, width * self.page_size)
        keep_first = min(keep_first, budget)
        kept, _, scores = kernels.kv_evict(self.k, self.v, self.page_table, self.lens, self.scores, budget, out,
                                           keep_first, min(keep_last, budget - keep_first))
        self.scores.zero_()
        self.scores[..., : scores.shape[-1]] = scores
        del self._free[len(self._free) - need:]
        for x, n, held in zip(new, self.lengths, self._held):
            self._free.extend(held if n > budget else held[x:])
        self._held = taken
        self._cut = self._cut or need > 0
        self.lengths = [min(n, budget) for n in self.lengths]
        self._upload()
        return kept


class B200GptOssAttention(nn.Module):
    """GptOssAttention (modeling_gpt_oss.py) over a ``PagedKVCache``: drafted tokens
    (or one token) of every sequence against the cached ones.

    Parameters ``q_proj``, ``k_proj``, ``v_proj``, ``o_proj`` (weight and bias) and
    ``sinks`` have transformers' names and shapes, on ``meta`` until bound.  It serves
    decoding and has no backward pass: one that reaches its attention raises."""

    def __init__(self, config, layer_idx: int = 0, dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.heads, self.kv_heads = config.num_attention_heads, config.num_key_value_heads
        self.head_dim = getattr(config, "head_dim", None) or config.hidden_size // self.heads
        types = getattr(config, "layer_types", None)
        kind = types[layer_idx] if types else "full_attention"
        self.window = config.sliding_window if kind == "sliding_attention" else 0
        bias = getattr(config, "attention_bias", True)
        H, D = config.hidden_size, self.head_dim
        with torch.device("meta"):
            self.q_proj = nn.Linear(H, self.heads * D, bias=bias, dtype=dtype)
            self.k_proj = nn.Linear(H, self.kv_heads * D, bias=bias, dtype=dtype)
            self.v_proj = nn.Linear(H, self.kv_heads * D, bias=bias, dtype=dtype)
            self.o_proj = nn.Linear(self.heads * D, H, bias=bias, dtype=dtype)
            self.sinks = nn.Parameter(torch.empty(self.heads, dtype=dtype))

    def forward(self, hidden_states: Tensor, positions: Tensor, cache: PagedKVCache, table: Tensor,
                tree_mask: Tensor | None = None):
        """hidden_states [B, T, H], positions [B, T] int32 (negative: unused) ->
        (output [B, T, H], turned q, lse); the last two go to ``cache.commit``."""
        B, T, _ = hidden_states.shape
        q = self.q_proj(hidden_states).view(B, T, self.heads, self.head_dim)
        k = self.k_proj(hidden_states).view(B, T, self.kv_heads, self.head_dim)
        v = self.v_proj(hidden_states).view(B, T, self.kv_heads, self.head_dim)
        q = cache.append(q, k, v, table, positions)
        out, lse = cache.attend(q, positions, tree_mask, self.sinks.float(), self.window)
        return self.o_proj(out.view(B, T, -1)), q, lse
