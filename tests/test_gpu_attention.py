"""The attention half of the decoder layer against its definition in 64 bits.

Tolerances.  bf16 has eight significant bits, so rounding to nearest is off by a
relative 2^-8 at most (1 + 2^-8 becomes 1).  Rotary: one rounding of an fp32
result whose own error (two products and a sum, 2^-24 each of |a c| + |b s|) is
far below it.  Attention: the output's rounding, 2^-8 |out|, and the rounding of
each weight w_j to bf16, at most 2^-8 sum w_j |v_j| together; both bounds are
reached by no typical value, which leaves room for the fp32 sums.  Logarithms and scores are
fp32 throughout: D products of bf16 are exact, their sum is off by at most
D 2^-24 sum |q k|, below 2e-5 at these sizes.
"""

import math

import pytest
import torch

from attention_cases import make_cache, make_tree, pages_for, poison_unused
from blockstreamer_b200 import attention, kernels
from oracle import attention as oatt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def to(*ts):
    return [t.to(DEV) if isinstance(t, torch.Tensor) else t for t in ts]


@pytest.fixture(autouse=True)
def status_is_clear():
    kernels.device_status(clear=True)
    yield
    assert kernels.device_status(clear=True) == 0


# ---------------------------------------------------------------- rotary
def rotary_close(got, want, x, dtype):
    eps = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22
    err = (got.double().cpu() - want).abs()
    assert bool((err <= eps * want.abs() + 2.0 ** -21 * x.double().abs().amax()).all()), err.max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (128, 128), (64, 32), (96, 48), (80, 80), (6, 2), (10, 10), (2, 2), (256, 64)])
def test_rotary_layouts_and_parts(dtype, interleaved, D, rot):
    g = torch.Generator().manual_seed(D + rot)
    table = attention.rotary_table(200, rot, 10000.0, device="cpu")
    for shape, hk in (((1, 5), 1), ((3, 7), 2)):
        q = torch.randn(*shape, 4, D, generator=g).to(dtype)
        k = torch.randn(*shape, hk, D, generator=g).to(dtype)
        pos = torch.randint(0, 200, shape, generator=g)
        pos[0, 1] = -1
        pos[0, 2] = 199
        qo, ko = kernels.rope(*to(q, k, table, pos.to(torch.int32)), interleaved=interleaved)
        rotary_close(qo, oatt.rotary(q, table, pos, interleaved), q, dtype)
        rotary_close(ko, oatt.rotary(k, table, pos, interleaved), k, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 2, 33, 5000])
def test_rotary_takes_views_of_a_fused_projection(dtype, tokens):
    g = torch.Generator().manual_seed(tokens)
    D, Hq, Hk = 64, 5, 2
    qkv = torch.randn(tokens, Hq + 2 * Hk, D, generator=g).to(dtype).to(DEV)
    table = attention.rotary_table(tokens + 9, D, 150000.0)
    pos = torch.arange(9, tokens + 9, device=DEV)
    q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hk]
    qo, ko = kernels.rope(q, k, table, pos)
    cs = table[pos].double()[:, None]
    for x, y in ((q, qo), (k, ko)):
        a, b = x.double()[..., :32], x.double()[..., 32:]
        want = torch.cat([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]], -1)
        rotary_close(y, want.cpu(), x.cpu(), dtype)
    alone, none = kernels.rope(q, None, table, pos)
    assert none is None and torch.equal(alone, qo)


@pytest.mark.parametrize("shift", [1, 2, 4])
def test_rotary_rows_off_the_16_byte_boundary(shift):
    g = torch.Generator().manual_seed(shift)
    store = torch.randn(40 * 67 + 8, generator=g).bfloat16().to(DEV)
    q = store[shift:].as_strided((10, 4, 64), (4 * 67, 67, 1))  # rows of odd distance and start
    table = attention.rotary_table(64, 64)
    pos = torch.arange(10, device=DEV, dtype=torch.int32)
    qo, _ = kernels.rope(q, None, table, pos)
    want, _ = kernels.rope(q.contiguous(), None, table, pos)
    assert torch.equal(qo, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(dtype, interleaved):
    g = torch.Generator().manual_seed(3)
    D, rot, B, T = 64, 48, 2, 9
    table = attention.rotary_table(50, rot, 1000.0, dict(rope_type="linear", factor=4.0), device=DEV)
    pos = torch.randint(0, 50, (B, T), generator=g)
    pos[1, 3] = -5
    q = torch.randn(B, T, 6, D, generator=g).to(dtype).to(DEV).requires_grad_()
    k = torch.randn(B, T, 2, D, generator=g).to(dtype).to(DEV).requires_grad_()
    dq = torch.randn(B, T, 6, D, generator=g).to(dtype).to(DEV)
    # a gradient that autograd hands over as a broadcast view
    dk = torch.randn(B, T, 2, 1, generator=g).to(dtype).to(DEV).expand(B, T, 2, D)
    qo, ko = attention.apply_rotary(q, k, table, pos.to(DEV), interleaved)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    rotary_close(gq, oatt.rotary(dq.cpu(), table.cpu(), pos, interleaved, inverse=True), dq.cpu(), dtype)
    rotary_close(gk, oatt.rotary(dk.cpu(), table.cpu(), pos, interleaved, inverse=True), dk.cpu(), dtype)
    # against differences: the turn is linear, so <f(q + v) - f(q), d> = <v, grad> up to the rounding of f
    if dtype == torch.float32:
        v = torch.randn(B, T, 6, D, generator=g).to(DEV)
        f1, _ = kernels.rope(q.detach() + v, None, table, pos.to(DEV), interleaved)
        lhs, rhs = ((f1 - qo.detach()).double() * dq).sum(), (v.double() * gq).sum()
        scale = (v.double().abs() * gq.abs()).sum()
        assert abs(float(lhs - rhs)) <= 2.0 ** -20 * float(scale)
    # one output alone
    (gq1,) = torch.autograd.grad(attention.apply_rotary(q, k, table, pos.to(DEV), interleaved)[0], (q,), dq)
    assert torch.equal(gq1, gq)


def test_rotary_position_beyond_the_table_is_reported():
    table = attention.rotary_table(8, 32)
    x = torch.ones(3, 1, 32, device=DEV)
    y, _ = kernels.rope(x, None, table, torch.tensor([7, 8, 2 ** 30], device=DEV))
    assert bool((y[1:] == 0).all()) and bool((y[0] != 0).any())
    assert kernels.device_status(clear=True) != 0


@pytest.mark.parametrize("T,Hq,Hkv,D,page,rot,interleaved,head_major", [
    (1, 8, 2, 64, 16, 64, False, False),
    (5, 5, 5, 80, 24, 40, True, True),
    (3, 4, 1, 8, 1, 8, False, False),
    (16, 16, 2, 128, 7, 128, False, True),
])
def test_rotary_append(T, Hq, Hkv, D, page, rot, interleaved, head_major):
    lens = [0, 1, 2 * page - 1, 37]
    kc, vc, table, L, g = make_cache(lens, T, Hkv, D, page, 11, head_major, fill=0.5)
    qkv = torch.randn(len(lens), T, Hq + 2 * Hkv, D, generator=g).bfloat16()
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
    pos = (L[:, None] + torch.arange(T)).to(torch.int32)
    pos[1, T - 1] = -1
    cs = attention.rotary_table(max(lens) + T + 1, rot, device="cpu")
    gk, gv = kc.to(DEV), vc.to(DEV)
    assert gk.stride() == kc.stride()
    qd = qkv.to(DEV)
    qo = kernels.rope_append(qd[:, :, :Hq], qd[:, :, Hq:Hq + Hkv], qd[:, :, Hq + Hkv:], *to(cs, pos), gk, gv,
                             *to(table, L), interleaved=interleaved)
    rotary_close(qo, oatt.rotary(q, cs, pos, interleaved), q, torch.bfloat16)
    kt = oatt.rotary(k, cs, pos, interleaved)
    want_k, want_v = kc.double(), vc.clone()
    for b, n in enumerate(lens):
        for t in range(T):
            if pos[b, t] >= 0:
                at = int(table[b, (n + t) // page]), (n + t) % page
                want_k[at], want_v[at] = kt[b, t], v[b, t]
    rotary_close(gk, want_k, k, torch.bfloat16)
    assert torch.equal(gv.cpu(), want_v)


def test_append_beyond_the_cache_is_dropped_and_reported():
    kc, vc, table, L, g = make_cache([6, 3], 2, 1, 32, 4, 5, fill=0.0)
    q = torch.randn(2, 2, 1, 32, generator=g).bfloat16().to(DEV)
    pos = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    cs = attention.rotary_table(16, 32)
    for bad_len, bad_page in ((7, None), (-1, None), (6, 99), (6, -3)):
        k0, v0 = kc.to(DEV), vc.to(DEV)
        lens, tab = L.clone(), table.clone()
        lens[0] = bad_len
        if bad_page is not None:
            tab[0, 1] = bad_page
        kernels.rope_append(q, q, q, cs, pos, k0, v0, *to(tab, lens))
        assert kernels.device_status(clear=True) != 0
        # the other sequence is as it should be
        j = int(L[1])
        assert torch.equal(v0.cpu()[int(table[1, j // 4]), j % 4], q[1, 0].cpu())


# ---------------------------------------------------------------- tree attention
def check_attention(q, kc, vc, table, lens, pos, mask=None, sinks=None, window=0, scale=None, seed=0):
    want, lse, spread = oatt.tree_attention(q, kc, vc, table, lens, pos, mask, sinks, window, scale)
    args = to(q, kc, vc, table, lens, pos)
    got, glse = kernels.tree_attention(*args, tree_mask=None if mask is None else mask.to(DEV),
                                       sinks=None if sinks is None else sinks.to(DEV), window=window, scale=scale)
    err = (got.double().cpu() - want).abs()
    tol = 2.0 ** -8 * (want.abs() + spread) + 1e-6
    assert bool((err <= tol).all()), (err / tol).max()
    glse = glse.double().cpu()
    assert torch.equal(glse == -math.inf, lse == -math.inf)
    fin = lse > -math.inf
    assert bool(((glse - lse)[fin].abs() <= 2e-5 * (1 + lse[fin].abs())).all())
    assert bool((got.cpu()[(want == 0).all(-1)] == 0).all())
    return got, glse


ATTENTION = [
    # T, Hq, Hkv, D, page, lens, window, sinks, tree
    (1, 8, 1, 64, 16, [300], 0, True, "chain"),
    (1, 1, 1, 64, 16, [0], 0, False, "chain"),
    (1, 8, 2, 64, 1, [0, 1, 2, 63, 64, 65], 0, True, "chain"),
    (1, 64, 8, 64, 64, [129, 5], 0, True, "chain"),
    (2, 6, 2, 128, 5, [31, 32, 33], 0, False, "each"),
    (7, 10, 2, 80, 24, [0, 1, 100, 47], 0, True, "each"),
    (13, 20, 4, 80, 24, [140, 0, 1, 200], 32, True, "each"),
    (5, 4, 4, 8, 3, [9, 17], 4, False, "each"),
    (16, 16, 2, 64, 64, [257, 3], 0, False, "shared"),
    (33, 4, 2, 32, 16, [40, 0], 0, True, "each"),
    (64, 4, 2, 128, 32, [130, 64], 0, False, "shared"),
    (64, 8, 1, 64, 16, [200], 50, True, "each"),
    (100, 2, 2, 96, 16, [70], 0, False, "each"),
    (256, 1, 1, 64, 128, [10], 0, True, "shared"),
    (3, 40, 1, 64, 8, [90, 11], 0, True, "chain"),
    (9, 24, 8, 40, 10, [55], 1, False, "each"),
]


@pytest.mark.parametrize("T,Hq,Hkv,D,page,lens,window,sinks,tree", ATTENTION)
@pytest.mark.parametrize("head_major", [False, True])
def test_tree_attention(T, Hq, Hkv, D, page, lens, window, sinks, tree, head_major):
    kc, vc, table, L, g = make_cache(lens, T, Hkv, D, page, T + D, head_major)
    mask, pos = make_tree(len(lens), T, lens, g, unused=min(2, T - 1))
    if tree == "chain":
        mask, pos = None, torch.where(pos >= 0, L[:, None] + torch.arange(T), -1).to(torch.int32)
    if tree == "shared":
        mask = mask[0]
        pos = torch.where(pos >= 0, L[:, None] + mask.sum(-1) - 1, -1).to(torch.int32)
    poison_unused(kc, table, L, pos)
    poison_unused(vc, table, L, pos)
    q = (torch.randn(len(lens), T, Hq, D, generator=g) * 2).bfloat16()
    s = torch.randn(Hq, generator=g) if sinks else None
    check_attention(q, kc, vc, table, L, pos, mask, s, window)


MORE_ROWS = [
    # pages without boxes: tiles of 32 rows, full and not, and of 16 at a head of 128
    (4, 8, 1, 32, 12, [129, 64], 0, False, "each"),
    (3, 20, 2, 64, 5, [100, 0], 9, True, "shared"),
    (9, 8, 1, 64, 20, [77], 0, True, "chain"),
    (5, 8, 1, 128, 10, [63, 64], 0, True, "each"),
    # rows to a kv head: 24 and 32; 165, 200, 384 and 512 (pairs of row tiles, the last half empty)
    (2, 12, 1, 64, 16, [70, 0], 0, True, "each"),
    (4, 8, 1, 32, 8, [129, 64], 0, False, "each"),
    (33, 40, 8, 128, 16, [140], 0, True, "each"),
    (40, 10, 2, 128, 8, [3, 200], 0, False, "shared"),
    (64, 24, 4, 128, 32, [127], 60, True, "each"),
    (128, 4, 1, 64, 64, [65, 0], 0, True, "chain"),
]


@pytest.mark.parametrize("T,Hq,Hkv,D,page,lens,window,sinks,tree", ATTENTION + MORE_ROWS)
def test_tree_attention_with_its_keys_cut(T, Hq, Hkv, D, page, lens, window, sinks, tree):
    """The same with a page table that reaches far: the keys may then be cut into pieces of
    several CTAs and joined (without a window), however few there are."""
    kc, vc, table, L, g = make_cache(lens, T, Hkv, D, page, T + D)
    mask, pos = make_tree(len(lens), T, lens, g, unused=min(3, T - 1))
    if tree == "chain":
        mask, pos = None, torch.where(pos >= 0, L[:, None] + torch.arange(T), -1).to(torch.int32)
    if tree == "shared":
        mask = mask[0]
        pos = torch.where(pos >= 0, L[:, None] + mask.sum(-1) - 1, -1).to(torch.int32)
    poison_unused(kc, table, L, pos)
    poison_unused(vc, table, L, pos)
    table = torch.cat([table, torch.zeros(len(lens), 5000 // page + 1, dtype=torch.int32)], 1)
    q = (torch.randn(len(lens), T, Hq, D, generator=g) * 2).bfloat16()
    s = torch.randn(Hq, generator=g) if sinks else None
    check_attention(q, kc, vc, table, L, pos, mask, s, window)


@pytest.mark.parametrize("T,Hq,Hkv,D,page,lens,window,sinks,tree", MORE_ROWS)
def test_tree_attention_of_more_rows(T, Hq, Hkv, D, page, lens, window, sinks, tree):
    kc, vc, table, L, g = make_cache(lens, T, Hkv, D, page, T + D, head_major=True)
    mask, pos = make_tree(len(lens), T, lens, g, unused=1)
    poison_unused(kc, table, L, pos)
    poison_unused(vc, table, L, pos)
    q = (torch.randn(len(lens), T, Hq, D, generator=g) * 2).bfloat16()
    s = torch.randn(Hq, generator=g) if sinks else None
    check_attention(q, kc, vc, table, L, pos, mask, s, window)


@pytest.mark.parametrize("B,T,Hq,Hkv,D,page,far,window", [
    (300, 1, 4, 2, 32, 8, False, 0), (300, 1, 4, 2, 32, 8, True, 0), (257, 2, 4, 1, 64, 3, True, 5),
    (140, 5, 8, 1, 64, 8, False, 0), (140, 5, 8, 1, 64, 8, True, 0), (129, 5, 8, 1, 128, 256, True, 0),
])
def test_tree_attention_of_many_sequences(B, T, Hq, Hkv, D, page, far, window):
    """More sequences than one step of the search for a CTA's range takes."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 12, (B,), generator=g).tolist()
    kc, vc, table, L, g = make_cache(lens, T, Hkv, D, page, B + T)
    mask, pos = make_tree(B, T, lens, g, unused=min(1, T - 1))
    poison_unused(kc, table, L, pos)
    poison_unused(vc, table, L, pos)
    if far:
        table = torch.cat([table, torch.zeros(B, 600 // page + 1, dtype=torch.int32)], 1)
    q = (torch.randn(B, T, Hq, D, generator=g) * 2).bfloat16()
    check_attention(q, kc, vc, table, L, pos, mask, torch.randn(Hq, generator=g), window)


@pytest.mark.parametrize("T,Hq,Hkv,D,scale", [(20, 8, 1, 64, 30.0), (40, 8, 1, 128, 30.0), (20, 8, 1, 64, -3.0), (1, 8, 1, 64, -3.0)])
def test_rows_whose_maximum_keeps_moving(T, Hq, Hkv, D, scale):
    """Scores of hundreds that grow along the keys: the reference moves, and the sums and
    outputs that were relative to it are rescaled; negative scales too.  The weights are
    taken against fp32 scores, which are off by up to 2^-24 D max|q k| scale here."""
    n, page = 700, 16
    kc, vc, table, L, g = make_cache([n], T, Hkv, D, page, 3)
    for j in range(n + T):
        kc[int(table[0, j // page]), j % page] *= 0.02 + 0.98 * j / n
    pos = (L[:, None] + torch.arange(T)).to(torch.int32)
    q = torch.randn(1, T, Hq, D, generator=g).bfloat16()
    want, lse, spread = oatt.tree_attention(q, kc, vc, table, L, pos, scale=scale / D ** 0.5)
    got, glse = kernels.tree_attention(*to(q, kc, vc, table, L, pos), scale=scale / D ** 0.5)
    off = 2.0 ** -24 * D * 16 * abs(scale) / D ** 0.5 * 4      # |q k| of single products up to 16, sums in fp32
    tol = (2.0 ** -8 + 2 * off) * (want.abs() + spread) + 1e-6
    assert bool(((got.double().cpu() - want).abs() <= tol).all())
    assert bool(((glse.double().cpu() - lse).abs() <= off + 1e-6 * lse.abs()).all())


def test_rows_that_attend_nothing():
    """A token whose mask is empty, with and without sinks; unused tokens; a whole sequence of them."""
    T, lens = 4, [0, 0, 5]
    kc, vc, table, L, g = make_cache(lens, T, 2, 64, 4, 8)
    q = torch.randn(3, T, 4, 64, generator=g).bfloat16()
    mask = torch.zeros(3, T, T, dtype=torch.bool)
    mask[:, 1, 1] = mask[:, 3, 1] = True
    pos = L[:, None].repeat(1, T).to(torch.int32)
    pos[1] = -1
    pos[2, 0] = -7
    for c in (kc, vc):
        poison_unused(c, table, L, pos)
    for sinks in (None, torch.tensor([0.5, -math.inf, 30.0, -30.0])):
        out, lse = check_attention(q, kc, vc, table, L, pos, mask, sinks)
        assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())
        if sinks is not None:
            assert lse[0, 0, 0] == pytest.approx(0.5) and lse[0, 0, 1] == -math.inf


def test_keys_no_row_attends_may_hold_anything():
    """NaN and infinity before a window, in unused drafts and behind the last slot are not seen."""
    T, lens, W = 3, [200, 90], 40
    kc, vc, table, L, g = make_cache(lens, T, 1, 64, 16, 9)
    for c in (kc, vc):
        for b, n in enumerate(lens):
            for j in range(0, n - W + 1):
                c[int(table[b, j // 16]), j % 16] = math.inf if j % 2 else math.nan
    pos = (L[:, None] + torch.arange(T)).to(torch.int32)
    q = torch.randn(2, T, 8, 64, generator=g).bfloat16()
    check_attention(q, kc, vc, table, L, pos, None, None, W)


def test_a_key_that_only_some_rows_attend_may_be_infinite():
    """A drafted key whose scores are infinite is masked by selection, not by arithmetic."""
    T, lens = 2, [20]
    kc, vc, table, L, g = make_cache(lens, T, 1, 64, 16, 10)
    kc[int(table[0, 21 // 16]), 21 % 16] = math.inf
    pos = (L[:, None] + torch.arange(T)).to(torch.int32)
    q = torch.ones(1, T, 8, 64).bfloat16()
    got, _ = kernels.tree_attention(*to(q, kc, vc, table, L, pos))
    want, _, spread = oatt.tree_attention(q[:, :1], kc, vc, table, L, pos[:, :1])
    assert bool(((got[:, 0].double().cpu() - want[:, 0]).abs() <= 2.0 ** -8 * (want[:, 0].abs() + spread[:, 0])).all())


def test_large_scores_and_equal_scores():
    T, lens = 1, [333]
    kc, vc, table, L, g = make_cache(lens, T, 1, 64, 16, 12)
    pos = L[:, None].to(torch.int32).clone()
    q = torch.randn(1, 1, 8, 64, generator=g).bfloat16()
    check_attention(q, kc, vc, table, L, pos, scale=20.0)
    check_attention(torch.zeros_like(q), kc, vc, table, L, pos)
    check_attention(q, kc, vc, table, L, pos, scale=0.0, sinks=torch.full((8,), 80.0))


@pytest.mark.parametrize("T,Hq,Hkv,D", [(1, 8, 1, 64), (8, 8, 1, 128), (40, 8, 1, 64)])
def test_long_sequences_are_split_and_joined(T, Hq, Hkv, D):
    """Lengths that many CTAs share, beside ones inside one CTA, against fp64 on the GPU; twice the same bits."""
    lens = [20011, 17, 4096, 0]
    page, g = 32, torch.Generator(device=DEV).manual_seed(1)
    P = pages_for(max(lens) + T, page)
    kc = torch.randn(4 * P, page, Hkv, D, generator=g, device=DEV).bfloat16()
    vc = torch.randn(4 * P, page, Hkv, D, generator=g, device=DEV).bfloat16()
    table = torch.randperm(4 * P, generator=g, device=DEV).reshape(4, P).to(torch.int32)
    L = torch.tensor(lens, dtype=torch.int32, device=DEV)
    pos = (L[:, None] + torch.arange(T, device=DEV)).to(torch.int32)
    q = torch.randn(4, T, Hq, D, generator=g, device=DEV).bfloat16()
    out, lse = kernels.tree_attention(q, kc, vc, table, L, pos)
    again = kernels.tree_attention(q, kc, vc, table, L, pos)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    for b, n in enumerate(lens):
        k = kc[table[b].long()].reshape(-1, D)[: n + T].double()
        v = vc[table[b].long()].reshape(-1, D)[: n + T].double()
        x = torch.einsum("thd,nd->thn", q[b].double(), k) * D ** -0.5
        see = torch.arange(n + T, device=DEV) <= pos[b][:, None]
        x = x.masked_fill(~see[:, None], -math.inf)
        w = x.softmax(-1)
        want, spread = w @ v, w @ v.abs()
        assert bool(((out[b].double() - want).abs() <= 2.0 ** -8 * (want.abs() + spread)).all())
        assert bool(((lse[b].double() - x.logsumexp(-1)).abs() <= 4e-5).all())


@pytest.mark.parametrize("T", [1, 40])
def test_cache_beyond_32_bit_offsets(T):
    """Pages whose offsets pass 2^31 elements (and 2^32 bytes)."""
    page, Hkv, D, n = 64, 8, 64, 100
    pages = (1 << 31) // (page * Hkv * D) + 8
    kc = torch.zeros(pages, page, Hkv, D, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros(pages, page, Hkv, D, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(2)
    table = torch.tensor([[pages - 1, 3, pages - 4]], dtype=torch.int32)
    small = torch.randn(2, 3, page, Hkv, D, generator=g).bfloat16()
    L = torch.tensor([n], dtype=torch.int32)
    pos = (L[:, None] + torch.arange(T)).to(torch.int32)
    q = torch.randn(1, T, 8, D, generator=g).bfloat16()
    for i, p in enumerate(table[0].tolist()):
        kc[p], vc[p] = small[0, i].to(DEV), small[1, i].to(DEV)
    got, lse = kernels.tree_attention(q.to(DEV), kc, vc, *to(table, L, pos))
    same = torch.arange(3, dtype=torch.int32)[None]
    want, wlse = kernels.tree_attention(*to(q, small[0], small[1], same, L, pos))
    assert torch.equal(got, want) and torch.equal(lse, wlse)
    qo = kernels.rope_append(q.to(DEV), q.to(DEV), q.to(DEV), attention.rotary_table(256, D), pos.to(DEV), kc, vc,
                             *to(table, L))
    j = n + T - 1
    assert torch.equal(vc[int(table[0, j // page]), j % page].cpu(), q[0, T - 1]) and qo.shape == q.shape
    scores = torch.zeros(1, Hkv, 3 * page, device=DEV)
    a = kernels.kv_scores_add(scores, q.to(DEV), lse, kc, *to(table, L))
    kept, _, _ = kernels.kv_evict(kc, vc, *to(table, L), a, 64, torch.tensor([[pages - 2]], dtype=torch.int32, device=DEV))
    i = int(kept[0, 5, 9])
    assert torch.equal(kc[pages - 2, 9, 5], kc[int(table[0, i // page]), i % page, 5])
    del kc, vc
    torch.cuda.empty_cache()


def test_attention_on_another_stream_and_in_a_graph():
    T, lens = 3, [77, 130]
    kc, vc, table, L, g = make_cache(lens, T, 2, 64, 16, 21)
    pos = (L[:, None] + torch.arange(T)).to(torch.int32)
    q = torch.randn(2, T, 8, 64, generator=g).bfloat16()
    args = to(q, kc, vc, table, L, pos)
    want, wlse = kernels.tree_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, lse = kernels.tree_attention(*args)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, wlse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = kernels.tree_attention(*args)
    args[0].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    again, _ = kernels.tree_attention(*args)
    assert torch.equal(out, again)


def test_bad_lengths_and_pages_are_reported_and_read_nothing_outside():
    T = 2
    kc, vc, table, L, g = make_cache([10, 20], T, 1, 64, 8, 22, fill=0.0)
    pos = (L[:, None] + torch.arange(T)).to(torch.int32)
    q = torch.randn(2, T, 4, 64, generator=g).bfloat16()
    want, _ = kernels.tree_attention(*to(q, kc, vc, table, L, pos))
    for field, value in (("len", 10 ** 6), ("len", -4), ("page", 10 ** 6), ("page", -1)):
        lens, tab = L.clone(), table.clone()
        if field == "len":
            lens[0] = value
        else:
            tab[0, 0] = value
        got, _ = kernels.tree_attention(*to(q, kc, vc, tab, lens, pos))
        assert kernels.device_status(clear=True) != 0
        assert torch.equal(got[1], want[1])


# ---------------------------------------------------------------- commit, scores, eviction
@pytest.mark.parametrize("page,D,head_major", [(16, 64, False), (3, 128, True), (24, 80, False)])
def test_tree_commit(page, D, head_major):
    T, lens = 9, [0, 5, 31]
    kc, vc, table, L, _ = make_cache(lens, T, 2, D, page, 31, head_major, fill=0.25)
    acc = torch.tensor([[0, 1, 2, 3], [1, 4, 8, -1], [-1, -1, -1, -1]], dtype=torch.int32)
    k, v = kc.to(DEV), vc.to(DEV)
    kernels.tree_commit(k, v, *to(table, L, acc), drafted=T)
    for c, d in ((kc, k), (vc, v)):
        want = c.clone()
        for b, n in enumerate(lens):
            for i, u in enumerate(acc[b].tolist()):
                if u >= 0:
                    want[int(table[b, (n + i) // page]), (n + i) % page] = oatt.slot(c, table, b, n + u)
        assert torch.equal(d.cpu(), want)


def test_tree_commit_refuses_a_list_that_does_not_ascend():
    kc, vc, table, L, _ = make_cache([3, 4], 5, 1, 32, 4, 32, fill=0.0)
    for row in ([2, 1, -1], [1, 1, 2], [-1, 2, 3], [0, 5, -1]):
        k, v = kc.to(DEV), vc.to(DEV)
        acc = torch.tensor([row, [1, 3, -1]], dtype=torch.int32)
        kernels.tree_commit(k, v, *to(table, L, acc), drafted=5)
        assert kernels.device_status(clear=True) != 0
        for j in range(8):
            assert torch.equal(oatt.slot(k.cpu(), table, 0, j), oatt.slot(kc, table, 0, j))
        assert torch.equal(oatt.slot(k.cpu(), table, 1, 4), oatt.slot(kc, table, 1, 5))


@pytest.mark.parametrize("T,A,Hq,Hkv,D,page,lens", [
    (1, 1, 8, 1, 64, 16, [0, 1, 40, 600]),
    (6, 6, 4, 2, 32, 5, [7, 30]),
    (11, 4, 10, 2, 80, 24, [0, 33, 100]),
    (8, 3, 12, 4, 128, 16, [63, 17]),
    (3, 3, 2, 2, 96, 7, [64, 200]),
])
def test_kv_scores(T, A, Hq, Hkv, D, page, lens):
    kc, _, table, L, g = make_cache(lens, T, Hkv, D, page, T + D)
    B, cap = len(lens), table.shape[1] * page
    q = torch.randn(B, T, Hq, D, generator=g).bfloat16()
    lse = torch.randn(B, T, Hq, generator=g) + 3
    lse[0, 0, 0] = -math.inf  # a row that attended nothing gives nothing
    acc = None
    if A < T:
        acc = torch.full((B, A), -1, dtype=torch.int32)
        for b in range(B):
            m = A if b == 0 else 1 + b % A
            acc[b, :m] = torch.randperm(T, generator=g)[:m].sort().values.to(torch.int32)
    scores = torch.rand(B, Hkv, cap, generator=g)
    for cut in (cap, max(1, cap - page // 2 - 1)):  # a capacity of scores below that of the table
        s = scores[:, :, :cut].contiguous()
        want = oatt.kv_scores(s, q, lse, kc, table, L, acc)
        gs = s.to(DEV)
        a = None if acc is None else acc.to(DEV)
        out = kernels.kv_scores_add(gs, *to(q, lse, kc, table, L), accepted=a)
        assert torch.equal(gs.cpu(), s)
        assert bool(((out.double().cpu() - want).abs() <= 2e-5 * want.abs() + 1e-6).all())
        same = kernels.kv_scores_add(gs, *to(q, lse, kc, table, L), accepted=a, out=gs)
        assert same is gs and torch.equal(gs, out)


@pytest.mark.parametrize("T,A,Hq,Hkv,D,page,lens", [
    (3, 3, 8, 1, 64, 16, [0, 125, 126, 400]),       # 24 rows: products of 16 keys
    (5, 4, 7, 1, 64, 8, [127, 128, 0]),             # 28 rows: tiles of 128, padded to 32
    (9, 9, 8, 4, 32, 64, [1, 300]),                 # 18
    (3, 3, 24, 4, 128, 128, [0, 253]),              # 18 at a head of 128
    (16, 16, 16, 2, 64, 32, [511, 5]),              # 128
    (20, 17, 8, 1, 96, 16, [130, 64, 700]),         # 136: two launches, the second of 8 rows
    (40, 33, 16, 2, 128, 48, [77, 129]),            # 264: three
    (2, 2, 128, 1, 64, 16, [1000]),                 # one token to a launch
    (40, 33, 16, 2, 128, 12, [77, 129]),            # pages without boxes
    (3, 2, 4, 2, 64, 256, [6] * 150),               # more sequences than one step of the search
    (5, 4, 8, 1, 64, 256, [3] * 131),
])
def test_kv_scores_of_many_rows(T, A, Hq, Hkv, D, page, lens):
    test_kv_scores(T, A, Hq, Hkv, D, page, lens)


def test_infinite_keys_reach_only_the_rows_that_count():
    """A key of infinities in view of every row: tokens not accepted and rows that attended
    nothing add nothing, whatever they would multiply."""
    T, n, page, D = 4, 300, 16, 64
    kc, _, table, L, g = make_cache([n], T, 1, D, page, 5)
    kc[int(table[0, 7 // page]), 7 % page] = -math.inf
    q = torch.rand(1, T, 8, D, generator=g).bfloat16() + 1
    lse = torch.full((1, T, 8), 5.0)
    lse[0, 1, 3] = -math.inf
    acc = torch.tensor([[0, 1, 3, -1]], dtype=torch.int32)
    s = torch.zeros(1, 1, table.shape[1] * page)
    out = kernels.kv_scores_add(*to(s, q, lse, kc, table, L), accepted=acc.to(DEV)).cpu()
    assert bool(out.isfinite().all()) and float(out[0, 0, 7]) == 0


def test_kv_scores_of_more_rows_than_fit_at_once():
    """Many query heads and tokens: the rows are taken in several launches, with the same sums."""
    T, Hq, D, page, n = 40, 64, 128, 16, 50
    kc, _, table, L, g = make_cache([n], T, 1, D, page, 77)
    q = torch.randn(1, T, Hq, D, generator=g).bfloat16()
    lse = torch.full((1, T, Hq), 5.0)
    s = torch.zeros(1, 1, table.shape[1] * page)
    out = kernels.kv_scores_add(*to(s, q, lse, kc, table, L)).double().cpu()
    k = torch.stack([oatt.slot(kc, table, 0, j)[0] for j in range(n + T)]).double()
    x = torch.einsum("thd,nd->thn", q[0].double(), k) * D ** -0.5 - 5.0
    see = torch.arange(n + T) <= n + torch.arange(T)[:, None]
    want = torch.where(see[:, None], x.exp(), 0.0).sum((0, 1))
    assert bool(((out[0, 0, : n + T] - want).abs() <= 2e-5 * want).all()) and bool((out[0, 0, n + T:] == 0).all())


def test_scores_of_attention_sum_to_the_rows():
    """Each row's weights sum to one (less the sink's), so a step adds Hq/Hkv per token and kv head."""
    lens = [37, 500]
    kc, vc, table, L, g = make_cache(lens, 1, 2, 64, 16, 41)
    pos = L[:, None].to(torch.int32).clone()
    q = torch.randn(2, 1, 16, 64, generator=g).bfloat16()
    args = to(q, kc, vc, table, L, pos)
    _, lse = kernels.tree_attention(*args)
    out = kernels.kv_scores_add(torch.zeros(2, 2, table.shape[1] * 16, device=DEV), args[0], lse, args[1], args[3], args[4])
    assert bool(((out.double().sum(-1) - 8).abs() <= 1e-3).all())


def check_evict(lens, scores, budget, first, last, page, D, head_major=False, same_pages=()):
    B, Hkv, cap = scores.shape
    kc, vc, table, L, g = make_cache(lens, 0, Hkv, D, page, budget, head_major, spare=B * pages_for(budget, page) + 1,
                                     fill=0.125)
    free = [p for p in range(kc.shape[0]) if p not in set(table.flatten().tolist())]
    width = pages_for(min(budget, max(cap, 1)), page)
    out_table = torch.tensor(free[: B * width], dtype=torch.int32).reshape(B, width)
    for b in same_pages:
        out_table[b] = table[b, :width]
    k, v = kc.to(DEV), vc.to(DEV)
    kept, new_lens, new_scores = kernels.kv_evict(k, v, *to(table, L, scores), budget, out_table.to(DEV), first, last)
    want = oatt.evict(scores, lens, budget, first, last)
    wk, wv, ws = kc.clone(), vc.clone(), torch.zeros(B, Hkv, width * page)
    for b in range(B):
        assert int(new_lens[b]) == min(lens[b], budget)
        for h in range(Hkv):
            row = want[b][h]
            assert kept[b, h].tolist() == row + [-1] * (budget - len(row)), (b, h)
            for i, j in enumerate(row):
                at = int(out_table[b, i // page]), i % page
                wk[at][h], wv[at][h] = oatt.slot(kc, table, b, j)[h], oatt.slot(vc, table, b, j)[h]
                ws[b, h, i] = scores[b, h, j]
    assert torch.equal(k.cpu(), wk) and torch.equal(v.cpu(), wv)
    assert torch.equal(torch.nan_to_num(new_scores.cpu(), nan=-7.0), torch.nan_to_num(ws, nan=-7.0))


@pytest.mark.parametrize("lens,budget,first,last,page,D,head_major", [
    ([100, 30, 0, 1, 64], 40, 4, 8, 16, 64, False),
    ([100, 99], 1, 0, 0, 7, 32, True),
    ([50, 77], 50, 25, 25, 24, 80, False),
    ([500], 499, 0, 0, 16, 128, False),
    ([33, 200], 64, 0, 64, 16, 64, True),
    ([20], 64, 2, 2, 16, 8, False),
])
def test_kv_evict(lens, budget, first, last, page, D, head_major):
    g = torch.Generator().manual_seed(budget)
    cap = pages_for(max(lens), page) * page
    scores = torch.randn(len(lens), 3, cap, generator=g)
    check_evict(lens, scores, budget, first, last, page, D, head_major)
    # many equal scores: the lowest slots go first
    check_evict(lens, (scores * 2).round() / 2, budget, first, last, page, D, head_major)
    check_evict(lens, torch.zeros_like(scores), budget, first, last, page, D, head_major)


@pytest.mark.parametrize("lens,budget,first,last", [
    ([5000, 4097], 100, 4, 8),              # two CTAs of a cluster to an item, then four and eight
    ([9001], 130, 0, 33),
    ([17000, 16385, 3], 300, 5, 0),
    ([25600, 24449] + [7] * 24, 90, 2, 9),  # more items than SMs / 2, scores not held
    ([200001], 257, 4, 64),                 # nor by eight CTAs
])
def test_kv_evict_of_long_caches(lens, budget, first, last):
    g = torch.Generator().manual_seed(len(lens))
    cap = pages_for(max(lens), 64) * 64
    scores = torch.randn(len(lens), 3, cap, generator=g)
    scores[0, 1] = (scores[0, 1] * 3).round()       # runs of equal scores over all the CTAs
    scores[0, 2] = scores[0, 2].clamp(max=0.25)     # the threshold itself is met by many
    check_evict(lens, scores, budget, first, last, 64, 8)
    if len(lens) == 1:                              # scores that start off 16 bytes, odd capacity
        check_evict(lens, scores[:, :, :lens[0]], budget, first, last, 64, 8)


def test_kv_evict_special_values():
    g = torch.Generator().manual_seed(6)
    scores = torch.randn(2, 2, 64, generator=g)
    scores[0, 0, ::3] = math.nan
    scores[0, 1, ::5] = math.inf
    scores[1, 0, 1::2] = -math.inf
    scores[1, 1, :32] = -0.0
    scores[1, 1, 32:] = 0.0
    check_evict([64, 60], scores, 30, 2, 3, 8, 32)
    check_evict([64, 60], scores, 62, 0, 1, 8, 32, same_pages=(1,))


@pytest.mark.parametrize("n", [8192, 8193, 70001])
def test_kv_evict_over_several_ctas(n):
    g = torch.Generator(device=DEV).manual_seed(n)
    page, D, budget = 128, 32, n // 3
    P, Q = pages_for(n, page), pages_for(budget, page)
    kc = torch.randn(P + Q, page, 1, D, generator=g, device=DEV).bfloat16()
    vc = torch.randn(P + Q, page, 1, D, generator=g, device=DEV).bfloat16()
    order = torch.randperm(P + Q, generator=g, device=DEV).to(torch.int32)
    table, out = order[None, :P].contiguous(), order[None, P:].contiguous()
    scores = torch.randn(1, 1, P * page, generator=g, device=DEV).mul(8).round().div(8)
    L = torch.tensor([n], dtype=torch.int32, device=DEV)
    k0 = kc.clone()
    kept, lens, new = kernels.kv_evict(kc, vc, table, L, scores, budget, out, 5, 100)
    rank = scores[0, 0, :n].clone()
    rank[:5] = rank[n - 100:] = math.inf
    want = rank.sort(descending=True, stable=True).indices[:budget].sort().values
    assert torch.equal(kept[0, 0].long(), want) and int(lens) == budget
    assert torch.equal(new[0, 0, :budget], scores[0, 0][want]) and bool((new[0, 0, budget:] == 0).all())
    i = torch.arange(budget, device=DEV)
    assert torch.equal(kc[out[0].long()[i // page], i % page, 0], k0[table[0].long()[want // page], want % page, 0])


# ---------------------------------------------------------------- refusals that need tensors on the GPU
def test_python_refusals():
    kc, vc, table, L, g = make_cache([10], 2, 2, 64, 8, 1, fill=0.0)
    q = torch.randn(1, 2, 4, 64, generator=g).bfloat16()
    pos = torch.tensor([[10, 11]], dtype=torch.int32)
    q, kc, vc, table, L, pos = to(q, kc, vc, table, L, pos)
    run = kernels.tree_attention
    with pytest.raises(ValueError, match="CUDA tensors only"):
        run(q.cpu(), kc, vc, table, L, pos)
    with pytest.raises(ValueError, match="bf16"):
        run(q.float(), kc, vc, table, L, pos)
    with pytest.raises(ValueError, match="bf16"):
        run(q, kc.float(), vc.float(), table, L, pos)
    with pytest.raises(ValueError, match="one shape"):
        run(q, kc, vc[:, :, :1], table, L, pos)
    with pytest.raises(ValueError, match="multiple"):
        run(q[:, :, :3], kc, vc, table, L, pos)
    with pytest.raises(ValueError, match="positions"):
        run(q, kc, vc, table, L, pos.long())
    with pytest.raises(ValueError, match="page_table"):
        run(q, kc, vc, table.long(), L, pos)
    with pytest.raises(ValueError, match="tree_mask"):
        run(q, kc, vc, table, L, pos, tree_mask=torch.ones(2, 3, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError, match="sinks"):
        run(q, kc, vc, table, L, pos, sinks=torch.zeros(4, device=DEV).bfloat16())
    with pytest.raises(ValueError, match="window"):
        run(q, kc, vc, table, L, pos, window=-1)
    with pytest.raises(ValueError, match="multiples of 8"):
        run(torch.randn(1, 2, 4, 65, device=DEV).bfloat16()[..., :64], kc, vc, table, L, pos)
    with pytest.raises(ValueError, match="table"):
        kernels.rope(q, None, torch.zeros(4, 33, 2, device=DEV), pos)
    with pytest.raises(ValueError, match="positions"):
        kernels.rope(q, None, torch.zeros(4, 32, 2, device=DEV), pos[:, :1])
    with pytest.raises(ValueError, match="budget"):
        kernels.kv_evict(kc, vc, table, L, torch.zeros(1, 2, 16, device=DEV), 4, table, 3, 2)
    with pytest.raises(ValueError, match="output pages"):
        kernels.kv_evict(kc, vc, table, L, torch.zeros(1, 2, 16, device=DEV), 12, table[:, :1])
    with pytest.raises(ValueError, match="accepted"):
        kernels.kv_scores_add(torch.zeros(1, 2, 16, device=DEV), q, torch.zeros(1, 2, 4, device=DEV), kc, table, L,
                              accepted=torch.zeros(1, 3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="scores"):
        kernels.kv_scores_add(torch.zeros(1, 2, 17, device=DEV), q, torch.zeros(1, 2, 4, device=DEV), kc, table, L)


def test_empty_batches():
    kc = torch.zeros(3, 8, 2, 64, dtype=torch.bfloat16, device=DEV)
    table = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
    L = torch.zeros(0, dtype=torch.int32, device=DEV)
    q = torch.zeros(0, 1, 4, 64, dtype=torch.bfloat16, device=DEV)
    out, lse = kernels.tree_attention(q, kc, kc.clone(), table, L, torch.zeros(0, 1, dtype=torch.int32, device=DEV))
    assert out.shape == q.shape and lse.shape == (0, 1, 4)
    x, _ = kernels.rope(q, None, torch.zeros(4, 32, 2, device=DEV), torch.zeros(0, 1, dtype=torch.int32, device=DEV))
    assert x.shape == q.shape
