"""Gradients around the attention half: the rotation's of first and second order, and
the operators that have none, which say so instead of dropping it."""

import types

import pytest
import torch

from blockstreamer_b200 import B200GptOssAttention, PagedKVCache, attention, kernels
from oracle import attention as oatt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("with_k", [False, True])
def test_rotary_second_derivative(dtype, interleaved, with_k):
    """The gradient R^T d is linear in d, so its derivative along w is the turn R w: one
    rounding (2^-8 relative in bf16, 2^-22 with the products and the sum in fp32) as the turn
    itself."""
    g = torch.Generator().manual_seed(4)
    D, rot, B, T = 64, 48, 2, 9
    table = attention.rotary_table(50, rot, 1000.0, device=DEV)
    pos = torch.randint(0, 50, (B, T), generator=g)
    pos[1, 3] = -1

    def make(heads):
        return torch.randn(B, T, heads, D, generator=g).to(dtype).to(DEV).requires_grad_()

    x = [make(6)] + ([make(2)] if with_k else [])
    d = [make(t.shape[2]) for t in x]
    w = [make(t.shape[2]).detach() for t in x]
    y = attention.apply_rotary(x[0], x[1] if with_k else None, table, pos.to(DEV), interleaved)
    first = torch.autograd.grad([t for t in y if t is not None], x, d, create_graph=True)
    plain = torch.autograd.grad(attention.apply_rotary(x[0], None, table, pos.to(DEV), interleaved)[0], x[0], d[0])
    assert torch.equal(first[0], plain[0])
    second = torch.autograd.grad(first, d, w)
    eps = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22
    for got, v in zip(second, w):
        want = oatt.rotary(v.cpu(), table.cpu(), pos, interleaved)
        err = (got.double().cpu() - want).abs()
        assert bool((err <= eps * want.abs() + 2.0 ** -21 * v.double().abs().max().cpu()).all())


def small_cache():
    return PagedKVCache(2, 8, 4, 2, 64, 16, DEV)


def test_operators_without_a_gradient_refuse_the_backward_pass():
    g = torch.Generator().manual_seed(1)
    table = attention.rotary_table(32, 64, device=DEV)
    q, k, v = (torch.randn(2, 3, h, 64, generator=g).bfloat16().to(DEV) for h in (4, 2, 2))
    pos = torch.arange(3, dtype=torch.int32, device=DEV).repeat(2, 1)
    plain_cache = small_cache()
    plain = plain_cache.append(q, k, v, table, pos)
    out0, lse0 = plain_cache.attend(plain, pos)
    assert not plain.requires_grad and not out0.requires_grad and not lse0.requires_grad
    for which in range(3):
        x = [t.clone().requires_grad_(i == which) for i, t in enumerate((q, k, v))]
        cache = small_cache()
        turned = cache.append(*x, table, pos)
        assert torch.equal(turned, plain)
        with pytest.raises(RuntimeError, match="no backward"):
            turned.float().sum().backward()
    cache = small_cache()
    cache.append(q, k, v, table, pos)
    asked = plain.clone().requires_grad_()
    out, lse = cache.attend(asked, pos)
    assert torch.equal(out, out0) and torch.equal(lse, lse0)
    for y in (out, lse):
        with pytest.raises(RuntimeError, match="no backward"):
            torch.autograd.grad(y.float().sum(), asked)
    sinks = torch.zeros(4, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        cache.attend(plain, pos, sinks=sinks)[0].float().sum().backward()
    scores = torch.zeros(2, 2, 16, device=DEV)
    for lse1 in (lse, lse0.clone().requires_grad_()):
        new = kernels.kv_scores_add(scores, plain, lse1, cache.k, cache.page_table, cache.lens)
        assert new.requires_grad
        with pytest.raises(RuntimeError, match="no backward"):
            new.sum().backward()
    with pytest.raises(RuntimeError, match="apply_rotary"):
        kernels.rope(asked, None, table, pos)[0].float().sum().backward()
    with torch.no_grad():
        assert not cache.attend(asked, pos)[0].requires_grad
        assert not kernels.rope(asked, None, table, pos)[0].requires_grad


@pytest.mark.parametrize("trains", ["hidden_states", "weights"])
def test_layer_refuses_the_backward_pass(trains):
    """A training loop that has the layer in it is told, the residual's gradient notwithstanding."""
    cfg = types.SimpleNamespace(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                sliding_window=0, attention_bias=True, layer_types=["full_attention"])
    m = B200GptOssAttention(cfg)
    g = torch.Generator().manual_seed(2)
    m.load_state_dict({n: (torch.randn(p.shape, generator=g) * 0.1).bfloat16() for n, p in m.named_parameters()},
                      assign=True)
    m = m.to(DEV).requires_grad_(trains == "weights")
    x = torch.randn(2, 3, 128, generator=g).bfloat16().to(DEV).requires_grad_(trains == "hidden_states")
    pos = torch.arange(3, dtype=torch.int32, device=DEV).repeat(2, 1)
    table = attention.rotary_table(32, 64, device=DEV)
    out, _, _ = m(x, pos, small_cache(), table)
    with pytest.raises(RuntimeError, match="no backward"):
        (x + out).float().sum().backward()
    with torch.no_grad():
        alone, _, _ = m(x, pos, small_cache(), table)
    assert torch.equal(alone, out)
