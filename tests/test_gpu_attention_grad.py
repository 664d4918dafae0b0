"""Gradients of the rotation, of first and second order."""

import pytest
import torch

from blockstreamer_b200 import attention
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
