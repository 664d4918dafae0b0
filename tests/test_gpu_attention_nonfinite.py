"""Attention where scores or values are not ordinary numbers, against the definition:
a key that a row attends counts with whatever its score is, one that it does not
attend has the weight zero.  Tolerances as for ordinary values: 2^-8 of the output
for its rounding and 2^-8 of the weighted values' magnitudes for the weights'."""

import math

import pytest
import torch

from attention_cases import make_cache
from blockstreamer_b200 import kernels
from oracle import attention as oatt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# (T, Hq, D): rows of a kv head 1, 8, 24, 40 | 80 and 128 | 160 and 256, heads of 64 and 128
ROWS = [(1, 1, 64), (1, 8, 128), (3, 8, 128), (5, 8, 64), (20, 4, 128), (32, 4, 64), (20, 8, 64), (32, 8, 128)]


def to(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


@pytest.fixture(autouse=True)
def status_is_clear():
    kernels.device_status(clear=True)
    yield
    assert kernels.device_status(clear=True) == 0


def chain(L, T):
    return (L[:, None] + torch.arange(T)).to(torch.int32)


def far(table, page, slots):
    """The same table with room for so many slots: items may then be cut between CTAs."""
    return torch.cat([table, torch.zeros(table.shape[0], slots // page + 1, dtype=torch.int32)], 1)


@pytest.mark.parametrize("T,Hq,D", ROWS)
def test_a_masked_value_has_no_weight(T, Hq, D):
    """A drafted value of 2^127 adds nothing to the rows that do not attend it, however small
    a weight other than zero would be (2^-126 of it is 2)."""
    n, page = 64, 16
    T = max(T, 2)
    kc, vc, table, L, g = make_cache([n], T, 1, D, page, T)
    big = [u for u in range(1, T) if u % 16 >= 1]
    for u in big:
        vc[int(table[0, (n + u) // page]), (n + u) % page] = 2.0 ** 127
    pos = chain(L, T)
    mask = torch.zeros(T, T, dtype=torch.bool)
    mask[:, ::16] = True      # every row attends only the drafts that are not big
    q = torch.randn(1, T, Hq, D, generator=g).bfloat16() * 0.1
    want, lse, spread = oatt.tree_attention(q, kc, vc, table, L, pos, mask)
    got, glse = kernels.tree_attention(*to(q, kc, vc, table, L, pos), tree_mask=mask.to(DEV))
    assert bool(((got.double().cpu() - want).abs() <= 2.0 ** -8 * (want.abs() + spread) + 1e-6).all())
    assert bool(((glse.double().cpu() - lse).abs() <= 2e-5 * (1 + lse.abs())).all())


@pytest.mark.parametrize("T,Hq,D", ROWS)
@pytest.mark.parametrize("slots", [0, 5000])
def test_a_key_of_nan_that_is_attended_is_seen_at_every_slot(T, Hq, D, slots):
    page, n = 16, 70
    kc, vc, table, L, g = make_cache([n] * 67, T, 1, D, page, T + D)
    for b in range(66):       # sequence b has it at slot b, the last one nowhere
        kc[int(table[b, b // page]), b % page] = math.nan
    q = torch.randn(67, T, Hq, D, generator=g).bfloat16()
    got, lse = kernels.tree_attention(*to(q, kc, vc, far(table, page, slots) if slots else table, L, chain(L, T)))
    assert bool(got[:66].isnan().all()) and bool(lse[:66].isnan().all())
    assert bool(got[66].isfinite().all()) and bool(lse[66].isfinite().all())
