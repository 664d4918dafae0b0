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


@pytest.mark.parametrize("T,Hq,D", ROWS)
@pytest.mark.parametrize("slots", [0, 5000])
@pytest.mark.parametrize("sinks", [False, True])
def test_a_row_whose_every_score_is_nan_is_nan(T, Hq, D, slots, sinks):
    """A query of NaN, in one sequence's first row; one whose only key is NaN; rows beside
    them keep their values."""
    page, lens = 16, [50, 0, 333]
    kc, vc, table, L, g = make_cache(lens, T, 1, D, page, T + D)
    q = torch.randn(3, T, Hq, D, generator=g).bfloat16()
    q[0, 0, 0] = math.nan
    kc[int(table[1, 0]), 0] = math.nan
    pos = chain(L, T)
    s = torch.randn(Hq, generator=g) if sinks else None
    want, wlse, spread = oatt.tree_attention(q, kc, vc, table, L, pos, None, s)
    got, lse = kernels.tree_attention(*to(q, kc, vc, far(table, page, slots) if slots else table, L, pos), sinks=to(s)[0])
    got, lse = got.double().cpu(), lse.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(lse.isnan(), wlse.isnan())
    assert bool(want[0, 0, 0].isnan().all()) and bool(want[1].isnan().all())
    ok = ~want.isnan()
    assert bool(((got - want)[ok].abs() <= (2.0 ** -8 * (want.abs() + spread) + 1e-6)[ok]).all())


@pytest.mark.parametrize("T,Hq,D", ROWS)
@pytest.mark.parametrize("first,last", [(0, 1024), (1024, 2048), (0, 1500)])
def test_a_piece_of_the_keys_that_is_all_nan_is_not_lost(T, Hq, D, first, last):
    """Keys that several CTAs share, of which some have nothing but NaN."""
    page, n = 64, 3000
    g = torch.Generator(device=DEV).manual_seed(T)
    P = -(-(n + T) // page)
    kc, vc = (torch.randn(P, page, 1, D, generator=g, device=DEV).bfloat16() for _ in range(2))
    kc.view(-1, 1, D)[first:last] = math.nan
    table = torch.arange(P, dtype=torch.int32, device=DEV)[None]
    L = torch.tensor([n], dtype=torch.int32)
    q = torch.randn(1, T, Hq, D, generator=g, device=DEV).bfloat16()
    got, lse = kernels.tree_attention(q, kc, vc, table, *to(L, chain(L, T)))
    assert bool(got.isnan().all()) and bool(lse.isnan().all())


@pytest.mark.parametrize("T,Hq,D", ROWS)
@pytest.mark.parametrize("slots", [0, 5000])
def test_keys_of_minus_infinity_are_as_if_they_were_not_there(T, Hq, D, slots):
    """Scores of -inf: weight zero; where a row has no others, 0 and the sink (or -inf)."""
    page, lens = 16, [200, 40]
    kc, vc, table, L, g = make_cache(lens, T, 1, D, page, T + D)
    q = torch.rand(2, T, Hq, D, generator=g).bfloat16() + 0.5
    for j in range(150):
        kc[int(table[0, j // page]), j % page] = -math.inf
    for j in range(40 + T):
        kc[int(table[1, j // page]), j % page] = -math.inf
    pos = chain(L, T)
    for s in (None, torch.linspace(-1, 1, Hq)):
        want, wlse, spread = oatt.tree_attention(q, kc, vc, table, L, pos, None, s)
        got, lse = kernels.tree_attention(*to(q, kc, vc, far(table, page, slots) if slots else table, L, pos), sinks=to(s)[0])
        got, lse = got.double().cpu(), lse.double().cpu()
        assert bool((got[1] == 0).all()) and bool(got[0].isfinite().all())
        assert bool(((got - want).abs() <= 2.0 ** -8 * (want.abs() + spread) + 1e-6).all())
        on = wlse > -math.inf
        assert torch.equal(lse > -math.inf, on)
        assert bool(((lse - wlse)[on].abs() <= 2e-5 * (1 + wlse[on].abs())).all())
