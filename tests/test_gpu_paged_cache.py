"""What the cache's operators do with lengths, pages and score widths that only the
device can see: the whole pool is compared, the pages of every sequence included.
Nothing here is rounded twice, so everything but the turned keys is compared exactly;
a turned key is one rounding of an fp32 result, 2^-8 relative at most."""

import pytest
import torch

from attention_cases import pages_for
from blockstreamer_b200 import attention, kernels
from oracle import attention as oatt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def to(*ts):
    return [t.to(DEV) for t in ts]


@pytest.fixture(autouse=True)
def status_is_clear():
    kernels.device_status(clear=True)
    yield
    assert kernels.device_status(clear=True) == 0


def two_sequences(page=8, heads=2, D=32, seed=0):
    """Sequence 0 holds 6 slots of pages 3 and 5, sequence 1 18 of pages 0, 7 and 2 (the pool's
    first and last page among them, none of its drafts in those): table rows of 24 slots."""
    g = torch.Generator().manual_seed(seed)
    kc = torch.randn(8, page, heads, D, generator=g).bfloat16()
    vc = torch.randn(8, page, heads, D, generator=g).bfloat16()
    table = torch.tensor([[3, 5, 4], [0, 7, 2]], dtype=torch.int32)
    return kc, vc, table, torch.tensor([6, 18], dtype=torch.int32), g


BAD_LENGTHS = [-1, -2, -2 ** 31, 22, 23, 24, 25, 2 ** 31 - 2]   # T = 3: 21 is the last good one


@pytest.mark.parametrize("bad", BAD_LENGTHS)
def test_commit_leaves_a_sequence_of_bad_length_as_it_is(bad):
    kc, vc, table, L, _ = two_sequences()
    acc = torch.tensor([[1, 2], [0, 2]], dtype=torch.int32)
    lens = torch.tensor([bad, 18], dtype=torch.int32)
    k, v = to(kc, vc)
    kernels.tree_commit(k, v, *to(table, lens, acc), drafted=3)
    assert kernels.device_status(clear=True) != 0
    for c, d in ((kc, k), (vc, v)):
        want = c.clone()
        want[2, 3] = c[2, 4]      # sequence 1: slot 18 + 2 to 18 + 1
        assert torch.equal(d.cpu(), want)


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 8, 99, 2 ** 31 - 1])
@pytest.mark.parametrize("where", [0, 1])
def test_commit_moves_no_row_to_or_from_a_page_outside_the_pool(bad, where):
    kc, vc, table, L, _ = two_sequences()
    acc = torch.tensor([[1, 2], [0, 2]], dtype=torch.int32)
    tab = table.clone()
    tab[0, where] = bad
    k, v = to(kc, vc)
    kernels.tree_commit(k, v, *to(tab, L, acc), drafted=3)
    assert kernels.device_status(clear=True) != 0
    for c, d in ((kc, k), (vc, v)):
        want = c.clone()
        want[2, 3] = c[2, 4]
        if where == 1:            # slot 7 to 6 lies in page 3 alone; slot 8 to 7 would come from the bad page
            want[3, 6] = c[3, 7]
        assert torch.equal(d.cpu(), want)


def append_to(kc, vc, table, lens, g, T=3):
    """Both caches after rows of three tokens, and the turned k and the v that were given."""
    heads, D = kc.shape[2:]
    q, k, v = (torch.randn(2, T, heads, D, generator=g).bfloat16() for _ in range(3))
    pos = torch.arange(T, dtype=torch.int32).repeat(2, 1) + 5
    cs = attention.rotary_table(16, D, device="cpu")
    gk, gv = to(kc, vc)
    kernels.rope_append(*to(q, k, v, cs, pos), gk, gv, *to(table, lens))
    return gk.cpu(), gv.cpu(), oatt.rotary(k, cs, pos), v


def check_append(kc, vc, gk, gv, kt, v, rows):
    """``rows``: (page, slot in it) of every row that was to be written, with its (sequence, token)."""
    wk, wv, written = kc.double(), vc.clone(), torch.zeros(kc.shape, dtype=torch.bool)
    for (page, row), (b, t) in rows.items():
        wk[page, row], wv[page, row], written[page, row] = kt[b, t], v[b, t], True
    assert torch.equal(gv, wv)
    assert torch.equal(gk[~written], kc[~written])
    assert bool(((gk.double() - wk).abs() <= 2.0 ** -8 * wk.abs() + 2.0 ** -20).all())


SECOND = {(2, 2): (1, 0), (2, 3): (1, 1), (2, 4): (1, 2)}   # slots 18, 19, 20 of sequence 1


@pytest.mark.parametrize("bad", BAD_LENGTHS)
def test_append_writes_nothing_for_a_sequence_of_bad_length(bad):
    kc, vc, table, L, g = two_sequences()
    got = append_to(kc, vc, table, torch.tensor([bad, 18], dtype=torch.int32), g)
    assert kernels.device_status(clear=True) != 0
    check_append(kc, vc, *got, SECOND)


@pytest.mark.parametrize("good", [0, 21])
def test_append_at_the_ends_of_a_page_table(good):
    kc, vc, table, L, g = two_sequences()
    got = append_to(kc, vc, table, torch.tensor([good, 18], dtype=torch.int32), g)
    at = {(3, t): (0, t) for t in range(3)} if good == 0 else {(4, 5 + t): (0, t) for t in range(3)}
    check_append(kc, vc, *got, {**SECOND, **at})


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 8, 99, 2 ** 31 - 1])
def test_append_drops_the_rows_of_a_page_outside_the_pool(bad):
    kc, vc, table, L, g = two_sequences()
    tab = table.clone()
    tab[0, 1] = bad
    got = append_to(kc, vc, tab, L, g)
    assert kernels.device_status(clear=True) != 0
    check_append(kc, vc, *got, {**SECOND, (3, 6): (0, 0), (3, 7): (0, 1)})
