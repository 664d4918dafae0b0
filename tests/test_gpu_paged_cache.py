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
