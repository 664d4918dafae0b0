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


@pytest.mark.parametrize("lens,width,budget,first,last", [
    ([100, 30, 0], 64, 40, 4, 8),       # longer than the scores, shorter, empty
    ([100, 64, 65], 64, 40, 0, 40),     # only the last ones are protected, all of them without a score
    ([100, 90], 32, 96, 0, 0),          # one sequence fits its budget
    ([100, 99], 1, 50, 2, 3),           # nearly nothing is scored
    ([9000], 100, 70, 1, 5),            # several CTAs to an item
    ([9000], 8995, 4500, 0, 2),         # and scores that do not start on 16 bytes
    ([60000] + [9] * 25, 40, 30, 1, 2), # not held in shared memory
])
def test_evict_counts_slots_behind_the_scores_as_zero(lens, width, budget, first, last):
    """The scores may be narrower than the page table: a slot without one has the score 0."""
    page, heads, D = 16, 3, 8
    g = torch.Generator().manual_seed(width)
    B, P, Q = len(lens), pages_for(max(lens), page), pages_for(min(budget, max(lens)), page)
    order = torch.randperm(B * (P + Q), generator=g).to(torch.int32)
    table, out = order[: B * P].view(B, P), order[B * P:].view(B, Q)
    kc = torch.randn(B * (P + Q), page, heads, D, generator=g).bfloat16()
    vc = torch.randn(B * (P + Q), page, heads, D, generator=g).bfloat16()
    scores = torch.randn(B, heads, width, generator=g)      # negative ones rank below a slot without a score
    full = torch.zeros(B, heads, P * page)
    full[..., :width] = scores
    k, v = to(kc, vc)
    kept, new_lens, new = kernels.kv_evict(k, v, *to(table, torch.tensor(lens, dtype=torch.int32), scores), budget,
                                           out.to(DEV), first, last)
    want = oatt.evict(full, lens, budget, first, last)
    wk, wv, ws = kc.clone(), vc.clone(), torch.zeros(B, heads, Q * page)
    assert new_lens.tolist() == [min(n, budget) for n in lens]
    for b in range(B):
        for h in range(heads):
            row = want[b][h]
            assert kept[b, h].tolist() == row + [-1] * (budget - len(row)), (b, h)
            i, j = torch.arange(len(row)), torch.tensor(row, dtype=torch.long)
            at, src = (out[b].long()[i // page], i % page, h), (table[b].long()[j // page], j % page, h)
            wk[at], wv[at], ws[b, h, : len(row)] = kc[src], vc[src], full[b, h, j]
    assert torch.equal(k.cpu(), wk) and torch.equal(v.cpu(), wv) and torch.equal(new.cpu(), ws)


def test_evict_to_fewer_pages_than_the_budget_is_reported():
    """A budget beyond the output pages is accepted where the scores say that no sequence
    needs them; one that does keeps its best slots, as many as the pages hold."""
    page, g = 8, torch.Generator().manual_seed(5)
    kc, vc = (torch.randn(9, page, 1, 8, generator=g).bfloat16() for _ in range(2))
    table, out = torch.arange(6, dtype=torch.int32)[None], torch.tensor([[6, 7]], dtype=torch.int32)
    scores = torch.rand(1, 1, 16, generator=g) + 1
    k, v = to(kc, vc)
    kept, lens, new = kernels.kv_evict(k, v, *to(table, torch.tensor([40], dtype=torch.int32), scores), 20, out.to(DEV), 1, 2)
    assert kernels.device_status(clear=True) != 0
    want = oatt.evict(torch.cat([scores, torch.zeros(1, 1, 32)], 2), [40], 16, 1, 2)[0][0]
    assert int(lens) == 16 and kept[0, 0].tolist() == want + [-1] * 4
    src = torch.tensor(want)
    for c, d in ((kc, k), (vc, v)):
        full = c.clone()
        full[6:8] = c[src // page, src % page].view(2, page, 1, 8)
        assert torch.equal(d.cpu(), full)
    assert new.shape == (1, 1, 16) and new[0, 0].cpu().tolist() == [float(scores[0, 0, j]) if j < 16 else 0.0 for j in want]


@pytest.mark.parametrize("behind", [-1, -2 ** 31, 10 ** 6])
@pytest.mark.parametrize("T,Hq,D,page,slots", [
    (8, 1, 64, 8, 0), (8, 2, 32, 5, 0), (8, 2, 128, 8, 0), (8, 2, 128, 8, 1000),    # few rows: boxes, copies, cut
    (8, 4, 64, 16, 2000), (20, 4, 128, 8, 0), (20, 8, 64, 8, 0), (20, 8, 64, 6, 0),  # tiles
])
def test_pages_behind_the_last_used_draft_are_not_looked_at(T, Hq, D, page, slots, behind):
    """A page table may hold anything where a sequence has no slot in use: its drafts not in
    use have no pages, nor have the entries behind the accepted ones."""
    heads, B, n, used = 2, 2, 13, [3, 2]
    g = torch.Generator().manual_seed(T)
    P = pages_for(n + T, page) + slots // page
    kc, vc = (torch.randn(B * P, page, heads, D, generator=g).bfloat16().to(DEV) for _ in range(2))
    table = torch.randperm(B * P, generator=g).to(torch.int32).view(B, P)
    L = torch.tensor([n, n + 1], dtype=torch.int32)
    pos = (L[:, None] + torch.arange(T)).to(torch.int32)
    bad = table.clone()
    for b in range(B):
        pos[b, used[b]:] = -1
        bad[b, pages_for(int(L[b]) + used[b], page):] = behind
    q = torch.randn(B, T, Hq * heads, D, generator=g).bfloat16()
    q, table, bad, L, pos = to(q, table, bad, L, pos)
    want, lse = kernels.tree_attention(q, kc, vc, table, L, pos)
    got, lse1 = kernels.tree_attention(q, kc, vc, bad, L, pos)
    assert torch.equal(got, want) and torch.equal(lse, lse1)
    acc = torch.full((B, T - 1), -1, dtype=torch.int32)
    acc[0, :2], acc[1, :1] = torch.tensor([0, 2]), torch.tensor([1])
    scores = torch.rand(B, heads, P * page, generator=g).to(DEV)
    a, b = (kernels.kv_scores_add(scores, q, lse, kc, t, L, accepted=acc.to(DEV)) for t in (table, bad))
    assert torch.equal(a, b)
    assert kernels.device_status(clear=False) == 0
    # where a used draft has no page it is reported still
    bad[0, int(L[0]) // page] = behind
    kernels.tree_attention(q, kc, vc, bad, L, pos)
    assert kernels.device_status(clear=True) != 0
    kernels.kv_scores_add(scores, q, lse, kc, bad, L, accepted=acc.to(DEV))
    assert kernels.device_status(clear=True) != 0
