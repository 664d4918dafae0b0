"""The host side of PagedKVCache, on the CPU with the operators replaced by recorders:
what it refuses, and that a refused call leaves the cache as it was."""

import copy

import pytest
import torch

from blockstreamer_b200 import attention
from blockstreamer_b200.attention import PagedKVCache


@pytest.fixture
def calls(monkeypatch):
    made = []

    class Recorder:
        def tree_commit(self, *a, **kw):
            made.append("commit")

        def kv_scores_add(self, *a, **kw):
            made.append("scores")

    monkeypatch.setattr(attention, "kernels", Recorder())
    return made


def cache(batch=2, pages=12, page_size=4, max_len=24, **kw):
    c = PagedKVCache(batch, pages, page_size, 1, 32, max_len, "cpu", **kw)
    c.reserve(5)
    return c


def state(c):
    return (list(c.lengths), c.lens.tolist(), c.page_table.tolist(), sorted(c._free), copy.deepcopy(c._held),
            None if c.scores is None else c.scores.clone().tolist())


@pytest.mark.parametrize("accepted,drafted,text", [
    ([[0, 2], [1, 1]], 5, "ascend"),
    ([[2, 1], []], 5, "ascend"),
    ([[0], [3, 5]], 5, "ascend"),
    ([[-1, 0], [0]], 5, "ascend"),
    ([[0]], 5, "2 lists"),
    ([[0], [1], [2]], 5, "2 lists"),
    ([], 5, "2 lists"),
    ([[0], [7, 8]], 9, "reserved"),   # two pages of four slots are
])
def test_commit_refuses_what_the_device_would_not_move(calls, accepted, drafted, text):
    c = cache(track_scores=True)
    before = state(c)
    with pytest.raises(ValueError, match=text):
        c.commit(accepted, drafted, torch.zeros(1), torch.zeros(1))
    assert state(c) == before and calls == []


def test_commit_advances_the_lengths(calls):
    c = cache(track_scores=True)
    c.commit([[0, 2, 4], []], 5, torch.zeros(1), torch.zeros(1))
    assert c.lengths == [3, 0] and c.lens.tolist() == [3, 0] and calls == ["commit", "scores"]
    c.commit([[], []], 5)
    assert c.lengths == [3, 0] and calls == ["commit", "scores"]
    c.reserve(2)
    c.commit([[0, 1], [1]], 2)
    assert c.lengths == [5, 1] and calls == ["commit", "scores", "commit"]


def evicting(monkeypatch, refuse=False):
    """kv_evict's shapes, or a refusal after its arguments are there."""
    def kv_evict(k, v, page_table, lens, scores, budget, out, keep_first=0, keep_last=0):
        made.append((budget, keep_first, keep_last, out.clone()))
        if refuse:
            raise ValueError("refused")
        kept = torch.full((*scores.shape[:2], budget), -1, dtype=torch.int32)
        return kept, lens, torch.zeros(*scores.shape[:2], out.shape[1] * k.shape[1])

    made = []
    monkeypatch.setattr(attention.kernels, "kv_evict", kv_evict)
    return made


def filled(lengths, pages=12, page_size=4, max_len=24):
    c = PagedKVCache(len(lengths), pages, page_size, 1, 32, max_len, "cpu", track_scores=True)
    c.lengths = [0] * len(lengths)
    for b, n in enumerate(lengths):
        c._held[b].extend(c._free.pop() for _ in range(-(-n // page_size)))
    c.lengths = list(lengths)
    c._upload()
    return c


def test_a_refused_eviction_loses_no_pages(monkeypatch):
    made = evicting(monkeypatch, refuse=True)
    c = filled([10, 5])
    before = state(c)
    with pytest.raises(ValueError, match="refused"):
        c.evict(6, keep_first=1, keep_last=2)
    assert len(made) == 1
    after = state(c)
    assert after[:3] == before[:3] and after[3] == before[3] and after[4:] == before[4:]


@pytest.mark.parametrize("kw,first,last", [
    (dict(), 4, 0),                             # by default the first four
    (dict(keep_last=4), 2, 4),                  # or as many of them as the last ones leave
    (dict(keep_last=6), 0, 6),
    (dict(keep_first=2, keep_last=4), 2, 4),
    (dict(keep_first=0), 0, 0),
])
def test_evict_protects_what_it_was_asked_to(monkeypatch, kw, first, last):
    made = evicting(monkeypatch)
    filled([10, 7]).evict(6, **kw)
    assert [m[:3] for m in made] == [(6, first, last)]


@pytest.mark.parametrize("kw", [dict(keep_first=7), dict(keep_last=7), dict(keep_first=3, keep_last=4),
                                dict(keep_first=-1), dict(keep_last=-1), dict(keep_first=6, keep_last=1)])
def test_evict_refuses_more_protected_slots_than_the_budget(monkeypatch, kw):
    made = evicting(monkeypatch)
    c = filled([10, 7])
    before = state(c)
    with pytest.raises(ValueError, match="keep_first"):
        c.evict(6, **kw)
    assert made == [] and state(c) == before


def test_evict_with_a_budget_beyond_every_sequence(monkeypatch):
    """Nothing is cut, so what is protected is all the same: the call's budget is what the pages hold."""
    made = evicting(monkeypatch)
    c = filled([3, 6])
    c.evict(500, keep_first=100, keep_last=300)
    budget, first, last, _ = made[0]
    assert budget == 8 and first + last <= 8 and c.lengths == [3, 6]


def test_evict_needs_pages_only_for_what_it_cuts(monkeypatch):
    """Sequences within the budget keep their pages, those of their slots; a nearly full
    pool, where eviction is wanted, is enough for the others."""
    made = evicting(monkeypatch)
    c = filled([16, 6, 0, 8], pages=10)     # 4 + 2 + 0 + 2 pages held, 2 free
    c._held[3].append(c._free.pop())        # and one reserved behind sequence 3: one free
    with pytest.raises(RuntimeError, match="needs 2 free pages, 1 are"):
        c.evict(8)
    own = [list(h) for h in c._held]
    assert made == []
    c._free.append(c._held[3].pop())
    spare = sorted(c._free)
    c.evict(8)
    out = made[0][3]
    assert c.lengths == [8, 6, 0, 8] and sorted(c._held[0]) == spare
    assert c._held[1] == own[1] and c._held[2] == [] and c._held[3] == own[3][:2]
    assert out[1].tolist() == own[1] and out[3].tolist() == own[3][:2] and out[0].tolist() == c._held[0]
    assert sorted(c._free) == sorted(own[0])
    assert c.page_table[3, :2].tolist() == own[3][:2] and c.lens.tolist() == [8, 6, 0, 8]


def test_evict_frees_pages_reserved_behind_a_short_sequence(monkeypatch):
    evicting(monkeypatch)
    c = filled([3])
    c.reserve(9)
    assert len(c._held[0]) == 3
    first = c._held[0][0]
    c.evict(100)
    assert c._held == [[first]] and len(c._free) == 11


def attending(monkeypatch):
    monkeypatch.setattr(attention.kernels, "tree_attention", lambda *a: ("out", "lse"), raising=False)


def test_scores_and_eviction_are_not_for_windowed_layers(calls, monkeypatch):
    """A key outside the window got no weight, so its score would be wrong; an eviction
    would go by such scores."""
    attending(monkeypatch)
    monkeypatch.setattr(attention.kernels, "kv_evict", None, raising=False)
    made = evicting(monkeypatch)
    c = cache(track_scores=True)
    q = torch.zeros(2, 5, 4, 32)
    pos = torch.zeros(2, 5, dtype=torch.int32)
    assert c.attend(q, pos, window=5) == ("out", "lse")     # nothing is outside it yet
    c.commit([[0, 1], [0]], 5, q, pos)
    assert calls == ["commit", "scores"]
    c.attend(q, pos, window=6)
    before = state(c)
    with pytest.raises(ValueError, match="window"):
        c.commit([[0], [0]], 5, q, pos)
    with pytest.raises(ValueError, match="window"):
        c.evict(2)
    assert state(c) == before and calls == ["commit", "scores"] and made == []
    c.commit([[0], [0]], 5)                                 # without scores it goes on
    assert c.lengths == [3, 2] and calls == ["commit", "scores", "commit"]


def test_a_window_after_an_eviction_is_refused(monkeypatch):
    """The window is told by slots, which are no positions any more."""
    attending(monkeypatch)
    evicting(monkeypatch)
    c = filled([7, 3])
    q, pos = torch.zeros(2, 1, 4, 32), torch.zeros(2, 1, dtype=torch.int32)
    c.evict(8)
    assert c.attend(q, pos, window=20) == ("out", "lse")    # nothing was cut
    c.evict(4)
    with pytest.raises(ValueError, match="evict"):
        c.attend(q, pos, window=20)
    assert c.attend(q, pos) == ("out", "lse")
