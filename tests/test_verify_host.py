"""The host's part of ModelRunner.verify, without a GPU: what it hands to the step, what it keeps, what it leaves of the reservations."""
import random

import plain_drafts as P
import pytest

from mini_sglang_b200.cache import CacheManager, OutOfPages, PagedKVNeed
from mini_sglang_b200.engine import DraftEntry
from mini_sglang_b200.engine.step import ModelRunner


def make_runner(model, vocab=9, num_pages=64, max_context_len=128, page_size=4, max_reqs=4):
    """A runner without a device: a step keeps the path of first children as `draft_accept` does; `model` gives the token after a sequence of tokens."""
    r = ModelRunner.__new__(ModelRunner)
    r.mgr = CacheManager({0: PagedKVNeed(2, 8)}, page_size=page_size, num_pages=num_pages, max_reqs=max_reqs, max_context_len=max_context_len)
    r.vocab_size, r.page_size, r.max_context_len, r.calls = vocab, page_size, max_context_len, 0
    r.drafts_supported = lambda: True

    def step(entries, lens, parents, depths, *_):
        r.calls += 1
        kept, tokens = [], []
        for e, up, depth in zip(entries, parents, depths):
            anc = [sorted(a) for a in P.ancestors(up)]
            assert depth == [len(a) - 1 for a in anc]
            after = [model([e.tokens[a] for a in path]) for path in anc]
            path = P.accepted(up, list(e.tokens), after)
            kept.append(len(path))
            tokens.append([after[i] for i in path] + [-1] * (len(up) - len(path)))
        return kept, tokens

    r._verify = step
    return r


def longest(up, tokens, model):
    """The model's tokens along the longest path that it agrees with, by trying every draft."""
    best = []
    for anc in (sorted(a) for a in P.ancestors(up)):
        said = [model([tokens[a] for a in anc[:k + 1]]) for k in range(len(anc))]
        if anc[0] == 0 and all(tokens[b] == s for b, s in zip(anc[1:], said)) and len(said) > len(best):
            best = said
    return best


def test_siblings_of_one_token():
    """The longer path hangs below the second of two siblings that hold the same token."""
    follow = {1: 2, 2: 3, 3: 4}
    runner = make_runner(lambda seq: follow[seq[-1]])
    slot = runner.mgr.open()
    assert runner.verify([DraftEntry(slot, [1, 2, 2, 3], [-1, 0, 0, 2])], None) == [[2, 3, 4]]
    assert int(runner.mgr.length[slot]) == 3


def test_the_path_kept_is_the_longest():
    rng = random.Random(4)
    gained = 0
    for _ in range(300):
        n, vocab = rng.randint(1, 24), rng.choice((2, 3, 5))
        up = [-1] + [rng.randrange(max(0, i - rng.choice((2, 9))), i) for i in range(1, n)]
        tokens = [rng.randrange(vocab) for _ in range(n)]
        table = {}

        def model(seq):
            return table.setdefault(tuple(seq), rng.randrange(vocab))

        runner = make_runner(model, vocab)
        slot = runner.mgr.open()
        got = runner.verify([DraftEntry(slot, tokens, up)], None)[0]
        assert got == longest(up, tokens, model)
        gained += len(got) > len(P.accepted(up, tokens, [model([tokens[a] for a in sorted(anc)]) for anc in P.ancestors(up)]))
    assert gained > 10                                   # trees where the first child alone would have lost tokens


def test_a_tree_beyond_the_context_is_refused_before_anything_is_taken():
    """The slot is named, and the entries ahead of it have taken no pages."""
    runner = make_runner(lambda seq: 1, max_context_len=20)
    a, b = runner.mgr.open(), runner.mgr.open()
    runner.mgr.reserve(b, 15)
    runner.mgr.commit(b, 15)
    free = runner.mgr.available_pages()
    with pytest.raises(ValueError, match=f"slot {b}: .*15.* 6 .*20"):
        runner.verify([DraftEntry(a, [1] * 9), DraftEntry(b, [1] * 6)], None)
    assert runner.mgr.available_pages() == free and runner.mgr.owned_pages(a) == [] and runner.calls == 0
    assert runner.verify([DraftEntry(a, [1] * 9), DraftEntry(b, [1] * 5)], None) == [[1] * 9, [1] * 5]
    assert int(runner.mgr.length[b]) == 20


@pytest.mark.parametrize("slot", [0, -1, 2, 99])
def test_slots_that_are_not_open_are_refused(slot):
    runner = make_runner(lambda seq: 1)
    a = runner.mgr.open()
    while runner.mgr.free_slots:
        runner.mgr.open()
    runner.mgr.close(2)
    free = runner.mgr.available_pages()
    with pytest.raises(ValueError, match=f"slot {slot} is not open"):
        runner.verify([DraftEntry(a, [1, 2]), DraftEntry(slot, [1, 2])], None)
    assert runner.mgr.available_pages() == free and int(runner.mgr.reserved[a]) == 0


@pytest.mark.parametrize("fails", [False, True])
def test_what_a_caller_has_reserved_stays_reserved(fails):
    runner = make_runner(lambda seq: 1)
    slot = runner.mgr.open()
    runner.mgr.reserve(slot, 30)
    runner.mgr.commit(slot, 10)

    def broken(*_):
        raise RuntimeError("a step that fails")

    if fails:
        runner._verify = broken
        with pytest.raises(RuntimeError, match="fails"):
            runner.verify([DraftEntry(slot, [1, 1, 1])], None)
    else:
        assert runner.verify([DraftEntry(slot, [1, 1, 1])], None) == [[1, 1, 1]]
    assert int(runner.mgr.length[slot]) == (10 if fails else 13) and int(runner.mgr.reserved[slot]) == 30
    with pytest.raises(OutOfPages):
        runner.verify([DraftEntry(slot, [1] * 90), DraftEntry(runner.mgr.open(), [1] * 128), DraftEntry(runner.mgr.open(), [1] * 128)], None)
    assert int(runner.mgr.reserved[slot]) == 30
    runner._verify = make_runner(lambda seq: 1)._verify
    assert len(runner.verify([DraftEntry(slot, [1] * 25)], None)[0]) == 25
    assert int(runner.mgr.reserved[slot]) == max(30, int(runner.mgr.length[slot]))


def test_drafts_lie_within_what_is_reserved_already():
    """Places that a caller reserved for the next tokens are the ones that the drafts take: no further pages, and nothing beyond the context limit."""
    runner = make_runner(lambda seq: 1, num_pages=5, max_context_len=20)
    slot = runner.mgr.open()
    runner.mgr.reserve(slot, 20)
    runner.mgr.commit(slot, 8)
    assert runner.verify([DraftEntry(slot, [1] * 12)], None) == [[1] * 12]
    assert int(runner.mgr.length[slot]) == int(runner.mgr.reserved[slot]) == 20
