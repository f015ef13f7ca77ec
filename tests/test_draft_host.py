"""Where drafts come from and how they become a tree (whisper_amd/draft.py): host logic, no GPU."""
import random

import pytest

from whisper_amd.draft import EngineDraft, NgramDraft, draft_tree

EOT = 99


def paths(tokens, parents):
    """every node as the ids from below the root to it"""
    out = []
    for j in range(1, len(tokens)):
        p, way = j, []
        while p > 0:
            way.append(tokens[p])
            p = parents[p]
        out.append(tuple(way[::-1]))
    return out


def test_tree_shares_beginnings_and_keeps_order():
    tokens, parents = draft_tree(7, [[1, 2, 3], [1, 2, 4], [5]], 16, 8, EOT)
    assert tokens[0] == 7 and parents[0] == -1
    assert all(-1 < p < j for j, p in enumerate(parents) if j)
    assert set(paths(tokens, parents)) == {(1,), (1, 2), (1, 2, 3), (1, 2, 4), (5,)}
    assert len(tokens) == 6


def test_tree_limits():
    assert draft_tree(3, [], 8, 8, EOT) == ([3], [-1])
    assert draft_tree(3, [[1, 2, 3]], 1, 8, EOT) == ([3], [-1])
    assert draft_tree(3, [[1, 2, 3]], 8, 0, EOT) == ([3], [-1])
    assert draft_tree(3, [[1, 2, 3]], 8, 2, EOT)[0] == [3, 1, 2]
    assert draft_tree(3, [[1, EOT, 3], [EOT], []], 8, 8, EOT) == ([3, 1], [-1, 0])
    tokens, parents = draft_tree(0, [[1, 2, 3, 4], [5, 6, 7, 8]], 5, 8, EOT)       # side by side: both begin
    assert tokens == [0, 1, 5, 2, 6] and parents == [-1, 0, 0, 1, 2]


def test_tree_of_random_candidates():
    rng = random.Random(0)
    for _ in range(200):
        cands = [[rng.randrange(4) for _ in range(rng.randrange(6))] for _ in range(rng.randrange(5))]
        most, deep = rng.randrange(1, 12), rng.randrange(7)
        tokens, parents = draft_tree(9, cands, most, deep, EOT)
        ways = paths(tokens, parents)
        assert len(tokens) <= most and len(set(ways)) == len(ways)
        assert all(len(w) <= deep and any(tuple(c[:len(w)]) == w for c in cands) for w in ways)
        if most >= 40:
            assert len(ways) == len({tuple(c[:i]) for c in cands for i in range(1, min(len(c), deep) + 1)})


def test_ngram_draft():
    d = NgramDraft(n=2, branches=2)
    assert d([[1, 2, 3, 1, 2, 4, 1, 2]], 2) == [[[4, 1], [3, 1]]]                 # the latest first
    assert d([[1, 2, 3, 9, 3]], 3) == [[[9, 3]]]                                   # one id where two never stood
    assert d([[1, 2, 3], [5], []], 3) == [[], [], []]
    with pytest.raises(ValueError):
        NgramDraft(n=0)
    with pytest.raises(ValueError):
        NgramDraft(branches=0)


def test_engine_draft_asks_for_every_row_or_none():
    class Engine:
        class dims:
            n_text_ctx = 8
        calls = []

        def decode_rows(self, rows, **kw):
            self.calls.append((list(map(list, rows)), kw))
            return {"tokens": [[1, 2] for _ in rows]}
    e = Engine()
    assert EngineDraft(e)([[1], [2, 3]], 2) == [[[1, 2]], [[1, 2]]]
    assert e.calls[0][1]["max_new_tokens"] == 2
    assert EngineDraft(e)([[1] * 8, [2]], 2) == [[], []] and len(e.calls) == 1       # no room in the draft's context
