"""transcribe_mel with another engine's drafts, several batches, alone and through lanes: greedy's ids in fewer passes."""
import pytest

from test_gpu_draft import make
from whisper_amd.draft import EngineDraft

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lanes", [0, 2])
def test_a_helper_over_several_batches(lanes):
    from whisper_amd.lanes import EngineLanes
    eng, mel, _ = make(max_batch=2, windows=5)
    helper = eng.replica()
    try:
        init = eng.initial_tokens(0)
        want = eng.transcribe_mel(mel, 15000, 0, 5, init, max_new_tokens=25)
        if lanes:
            with EngineLanes([eng.replica() for _ in range(lanes)]) as many:
                got = many.transcribe_mel(mel, 15000, 0, 5, init, max_new_tokens=25, draft=EngineDraft(helper))
                with pytest.raises(ValueError):
                    many.transcribe_mel(mel, 15000, 0, 5, init, draft=EngineDraft(many.engines[1]))
        else:
            got = eng.transcribe_mel(mel, 15000, 0, 5, init, max_new_tokens=25, draft=EngineDraft(helper))
        assert got["tokens"] == want["tokens"]
        assert got["steps"] <= 3 * (2 + -(-26 // 9))                # the same model: every draft of 8 agrees, three batches
        small = eng.replica(max_batch=1)
        with pytest.raises(ValueError):
            eng.transcribe_mel(mel, 15000, 0, 5, init, draft=EngineDraft(small))
        small.close()
        with pytest.raises(ValueError):
            eng.transcribe_mel(mel, 15000, 0, 5, init, draft=EngineDraft(eng))
    finally:
        helper.close()
        eng.close()


class Noted:
    """what a drafter is asked, and drafts that agree"""

    def __init__(self, full):
        self.full, self.asked = full, []

    def __call__(self, rows, k):
        self.asked.append([list(r) for r in rows])
        return [[f[len(r):len(r) + k]] for r, f in zip(rows, self.full)]


@pytest.mark.parametrize("long_row", [False, True])
def test_rows_that_need_no_draft_are_given_as_their_prompt(long_row):
    """finished rows, and rows at their limit or at the end of the context, stop nobody else's drafts: EngineDraft asks for all rows or none"""
    eng, _, encode = make(max_batch=4, windows=2)
    if long_row:
        eng.set_suppress_ids([*eng.suppress_ids, eng.tok.eot])
    helper = eng.replica()
    try:
        encode(helper)
        base = eng.initial_tokens(0)
        # no end to pick: the first row fills its context (448 positions) 200 ids before the second, which goes on
        ps = [[eng.tok.sot_prev] + [int(x) for x in range(1, 201)] + list(base) if long_row else list(base), [eng.tok.sot_prev, 5, 6, 7] + list(base)]
        limit = 440 if long_row else 40
        want = eng.decode_rows(ps, max_new_tokens=limit)["tokens"]
        ends = [len(p) + len(t) for p, t in zip(ps, want)]
        if long_row:
            assert ends[0] == eng.dims.n_text_ctx + 1 and ends[1] > 440
        noted = Noted([p + t + [eng.tok.eot] for p, t in zip(ps, want)])
        got = eng.decode_draft(ps, noted, n_nodes=9, n_draft=8, max_new_tokens=limit)
        assert got["tokens"] == want
        for rows in noted.asked:
            for r, p, end in zip(rows, ps, ends):
                assert r[:len(p)] == p and len(r) < eng.dims.n_text_ctx and (len(r) <= end or r == p)
        got = eng.decode_draft(ps, EngineDraft(helper), n_nodes=9, n_draft=8, max_new_tokens=limit)
        assert got["tokens"] == want
        assert got["passes"] <= 2 + -(-(max(map(len, want)) + 1) // 9) + 1
    finally:
        helper.close()
        eng.close()
