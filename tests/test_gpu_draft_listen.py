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
