"""Numbers of the drafted pass that ctypes would cut to 32 bits (WhisperEngine.draft_logits): refused before the library is asked."""
import types

import pytest
import torch

from whisper_amd.engine import WhisperEngine


class Reached(Exception):
    pass


class Lib:
    def wx_logit_stride(self, handle):
        raise Reached


@pytest.mark.parametrize("group", [(1 << 32) + 1, 1 << 31, 0, -1, -(1 << 32) + 1])
def test_group_out_of_range(group):
    self = types.SimpleNamespace(torch_device=torch.device("cpu"), lib=Lib(), handle=None)
    ids = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError):
        WhisperEngine.draft_logits(self, None, ids[0], ids, group=group)
    with pytest.raises(Reached):
        WhisperEngine.draft_logits(self, None, ids[0], ids, group=1)
    with pytest.raises(TypeError):
        WhisperEngine.draft_logits(self, None, ids[0], ids, group=1.5)
