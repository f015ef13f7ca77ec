"""A drafter that listens (EngineDraft) through transcribe_mel, alone and shared by lanes: host logic, on stand-ins for the engines."""
import threading
import time
import types

import pytest
import torch

from whisper_amd.audio import N_FRAMES
from whisper_amd.draft import EngineDraft
from whisper_amd.engine import WhisperEngine
from whisper_amd.lanes import EngineLanes


class StandIn:
    """encode() notes which windows it was given (the first sample of each); decode_rows() answers with them and notes calls that overlap"""
    transcribe_mel = WhisperEngine.transcribe_mel

    def __init__(self, max_batch=2, n_vocab=100, n_mels=4, device="cpu"):
        self.max_batch, self.precision, self.torch_device = max_batch, "fp32", torch.device(device)
        self.dims = types.SimpleNamespace(n_vocab=n_vocab, n_mels=n_mels, n_text_ctx=16)
        self.encode_gate, self.windows, self.inside, self.overlaps, self.calls = None, None, 0, 0, 0
        self.lock = threading.Lock()

    def busy(self):
        with self.lock:
            self.inside += 1
            self.overlaps += self.inside > 1
        time.sleep(0.003)
        with self.lock:
            self.inside -= 1

    def encode(self, mel, win_stride, row_stride, n_valid, B):
        assert (win_stride, row_stride) == (N_FRAMES, mel.stride(0)) and n_valid == mel.shape[1]
        self.busy()
        self.windows = [float(mel[0, b * win_stride]) for b in range(B)]

    def decode_rows(self, rows, **kw):
        self.calls += 1
        self.busy()
        return {"tokens": [[int(w)] for w in self.windows]}

    def decode_draft(self, prompts, drafter, **kw):
        heard = [int(w) for w in self.windows]
        for _ in range(3):                             # a pass each: the drafts are of the windows that are decoded
            assert drafter([list(p) for p in prompts], 4) == [[[w]] for w in heard]
        return {"tokens": [[w] for w in heard], "sum_logprobs": [0.0] * len(heard), "no_speech_probs": [0.0] * len(heard), "steps": 3}


def mel_of(n):
    mel = torch.zeros(4, n * N_FRAMES)
    mel[0, ::N_FRAMES] = torch.arange(n).float()
    return mel


def test_the_helper_hears_every_batch():
    helper = StandIn()
    got = StandIn().transcribe_mel(mel_of(5), 5 * N_FRAMES, 0, 5, [1, 2], draft=EngineDraft(helper))
    assert got["tokens"] == [[i] for i in range(5)] and helper.calls == 9


def test_lanes_share_a_helper():
    helper, lanes = StandIn(), EngineLanes([StandIn() for _ in range(3)])
    try:
        for draft in (EngineDraft(helper), EngineDraft(helper)):
            got = lanes.transcribe_mel(mel_of(13), 13 * N_FRAMES, 0, 13, [1, 2], draft=draft)
            assert got["tokens"] == [[i] for i in range(13)]
        assert helper.overlaps == 0 and helper.calls == 2 * 7 * 3
    finally:
        for ln in lanes._lanes:
            ln.engine.close = lambda: None
        lanes.close()


def test_two_drafters_on_one_helper_take_turns():
    helper, drafts = StandIn(), None
    helper.windows = [7.0]
    drafts = [EngineDraft(helper) for _ in range(4)]
    threads = [threading.Thread(target=lambda d=d: [d([[1]], 2) for _ in range(5)]) for d in drafts]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert helper.calls == 20 and helper.overlaps == 0


def test_helpers_that_do_not_fit():
    mel, e = mel_of(4), StandIn()
    for bad in (StandIn(max_batch=1), StandIn(n_vocab=99), StandIn(n_mels=5), StandIn(device="meta"), e):
        with pytest.raises(ValueError):
            e.transcribe_mel(mel, 4 * N_FRAMES, 0, 4, [1], draft=EngineDraft(bad))
    lanes = EngineLanes([StandIn(), StandIn()])
    try:
        with pytest.raises(ValueError):
            lanes.transcribe_mel(mel, 4 * N_FRAMES, 0, 4, [1], draft=EngineDraft(lanes.engines[1]))
    finally:
        for ln in lanes._lanes:
            ln.engine.close = lambda: None
        lanes.close()


def test_a_helper_whose_batch_failed_is_free_again():
    helper = StandIn()

    class Broken(StandIn):
        def decode_draft(self, *a, **kw):
            raise RuntimeError("no")
    draft = EngineDraft(helper)
    with pytest.raises(RuntimeError):
        Broken().transcribe_mel(mel_of(1), N_FRAMES, 0, 1, [1], draft=draft)
    done = []
    t = threading.Thread(target=lambda: done.append(StandIn().transcribe_mel(mel_of(2), 2 * N_FRAMES, 0, 2, [1], draft=draft)["tokens"]))
    t.start()
    t.join(timeout=30)
    assert done == [[[0], [1]]]
