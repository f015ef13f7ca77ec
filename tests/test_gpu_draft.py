"""Drafted decoding of the engine (wx_draft_logits, WhisperEngine.decode_draft): the drafted nodes' logits against the decoder's own,
position by position, and greedy's ids whatever the drafts."""
import numpy as np
import pytest
import torch

from oracle import whisper_oracle as wo
from whisper_amd import checkpoint as ck
from whisper_amd.draft import EngineDraft, NgramDraft

pytestmark = pytest.mark.gpu


def make(precision="fp32", max_batch=4, name="micro", windows=3, eot_boost=1.0, **kw):
    from whisper_amd.engine import WhisperEngine
    dims = ck.dims_for(name)
    eng = WhisperEngine(dims, ck.synthetic_state_dict(dims, seed=0, eot_boost=eot_boost), precision=precision, max_batch=max_batch, **kw)
    audio = torch.from_numpy(np.concatenate([wo.varied_audio(i, 16000 * 30) for i in range(windows)])).cuda()
    mel = eng.log_mel(audio)
    encode = lambda e: e.encode(mel, 3000, mel.stride(0), audio.numel() // 160, min(windows, max_batch))  # noqa: E731
    encode(eng)
    return eng, mel, encode


def prompts(eng, extra=((), (5, 6, 7), (11, 12))):
    base = eng.initial_tokens(0)
    return [[eng.tok.sot_prev, *e, *base] if e else list(base) for e in extra]


class Given:
    """drafts made from each row's whole greedy text: right, wrong from some id on, or mixed with wrong branches"""

    def __init__(self, full, kind, seed=0):
        self.full, self.kind, self.rng = full, kind, np.random.RandomState(seed)

    def __call__(self, rows, k):
        out = []
        for ids, full in zip(rows, self.full):
            true = full[len(ids):len(ids) + k]
            wrong = self.rng.randint(0, 300, k).tolist()
            out.append({"none": [], "right": [true], "wrong": [wrong], "empty": [[]],
                        "mixed": [wrong, true[:2] + wrong, true, true]}[self.kind])
        return out


@pytest.mark.parametrize("kind", ["none", "right", "wrong", "mixed", "empty"])
@pytest.mark.parametrize("n_nodes", [1, 7, 64])
def test_ids_are_greedys_whatever_the_drafts(kind, n_nodes):
    eng, _, _ = make()
    try:
        ps = prompts(eng)
        want = eng.decode_rows(ps, max_new_tokens=40)
        full = [p + t + [eng.tok.eot] for p, t in zip(ps, want["tokens"])]
        got = eng.decode_draft(ps, Given(full, kind), n_nodes=n_nodes, n_draft=6, max_new_tokens=40)
        assert got["tokens"] == want["tokens"]
        np.testing.assert_allclose(got["sum_logprobs"], want["sum_logprobs"], rtol=1e-4, atol=1e-3)      # the bars of the fp32 engine's own tests
        np.testing.assert_allclose(got["no_speech_probs"], want["no_speech_probs"], rtol=1e-3, atol=1e-6)
        longest = max(len(t) for t in want["tokens"])
        if kind == "right" and n_nodes > 1:
            assert got["passes"] <= 2 + -(-longest // min(n_nodes, 7)) and got["accepted"] > 0
        if kind in ("none", "empty") or n_nodes == 1:
            assert got["accepted"] == 0 and longest <= got["passes"] <= longest + 1
    finally:
        eng.close()


def test_a_whole_context_and_ngrams():
    """no end in sight: the rows run to the last position of the context, one of them from a long prompt"""
    eng, _, _ = make(eot_boost=-50.0, windows=2)
    try:
        base = eng.initial_tokens(0)
        ps = [list(base), [eng.tok.sot_prev] + [int(x) for x in np.random.RandomState(0).randint(0, 300, 200)] + list(base)]
        for limit in (0, 446):
            want = eng.decode_rows(ps, max_new_tokens=limit)
            got = eng.decode_draft(ps, NgramDraft(3, 3), n_nodes=24, n_draft=12, max_new_tokens=limit)
            assert got["tokens"] == want["tokens"]
            np.testing.assert_allclose(got["sum_logprobs"], want["sum_logprobs"], rtol=1e-4, atol=1e-2)
            assert got["passes"] <= max(len(t) for t in want["tokens"]) + 1
    finally:
        eng.close()


def test_another_engines_drafts():
    eng, _, encode = make(max_batch=4)
    helper = eng.replica()
    try:
        encode(helper)
        ps = prompts(eng)
        want = eng.decode_rows(ps, max_new_tokens=30)
        got = eng.decode_draft(ps, EngineDraft(helper), n_nodes=9, n_draft=8, max_new_tokens=30)
        assert got["tokens"] == want["tokens"] and got["accepted"] > 0
        longest = max(len(t) for t in want["tokens"])
        assert got["passes"] <= 2 + -(-longest // 9) + 1                       # the same model: every draft agrees
    finally:
        helper.close()
        eng.close()


@pytest.mark.parametrize("precision,max_batch", [("fp32", 4), ("bf16", 4), ("bf16", 32)])
def test_node_logits_against_the_decoder(precision, max_batch, monkeypatch):
    """the logits of every node of a tree = the decoder's for the prompt and the path to the node; two entries listen to each window.  Drafted
    passes attend cached cross K/V; an engine whose own decode attends the encoder output instead (bf16, 32 rows and up: other rounding
    points) is held to the decoder of one that is made with cached K/V."""
    eng, _, _ = make(precision, max_batch, windows=2)
    ref = eng
    if eng.cross_form != "kv":
        monkeypatch.setenv("WX_NO_XATTN", "1")
        ref, _, _ = make(precision, max_batch, windows=2)
        assert ref.cross_form == "kv"
    try:
        rng = np.random.RandomState(1)
        N, prompt = 7, rng.randint(0, 300, (4, 5)).astype(np.int32)
        par = np.array([[-1, 0, 0, 1, 3, 2, -1]] * 4, np.int32)
        tok = rng.randint(0, 300, (4, N)).astype(np.int32)
        cache = eng.draft_cache(4)
        i32 = lambda a: torch.tensor(np.ascontiguousarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
        slots = i32([2, 0, 3, 1])
        cache.reserve(slots, 5)
        assert eng.draft_logits(cache, slots, i32(prompt), group=2, want_logits=False) is None
        cache.commit(slots, i32([[0, 1, 2, 3, 4]] * 4), i32([5] * 4))
        cache.reserve(slots, N)
        got = eng.draft_logits(cache, slots, i32(tok), i32(par), group=2).cpu().numpy()
        again = eng.draft_logits(cache, slots, i32(tok), i32(par), group=2).cpu().numpy()
        np.testing.assert_array_equal(got, again)
        worst = 0.0
        for e in range(4):
            for j in range(N):
                way, p = [], j
                while p >= 0:
                    way.append(int(tok[e, p]))
                    p = int(par[e, p])
                seq = [int(x) for x in prompt[e]] + way[::-1]
                # entry e listens to window e // 2: decode both windows, read that one
                want = ref.decoder_logits(torch.tensor([seq, seq]))[e // 2, -1].cpu().numpy()
                worst = max(worst, float(np.abs(got[e, j] - want).max() / np.abs(want).max()))
        # fp32: the bar of the engine's own logit tests; bf16: the activations of every layer are rounded to half a step of 2^-8 by both sides, at places
        # that differ by the order of sums: a few such steps of the largest logit
        assert worst < (1e-4 if precision == "fp32" else 6 * 2.0 ** -8), worst
    finally:
        if ref is not eng:
            ref.close()
        eng.close()


@pytest.mark.parametrize("group,N", [(1, 1), (1, 2), (1, 8), (1, 9), (1, 40), (2, 21), (3, 53), (3, 54)])
@pytest.mark.parametrize("windows", [1, 2])
def test_every_size_of_pass(group, N, windows):
    """chains of every number of rows a pass treats differently, against the decoder's logits position by position, the second half of the
    rows behind a committed first half.

    fp32: the bar of the engine's own logit tests.  bf16: this network of random weights amplifies a rounding, so the bar is its own: the
    decoder's distance from the fp32 engine's logits.  That distance comes from half a step of 2^-8 in every weight and in every stored
    activation, two kinds at each of ten products a layer.  Pass and decoder share the weights; they round differently at three places a
    layer (the probabilities of both attentions, and sums of another order), on two sides: sqrt(2 x 3 / 20) = 0.55 of it if errors add up
    as a random walk does.  Half of it is asked for; a row that met a wrong row, weight or window is off by about the logits' size."""
    dist = lambda a, b: float(((a - b).abs().amax(-1) / b.abs().amax(-1)).max())  # noqa: E731
    n, rng = windows * group, np.random.RandomState(N)
    tok = rng.randint(0, 300, (n, 2 * N)).astype(np.int32)
    seen = {}
    for precision in ("fp32", "bf16"):
        eng, _, _ = make(precision, 2, name="tiny", windows=windows)
        try:
            assert eng.cross_form == "kv"
            cache = eng.draft_cache(n)
            slots = torch.arange(n, dtype=torch.int32, device="cuda")
            d = torch.from_numpy(tok).cuda()
            got = []
            for half in (0, 1):
                cache.reserve(slots, N)
                got.append(eng.draft_logits(cache, slots, d[:, half * N:half * N + N].contiguous(), group=group))
                path = torch.arange(N, dtype=torch.int32, device="cuda").repeat(n, 1)
                assert not cache.commit(slots, path, torch.full((n,), N, dtype=torch.int32, device="cuda")).any()
            got = torch.cat(got, 1).cpu()
            want = torch.empty_like(got)
            for k in range(group):                                   # entry k of every window's group
                want[k::group] = eng.decoder_logits(torch.from_numpy(tok[k::group].copy())).cpu()[..., :got.shape[-1]]
            seen[precision] = got, want
        finally:
            eng.close()
    assert dist(*seen["fp32"]) < 1e-4
    assert dist(*seen["bf16"]) <= 0.5 * dist(seen["bf16"][1], seen["fp32"][1])


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
def test_a_captured_pass(precision):
    """a drafted step (reserve, pass, verification, commit) captured once and replayed, other ids each time, the same as eager steps"""
    from whisper_amd.draft import verify_tree
    eng, _, _ = make(precision, 2, windows=2)
    try:
        n, N = 2, 5
        i32 = lambda a: torch.tensor(np.ascontiguousarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
        par, slots, tok = i32([[-1, 0, 0, 1, 3]] * n), i32([1, 0]), i32(np.zeros((n, N)))
        caches = [eng.draft_cache(n) for _ in range(2)]

        def step(cache):
            cache.reserve(slots, N)
            logits = eng.draft_logits(cache, slots, tok, par)
            r = verify_tree(logits, tok, par)
            cache.commit(slots, r["path"], r["n_accept"])
            return logits, r
        ids = [np.random.RandomState(i).randint(0, 300, (n, N)) for i in range(5)]
        tok.copy_(i32(ids[0]))
        for c in caches:                                             # warm
            step(c)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits, r = step(caches[0])
        for x in ids[1:]:
            tok.copy_(i32(x))
            want = step(caches[1])
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(logits, want[0]) and all(torch.equal(r[k], want[1][k]) for k in r)
            assert torch.equal(caches[0].lens, caches[1].lens)
    finally:
        eng.close()


def test_no_capture_where_keys_are_projected():
    from whisper_amd._lib import WxError
    eng, _, _ = make("bf16", 32, windows=1)
    try:
        assert eng.cross_form == "encoder_output"
        cache, one = eng.draft_cache(1), torch.zeros(1, dtype=torch.int32, device="cuda")
        cache.reserve(one, 1)
        eng.draft_logits(cache, one, one.view(1, 1))
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            one.add_(0)
            with pytest.raises(WxError, match="captured"):
                eng.draft_logits(cache, one, one.view(1, 1))
    finally:
        eng.close()


def test_windows_path_with_ngram_drafts():
    eng, mel, _ = make(max_batch=2, windows=3)
    try:
        init = eng.initial_tokens(0)
        want = eng.transcribe_mel(mel, 9000, 0, 3, init, max_new_tokens=25)
        got = eng.transcribe_mel(mel, 9000, 0, 3, init, max_new_tokens=25, draft="ngram")
        assert got["tokens"] == want["tokens"]
        np.testing.assert_allclose(got["sum_logprobs"], want["sum_logprobs"], rtol=1e-4, atol=1e-3)
        with pytest.raises(ValueError):
            eng.transcribe_mel(mel, 9000, 0, 3, init, draft="ngram", beam_size=2)
        with pytest.raises(ValueError):
            eng.transcribe_mel(mel, 9000, 0, 3, init, draft="other")
    finally:
        eng.close()


def test_refusals():
    from whisper_amd._lib import WxError
    from whisper_amd.kvcache import PagedKVCache
    eng, _, _ = make(windows=2)
    try:
        base = eng.initial_tokens(0)
        for bad in ([[]], [[1, 2]], [base * 300], [base + [10 ** 7]]):
            with pytest.raises(ValueError):
                eng.decode_draft(bad)
        for kw in (dict(without_timestamps=False), dict(n_nodes=0), dict(n_nodes=65), dict(n_draft=0)):
            with pytest.raises(ValueError):
                eng.decode_draft([base], **kw)
        with pytest.raises(WxError, match="group"):
            eng.decode_draft([base] * 3)                                       # three rows, two windows
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        cache = eng.draft_cache(2)
        with pytest.raises(ValueError):
            eng.draft_cache(2, 65)
        with pytest.raises(ValueError):
            eng.draft_logits(cache, i32([0]), i32([[1, 2]]), i32([[0]]))
        other = PagedKVCache.allocate(1, eng.dims.n_text_head, 64, 8, 2, 4, dtype=torch.bfloat16)
        with pytest.raises(WxError, match="precision"):
            eng.draft_logits(other, i32([0]), i32([[1]]))
        wide = PagedKVCache.allocate(eng.dims.n_text_layer, eng.dims.n_text_head, 64, 8, 2, 64, dtype=torch.float32)
        with pytest.raises(WxError, match="512"):
            eng.draft_logits(wide, i32([0]), i32([[1]]))
    finally:
        eng.close()
