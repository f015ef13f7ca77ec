"""Drafted decoding in bf16, on engines with cached keys and values and on those that attend the encoder output: where its ids part from greedy's, the
decoder holds both for as good as equal, and its log-probabilities are the decoder's for the ids it gives."""
import numpy as np
import pytest
import torch

from test_gpu_draft import Given, make, prompts
from whisper_amd.draft import NgramDraft

pytestmark = pytest.mark.gpu


def forced(eng, rows):
    """logits of the single-step decoder and of drafted passes (chains of 16) for whole rows, padded"""
    n, L = len(rows), max(map(len, rows))
    ids = np.full((n, L), eng.tok.eot, np.int32)
    for b, r in enumerate(rows):
        ids[b, :len(r)] = r
    d = torch.from_numpy(ids).cuda()
    slots, cache, got = torch.arange(n, dtype=torch.int32, device="cuda"), eng.draft_cache(n), []
    for at in range(0, L, 16):
        w = min(16, L - at)
        cache.reserve(slots, w)
        got.append(eng.draft_logits(cache, slots, d[:, at:at + w].contiguous()))
        cache.commit(slots, torch.arange(w, dtype=torch.int32, device="cuda").repeat(n, 1), torch.full((n,), w, dtype=torch.int32, device="cuda"))
    return eng.decoder_logits(torch.from_numpy(ids)).double().cpu(), torch.cat(got, 1).double().cpu()


@pytest.mark.parametrize("max_batch,form", [(4, "kv"), (32, "encoder_output")])
@pytest.mark.parametrize("name", ["micro", "tiny"])
@pytest.mark.parametrize("kind", ["none", "right", "mixed", "ngram"])
def test_bf16_ids_and_log_probabilities(max_batch, form, name, kind):
    """Two logits of one position are each off by at most the largest distance between the pass's and the decoder's logits of the row, measured here
    on the ids that came out: the decoder's margin between greedy's id and the draft's is at most twice that, and a log-probability (a logit less a
    logarithm of a sum of exponentials, which moves by no more than its largest term) as well, for every id."""
    eng, _, _ = make("bf16", max_batch, name=name)
    try:
        assert eng.cross_form == form
        ps = prompts(eng)
        want = eng.decode_rows(ps, max_new_tokens=40)["tokens"]
        drafter = NgramDraft(2, 3) if kind == "ngram" else Given([p + t + [eng.tok.eot] for p, t in zip(ps, want)], kind)
        got = eng.decode_draft(ps, drafter, n_nodes=9, n_draft=6, max_new_tokens=40)
        # the ids that were scored: the text, and the end where the row did not reach its limit
        rows = [p + t + ([eng.tok.eot] if len(t) < 40 else []) for p, t in zip(ps, got["tokens"])]
        dec, dra = forced(eng, rows)
        for b, (p, row) in enumerate(zip(ps, rows)):
            off = float((dec[b, len(p) - 1:len(row)] - dra[b, len(p) - 1:len(row)]).abs().max())
            theirs, score = p + want[b] + [eng.tok.eot], 0.0
            parted = False
            for at in range(len(p), len(row)):
                x = dec[b, at - 1].clone()
                x[list(eng.suppress_ids) + ([eng.tok.blank, eng.tok.eot] if at == len(p) else [])] = -np.inf
                score += float(torch.log_softmax(x, -1)[row[at]])
                if not parted and at < len(theirs) and theirs[at] != row[at]:
                    parted = True
                    assert float(x[theirs[at]] - x[row[at]]) <= 2 * off, (b, at)
                if not parted:
                    assert float(x.max() - x[row[at]]) <= 2 * off, (b, at)
            assert abs(got["sum_logprobs"][b] - score) <= 2 * off * (len(row) - len(p)) + 1e-3, (b, got["sum_logprobs"][b], score)
    finally:
        eng.close()
