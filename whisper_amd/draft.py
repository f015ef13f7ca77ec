"""Drafted (speculative) decoding: greedy verification of drafted token trees (include/whisper_amd.h, ``wx_tree_verify``), where drafts come
from, and how candidates become a tree.  ``WhisperEngine.decode_draft`` is the loop that uses them.

A drafter is called with the ids of every row so far (prompt included) and the number of ids wanted, and returns for every row a list of
candidate continuations (lists of ids; none, one or several, of any length).  A row that needs none (it is finished, or at its limit) is
given as its prompt, and what comes back for it is not looked at.  ``EngineLanes`` calls one drafter from the threads of all lanes.

A drafter that needs the audio has a method ``listening(engine, mel, win_stride, row_stride, n_valid_frames, B)``: a context manager that
``transcribe_mel`` enters with the arguments of ``engine``'s last ``encode`` and leaves when these windows are decoded."""
from __future__ import annotations

import contextlib
import ctypes
import threading
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib
from .kvcache import _PRECISION, _check, _raw_stream


def verify_tree(logits: torch.Tensor, tokens: torch.Tensor, parents: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
                suppress: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
    """Greedy verification of a draft.  ``logits`` [n, n_nodes <= 64, n_vocab] (float32 or bfloat16): what the model answers to drafted
    token ``tokens[i, j]``, which follows token ``parents[i, j]`` (None: a chain); node 0 is the last token that is certain already.
    ``counts`` [n]: nodes that are there; ``suppress`` [n_vocab] (uint8): ids that must not be picked.

    Returns ``pick`` and ``logprob`` [n, n_nodes]: every node's largest logit's id (the lowest of equals) and its log-probability among
    the ids that are allowed; ``path`` [n, n_nodes] (padded with -1) and ``n_accept`` [n]: the nodes from node 0 down, each the first
    child whose token is its parent's pick; ``next`` [n]: the pick at the path's end, the one new token."""
    if logits.dim() != 3 or logits.dtype not in _PRECISION or not logits.is_cuda:
        raise ValueError("logits must be [n, n_nodes, n_vocab], float32 or bfloat16, on a GPU")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("logits require a gradient: verification has none (detach them)")
    n, nodes, vocab = logits.shape
    dev = logits.device
    if vocab and logits.stride(-1) != 1:
        logits = logits.contiguous()
    for t, what, shape, dtype in ((tokens, "tokens", (n, nodes), torch.int32), (parents, "parents", (n, nodes), torch.int32),
                                  (counts, "counts", (n,), torch.int32), (suppress, "suppress", (vocab,), torch.uint8)):
        if t is None and what != "tokens":
            continue
        if not torch.is_tensor(t) or t.dtype != dtype or t.device != dev or tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError(f"{what} must be a contiguous {dtype} tensor {list(shape)} on {dev}")
    lib = _lib.load()
    # one allocation for the whole numbers (each tensor is a host call), one for the log-probabilities
    cells = n * nodes
    a = _lib.WxTreeCheck(n, nodes, vocab, _PRECISION[logits.dtype], dev.index, logits.data_ptr(), logits.stride(0), logits.stride(1), tokens.data_ptr(),
                         None if parents is None else parents.data_ptr(), None if counts is None else counts.data_ptr(),
                         None if suppress is None else suppress.data_ptr())
    ref = ctypes.byref(a)
    need = lib.wx_tree_verify_work_bytes(ref)
    if need < 0:
        _check(int(need), "wx_tree_verify")
    buf = torch.empty(need // 4 + 2 * cells + 2 * n, dtype=torch.int32, device=dev)
    logprob = torch.empty((n, nodes), dtype=torch.float32, device=dev)
    _, pick, path, accept, follow = buf.split_with_sizes((need // 4, cells, cells, n, n))
    base = buf.data_ptr()
    a.d_work, a.work_bytes = base, need
    a.d_pick, a.d_path = base + need, base + need + 4 * cells
    a.d_n_accept, a.d_next = base + need + 8 * cells, base + need + 8 * cells + 4 * n
    a.d_logprob = logprob.data_ptr()
    _check(lib.wx_tree_verify(ref, _raw_stream(dev.index)), "wx_tree_verify")
    return {"pick": pick.view(n, nodes), "logprob": logprob, "path": path.view(n, nodes), "n_accept": accept, "next": follow}


def draft_tree(last: int, candidates: Sequence[Sequence[int]], max_nodes: int, max_depth: int, stop: int) -> Tuple[List[int], List[int]]:
    """Candidate continuations as one tree with shared beginnings: (tokens, parents), node 0 is ``last``, the id that is certain.  At most
    ``max_nodes`` nodes, ``max_depth`` ids below the root; a candidate ends before the id ``stop``.  The candidates grow side by side, id by
    id, so that a small tree holds the beginning of each."""
    tokens, parents = [int(last)], [-1]
    child: Dict[Tuple[int, int], int] = {}
    at = [0] * len(candidates)
    alive = list(range(len(candidates)))
    depth = 0
    while alive and depth < max_depth:
        going = []
        for c in alive:
            if depth >= len(candidates[c]) or int(candidates[c][depth]) == stop:
                continue
            key = (at[c], int(candidates[c][depth]))
            if key not in child:
                if len(tokens) >= max_nodes:
                    continue
                child[key] = len(tokens)
                tokens.append(key[1])
                parents.append(key[0])
            at[c] = child[key]
            going.append(c)
        alive, depth = going, depth + 1
    return tokens, parents


class NgramDraft:
    """Drafts from the row's own text: what followed the last occurrences of its last ``n`` ids (and, where there is none, of fewer, down
    to one), the latest first, up to ``branches`` of them.  Costs nothing on the GPU; speech repeats itself, and a prompt holds names."""

    def __init__(self, n: int = 3, branches: int = 2):
        if n < 1 or branches < 1:
            raise ValueError("n and branches must be at least 1")
        self.n, self.branches = int(n), int(branches)

    def __call__(self, rows: Sequence[Sequence[int]], k: int) -> List[List[List[int]]]:
        out = []
        for ids in rows:
            ids, found = list(ids), []
            for n in range(min(self.n, len(ids) - 1), 0, -1):
                tail = ids[-n:]
                for i in range(len(ids) - n - 1, -1, -1):
                    if ids[i:i + n] == tail:
                        found.append(ids[i + n:i + n + k])
                        if len(found) == self.branches:
                            break
                if found:
                    break
            out.append(found)
        return out


class EngineDraft:
    """Drafts from another engine with the same vocabulary (a smaller model): its greedy continuation of every row.  ``transcribe_mel`` has
    it encode each batch of windows as well (``listening``); where ``decode_draft`` is called directly, it must have encoded the same windows.
    The helper serves one batch at a time: lanes that share it decode in turn."""

    def __init__(self, engine):
        self.engine = engine
        self._turn = vars(engine).setdefault("_draft_turn", threading.RLock())     # one for each helper, whatever EngineDraft it is in

    @contextlib.contextmanager
    def listening(self, engine, mel, win_stride: int, row_stride: int, n_valid_frames: int, B: int):
        helper = self.engine
        if helper is engine:
            raise ValueError("an engine cannot draft for itself: a replica() can")
        if (helper.dims.n_vocab, helper.dims.n_mels, helper.torch_device) != (engine.dims.n_vocab, engine.dims.n_mels, engine.torch_device):
            raise ValueError("the drafting engine needs the same vocabulary, number of mel bands and device")
        if helper.max_batch < B:
            raise ValueError(f"the drafting engine takes {helper.max_batch} windows a batch, {B} are needed")
        with self._turn:
            helper.encode(mel, win_stride, row_stride, n_valid_frames, B)
            try:
                yield self
            finally:
                if helper.torch_device.type == "cuda":                              # the next batch may be on another stream
                    torch.cuda.current_stream(helper.torch_device).synchronize()

    def __call__(self, rows: Sequence[Sequence[int]], k: int) -> List[List[List[int]]]:
        room = self.engine.dims.n_text_ctx - 1
        if any(len(r) > room for r in rows):
            return [[] for _ in rows]
        with self._turn:
            return [[t] for t in self.engine.decode_rows(rows, max_new_tokens=k, suppress_blank=False)["tokens"]]
