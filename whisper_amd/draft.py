"""Drafted (speculative) decoding: greedy verification of drafted token trees (include/whisper_amd.h, ``wx_tree_verify``)."""
from __future__ import annotations

import ctypes
from typing import Dict, Optional

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
    i32 = dict(dtype=torch.int32, device=dev)
    pick, path, accept, follow = torch.empty((n, nodes), **i32), torch.empty((n, nodes), **i32), torch.empty(n, **i32), torch.empty(n, **i32)
    logprob = torch.empty((n, nodes), dtype=torch.float32, device=dev)
    a = _lib.WxTreeCheck(n, nodes, vocab, _PRECISION[logits.dtype], dev.index, logits.data_ptr(), logits.stride(0), logits.stride(1), tokens.data_ptr(),
                         None if parents is None else parents.data_ptr(), None if counts is None else counts.data_ptr(),
                         None if suppress is None else suppress.data_ptr(), pick.data_ptr(), logprob.data_ptr(), path.data_ptr(), accept.data_ptr(),
                         follow.data_ptr())
    ref = ctypes.byref(a)
    need = lib.wx_tree_verify_work_bytes(ref)
    if need < 0:
        _check(int(need), "wx_tree_verify")
    work = torch.empty(need, dtype=torch.uint8, device=dev)
    a.d_work, a.work_bytes = work.data_ptr(), need
    _check(lib.wx_tree_verify(ref, _raw_stream(dev.index)), "wx_tree_verify")
    return {"pick": pick, "logprob": logprob, "path": path, "n_accept": accept, "next": follow}
