"""A paged key/value cache on the device and the operators of drafted decoding over it (include/whisper_amd.h, ``wx_cache_*`` and
``wx_tree_attention``): slots of sequences that share pages (``fork``), take them (``reserve``), give them up (``truncate``, ``free``),
hold a draft behind their committed tokens (``append``, or ``attend`` with the draft's keys and values), keep its accepted path
(``commit``), and a pool that closes up (``compact``).

Nothing here waits for the GPU: lists of slots, lengths and statuses are device tensors, so a whole drafted step can be captured into a
graph.  A cache is used by one stream of work at a time.

    cache = PagedKVCache.allocate(n_layers=32, n_kv_heads=20, head_dim=64, n_pages=1024, max_seqs=64, max_pages=28)
    slots = torch.arange(16, dtype=torch.int32, device="cuda")
    cache.reserve(slots, 24)                                             # room for a draft of 24 tokens
    for layer in range(32):
        o = cache.attend(layer, slots, q, parents, k=k, v=v)             # q [16, 24, heads, 64]; k, v [16, 24, 20, 64]
    r = draft.verify_tree(logits, tokens, parents)
    cache.commit(slots, r["path"], r["n_accept"])

The reference keeps one dense cache per call inside the model (ref:app/transcription/speech_recognition.py:55) and has none of this.
"""
from __future__ import annotations

import ctypes
import operator
from typing import Optional, Union

import torch

from . import _lib

_PRECISION = {torch.float32: 0, torch.bfloat16: 1}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _check(rc: int, what: str) -> None:
    if rc != 0:
        _lib.check(rc, what)


class PagedKVCache:
    """The buffers of a cache and the calls on it.  ``k`` and ``v`` [n_layers, n_pages, n_kv_heads, page_size, head_dim] (float32 or
    bfloat16), ``table`` [max_seqs, max_pages], ``refs`` [n_pages], ``lens`` and ``held`` [max_seqs] (int32), all contiguous on one
    GPU, are adopted as they are; ``allocate`` makes empty ones.  Slot s's token t is row ``t % page_size`` of page
    ``table[s, t // page_size]``."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, refs: torch.Tensor, lens: torch.Tensor, held: torch.Tensor):
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _PRECISION:
            raise ValueError("k and v must be [n_layers, n_pages, n_kv_heads, page_size, head_dim], float32 or bfloat16")
        n_layers, n_pages, n_kv_heads, page_size, head_dim = k.shape
        if table.dim() != 2 or refs.shape != (n_pages,) or lens.shape != (table.shape[0],) or held.shape != lens.shape:
            raise ValueError("table [max_seqs, max_pages], refs [n_pages], lens and held [max_seqs] do not fit the pools")
        for t in (table, refs, lens, held):
            if t.dtype != torch.int32:
                raise ValueError("table, refs, lens and held must be int32")
        for t in (k, v, table, refs, lens, held):
            if not t.is_cuda or t.device != k.device or not t.is_contiguous():
                raise ValueError("the cache's tensors must be contiguous and on one GPU")
        self.lib = _lib.load()
        self.k, self.v, self.table, self.refs, self.lens, self.held = k, v, table, refs, lens, held
        self.n_layers, self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = n_layers, n_pages, n_kv_heads, page_size, head_dim
        self.max_seqs, self.max_pages = table.shape
        self.device, self.dtype, self._index = k.device, k.dtype, k.device.index
        self._c = _lib.WxCache(
            d_k=k.data_ptr(), d_v=v.data_ptr(), d_table=table.data_ptr(), d_refs=refs.data_ptr(), d_lens=lens.data_ptr(), d_held=held.data_ptr(),
            n_layer=n_layers, n_pages=n_pages, n_kv_head=n_kv_heads, page_size=page_size, head_dim=head_dim, max_seqs=self.max_seqs,
            max_pages=self.max_pages, precision=_PRECISION[k.dtype], device=self._index)
        self._ref = ctypes.byref(self._c)
        ints = self.lib.wx_cache_work_ints(self._ref)
        if ints < 0:
            _check(int(ints), "wx_cache_work_ints")
        self._work = torch.empty(int(ints), dtype=torch.int32, device=self.device)
        self._c.d_work = self._work.data_ptr()
        _check(self.lib.wx_cache_truncate(self._ref, None, None, 0, None, None), "PagedKVCache")    # the host-side checks, no launch

    @classmethod
    def allocate(cls, n_layers: int, n_kv_heads: int, head_dim: int, n_pages: int, max_seqs: int, max_pages: int, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device: Union[int, str, torch.device] = 0) -> "PagedKVCache":
        """An empty cache: every slot free, every page free.  Its pools are not filled: no operator lets unwritten rows show."""
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                   torch.full((max_seqs, max_pages), -1, **i32), torch.zeros(n_pages, **i32), torch.zeros(max_seqs, **i32), torch.zeros(max_seqs, **i32))

    # -- arguments ----------------------------------------------------------------------------------------
    def _ids(self, t, what: str, n: Optional[int] = None, cols: Optional[int] = None) -> torch.Tensor:
        if not torch.is_tensor(t):
            t = torch.tensor(list(t), dtype=torch.int32, device=self.device)
        shape = t.shape
        if t.dtype is not torch.int32 or t.get_device() != self._index or not t.is_contiguous() or len(shape) != (1 if cols is None else 2) or \
                (n is not None and shape[0] != n) or (cols is not None and shape[1] != cols):
            want = f"[{'n' if n is None else n}{'' if cols is None else f', {cols}'}]"
            raise ValueError(f"{what} must be a contiguous int32 tensor {want} on {self.device}")
        return t

    @staticmethod
    def _int(x, what: str, least: int = 0, below: int = 1 << 31) -> int:
        x = operator.index(x)                                       # ctypes would cut a number to 32 bits without a word
        if not least <= x < below:
            raise ValueError(f"{what} must be {least} .. {below - 1}")
        return x

    def _rows(self, t: torch.Tensor, what: str, shape: tuple) -> torch.Tensor:
        if t.dtype != self.dtype or t.device != self.device or tuple(t.shape) != shape:
            raise ValueError(f"{what} must be {self.dtype} {list(shape)} on {self.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what} requires a gradient: the cache's operators have none (detach it)")
        return t if t.stride(-1) == 1 or t.numel() == 0 else t.contiguous()

    # -- pages --------------------------------------------------------------------------------------------
    def truncate(self, seqs, lens=None) -> torch.Tensor:
        """Slot ``seqs[i]`` keeps its first ``lens[i]`` tokens (None: none, the slot is freed) and gives up the pages behind them.
        Returns the status of every entry (0, or the negative ``wx_status`` of one that was refused and changed nothing)."""
        seqs = self._ids(seqs, "seqs")
        n = seqs.shape[0]
        if lens is not None:
            lens = self._ids(lens, "lens", n)
        status = torch.empty_like(seqs)
        _check(self.lib.wx_cache_truncate(self._ref, seqs.data_ptr(), None if lens is None else lens.data_ptr(), n, status.data_ptr(),
                                          _raw_stream(self._index)), "wx_cache_truncate")
        return status

    def free(self, seqs) -> torch.Tensor:
        """``truncate`` to nothing."""
        return self.truncate(seqs)

    def fork(self, dst, src) -> torch.Tensor:
        """Slot ``dst[i]`` becomes what slot ``src[i]`` was before the call, on the same pages (shared until ``reserve`` copies the last,
        partly filled one); what it held is given up.  Sources may repeat and may be destinations too."""
        dst = self._ids(dst, "dst")
        n = dst.shape[0]
        src = self._ids(src, "src", n)
        status = torch.empty_like(dst)
        _check(self.lib.wx_cache_fork(self._ref, dst.data_ptr(), src.data_ptr(), n, status.data_ptr(), _raw_stream(self._index)), "wx_cache_fork")
        return status

    def reserve(self, seqs, extra) -> torch.Tensor:
        """Room for ``extra`` (a number, or one for each slot) more tokens behind the committed ones, in pages of the slot's own.  Pages
        are taken lowest number first, in the order of the list; status -3 where they run out."""
        seqs = self._ids(seqs, "seqs")
        n = seqs.shape[0]
        each = None
        if hasattr(extra, "__index__") and not torch.is_tensor(extra):
            extra = self._int(extra, "extra")
        else:
            each = self._ids(extra, "extra", n)
        status = torch.empty_like(seqs)
        _check(self.lib.wx_cache_reserve(self._ref, seqs.data_ptr(), None if each is None else each.data_ptr(), extra if each is None else 0, n,
                                         status.data_ptr(), _raw_stream(self._index)), "wx_cache_reserve")
        return status

    def append(self, seqs, k: torch.Tensor, v: torch.Tensor, counts=None, layer: Optional[int] = None) -> None:
        """Rows of drafted tokens to their places behind the committed ones (reserved before): ``k``, ``v`` [n_layers, n, n_nodes,
        n_kv_heads, head_dim], or [n, n_nodes, n_kv_heads, head_dim] for one ``layer``.  The lengths stay as they are."""
        seqs = self._ids(seqs, "seqs")
        n = seqs.shape[0]
        if k.dim() != (5 if layer is None else 4):
            raise ValueError("k and v must be [n_layers, n, n_nodes, n_kv_heads, head_dim], or without n_layers for one layer")
        if layer is not None:
            layer = self._int(layer, "layer", 0, self.n_layers)
        lead = (self.n_layers,) if layer is None else ()
        shape = (*lead, n, k.shape[-3], self.n_kv_heads, self.head_dim)
        k, v = self._rows(k, "k", shape), self._rows(v, "v", shape)
        if counts is not None:
            counts = self._ids(counts, "counts", n)
        strides = [(ctypes.c_int64 * 4)(*(t.stride()[:4] if layer is None else (0, *t.stride()[:3]))) for t in (k, v)]
        _check(self.lib.wx_cache_append(self._ref, seqs.data_ptr(), None if counts is None else counts.data_ptr(), n, shape[-3], layer or 0,
                                        self.n_layers if layer is None else 1, k.data_ptr(), strides[0], v.data_ptr(), strides[1],
                                        _raw_stream(self._index)), "wx_cache_append")

    def commit(self, seqs, path, counts) -> torch.Tensor:
        """The accepted path of a draft: the row of drafted token ``path[i, k]`` moves to the k-th place behind the committed tokens, for
        k < ``counts[i]``, and the length grows by ``counts[i]``."""
        seqs = self._ids(seqs, "seqs")
        n = seqs.shape[0]
        counts = self._ids(counts, "counts", n)
        nodes = path.shape[-1] if torch.is_tensor(path) else -1
        path = self._ids(path, "path", n, nodes)
        status = torch.empty_like(seqs)
        _check(self.lib.wx_cache_commit(self._ref, seqs.data_ptr(), path.data_ptr(), counts.data_ptr(), n, nodes, status.data_ptr(),
                                        _raw_stream(self._index)), "wx_cache_commit")
        return status

    def compact(self) -> torch.Tensor:
        """The live pages move to the lowest numbers; returns how many there are ([1], int32): pages from there on are free."""
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        _check(self.lib.wx_cache_compact(self._ref, live.data_ptr(), _raw_stream(self._index)), "wx_cache_compact")
        return live

    # -- attention ------------------------------------------------------------------------------------------
    def attend(self, layer: int, seqs, q: torch.Tensor, parents=None, k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None,
               counts=None, scale: Optional[float] = None, split_tokens: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of drafted tokens: ``q`` [n, n_nodes <= 64, n_heads, head_dim]; node i of slot ``seqs[i]`` attends the committed
        tokens, itself and its ancestors by ``parents`` [n, n_nodes] (-1: follows the committed tokens; None: a chain).  ``k``, ``v``
        [n, n_nodes, n_kv_heads, head_dim] are appended first, or lie there already (None).  ``counts`` [n]: nodes that are there; the rows
        of the others, and of slot -1, are 0.  Slots that are out of range, not reserved far enough or listed twice while appending,
        and nodes with a parent out of range, give NaN.  ``scale``: head_dim ** -0.5 by default.  ``split_tokens``: see
        include/whisper_amd.h; > 0 makes a slot's result independent of the rest of the batch."""
        seqs = self._ids(seqs, "seqs")
        n = seqs.shape[0]
        if q.dim() != 4:
            raise ValueError("q must be [n, n_nodes, n_heads, head_dim]")
        nodes, heads = q.shape[1], q.shape[2]
        layer, split_tokens = self._int(layer, "layer", 0, self.n_layers), self._int(split_tokens, "split_tokens")
        q = self._rows(q, "q", (n, nodes, heads, self.head_dim))
        if (k is None) != (v is None):
            raise ValueError("k and v come together")
        if k is not None:
            shape = (n, nodes, self.n_kv_heads, self.head_dim)
            k, v = self._rows(k, "k", shape), self._rows(v, "v", shape)
        if parents is not None:
            parents = self._ids(parents, "parents", n, nodes)
        if counts is not None:
            counts = self._ids(counts, "counts", n)
        if out is None:
            out = torch.empty_like(q)
        elif self._rows(out, "out", (n, nodes, heads, self.head_dim)) is not out:
            raise ValueError("out's last dimension must be contiguous")
        a = _lib.WxTreeAttn(
            layer, n, nodes, heads, seqs.data_ptr(), None if parents is None else parents.data_ptr(), None if counts is None else counts.data_ptr(),
            q.data_ptr(), *q.stride()[:3], *((None, 0, 0, 0) if k is None else (k.data_ptr(), *k.stride()[:3])),
            *((None, 0, 0, 0) if v is None else (v.data_ptr(), *v.stride()[:3])), out.data_ptr(), *out.stride()[:3],
            self.head_dim ** -0.5 if scale is None else scale, split_tokens)
        ref = ctypes.byref(a)
        need = self.lib.wx_tree_attention_work_bytes(self._ref, ref)
        if need < 0:
            _check(int(need), "wx_tree_attention")
        if need > 0:
            work = torch.empty(need, dtype=torch.uint8, device=self.device)
            a.d_work, a.work_bytes = work.data_ptr(), need
        _check(self.lib.wx_tree_attention(self._ref, ref, _raw_stream(self._index)), "wx_tree_attention")
        return out
