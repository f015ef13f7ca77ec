"""Refusals of the paged cache's C entry points (include/whisper_amd.h, wx_cache_*, wx_tree_*): all of them are decided on the host before
any HIP call, so they are tested without a GPU."""
import ctypes

import pytest

from whisper_amd import _lib

A = 1 << 20          # an aligned address that nothing reads


def cache(**kw):
    base = dict(d_k=A, d_v=A, d_table=A, d_refs=A, d_lens=A, d_held=A, d_work=A, n_layer=2, n_pages=8, n_kv_head=2, page_size=16,
                head_dim=64, max_seqs=4, max_pages=4, precision=1, device=0)
    base.update(kw)
    return _lib.WxCache(**base)


def attn(**kw):
    base = dict(layer=0, n=1, n_nodes=4, n_head=2, d_seqs=A, d_q=A, d_out=A, q_head=64, o_head=64, scale=1.0)
    base.update(kw)
    return _lib.WxTreeAttn(**base)


def check(**kw):
    base = dict(n=1, n_nodes=4, n_vocab=100, precision=0, device=0, d_logits=A, d_tokens=A, d_pick=A, d_logprob=A, d_path=A, d_n_accept=A,
                d_next=A, d_work=A, work_bytes=1 << 20)
    base.update(kw)
    return _lib.WxTreeCheck(**base)


@pytest.mark.parametrize("kw", [dict(d_k=0), dict(d_table=0), dict(d_work=0), dict(page_size=8), dict(n_pages=0x40000000), dict(page_size=48), dict(page_size=512), dict(head_dim=80),
                                dict(n_pages=0), dict(max_seqs=0), dict(max_seqs=8193), dict(max_pages=0), dict(precision=2), dict(n_layer=0),
                                dict(n_kv_head=0), dict(d_k=A + 4), dict(d_refs=A + 8), dict(max_pages=1 << 28)])
def test_bad_cache_is_refused_by_every_call(kw):
    lib, c = _lib.load(), cache(**kw)
    r, s = ctypes.byref(c), (ctypes.c_int64 * 4)()
    assert lib.wx_cache_truncate(r, A, None, 1, None, None) == -1
    assert lib.wx_cache_fork(r, A, A, 1, None, None) == -1
    assert lib.wx_cache_reserve(r, A, None, 1, 1, None, None) == -1
    assert lib.wx_cache_append(r, A, None, 1, 1, 0, 1, A, s, A, s, None) == -1
    assert lib.wx_cache_commit(r, A, A, A, 1, 1, None, None) == -1
    assert lib.wx_cache_compact(r, None, None) == -1
    assert lib.wx_tree_attention(r, ctypes.byref(attn()), None) == -1
    assert lib.wx_last_error()


def test_null_and_lists():
    lib, c = _lib.load(), cache()
    r, s = ctypes.byref(c), (ctypes.c_int64 * 4)()
    for n in (-1, 5):                                               # more entries than slots cannot be distinct
        assert lib.wx_cache_truncate(r, A, None, n, None, None) == -1
        assert lib.wx_cache_fork(r, A, A, n, None, None) == -1
        assert lib.wx_cache_reserve(r, A, None, 1, n, None, None) == -1
    assert lib.wx_cache_truncate(None, A, None, 1, None, None) == -1
    assert lib.wx_cache_truncate(r, None, None, 1, None, None) == -1
    assert lib.wx_cache_fork(r, A, None, 1, None, None) == -1
    assert lib.wx_cache_reserve(r, A, None, -1, 1, None, None) == -1
    assert lib.wx_cache_commit(r, A, None, A, 1, 1, None, None) == -1
    assert lib.wx_cache_commit(r, A, A, None, 1, 1, None, None) == -1
    for layer0, layers in ((-1, 1), (0, 3), (2, 1), (0, 0)):
        assert lib.wx_cache_append(r, A, None, 1, 1, layer0, layers, A, s, A, s, None) == -1
    assert lib.wx_cache_append(r, A, None, 1, 1, 0, 1, A + 2, s, A, s, None) == -1
    odd = (ctypes.c_int64 * 4)(0, 0, 0, 12)
    assert lib.wx_cache_append(r, A, None, 1, 1, 0, 1, A, odd, A, s, None) == -1
    # nothing to do is allowed, without a GPU too
    assert lib.wx_cache_truncate(r, None, None, 0, None, None) == 0
    assert lib.wx_cache_fork(r, None, None, 0, None, None) == 0
    assert lib.wx_cache_reserve(r, None, None, 3, 0, None, None) == 0
    assert lib.wx_cache_work_ints(r) > 8 and lib.wx_cache_work_ints(None) == -1


@pytest.mark.parametrize("kw", [dict(layer=2), dict(layer=-1), dict(n=-1), dict(n=8193), dict(n_nodes=0), dict(n_nodes=65), dict(n_head=3), dict(n_head=1),
                                dict(n_head=34), dict(split_tokens=-1), dict(d_q=0), dict(d_seqs=0), dict(d_out=0), dict(d_kn=A), dict(d_vn=A),
                                dict(q_head=60), dict(o_node=-8), dict(d_q=A + 8), dict(d_kn=A, d_vn=A, kn_head=4)])
def test_bad_attention_is_refused(kw):
    lib, c = _lib.load(), cache()
    assert lib.wx_tree_attention(ctypes.byref(c), ctypes.byref(attn(**kw)), None) == -1


def test_empty_attention():
    lib, c = _lib.load(), cache()
    assert lib.wx_tree_attention(ctypes.byref(c), ctypes.byref(attn(n=0)), None) == 0
    assert lib.wx_tree_attention(ctypes.byref(c), None, None) == -1


@pytest.mark.parametrize("kw", [dict(n=-1), dict(n=65536), dict(n_nodes=0), dict(n_nodes=65), dict(n_vocab=0), dict(precision=3), dict(d_logits=0), dict(d_tokens=0),
                                dict(d_next=0), dict(d_work=0), dict(work_bytes=1), dict(l_seq=-1)])
def test_bad_verification_is_refused(kw):
    assert _lib.load().wx_tree_verify(ctypes.byref(check(**kw)), None) == -1


def test_empty_verification():
    lib = _lib.load()
    assert lib.wx_tree_verify(ctypes.byref(check(n=0)), None) == 0 and lib.wx_tree_verify(None, None) == -1
