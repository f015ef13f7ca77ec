"""Pages of a key/value cache on the GPU (whisper_amd/kvcache.py) against the entry-by-entry model of tests/kv_model.py: whole numbers and
copied rows have to be equal."""
import numpy as np
import pytest
import torch

from kv_model import INVALID, NOMEM, OK, PageModel
from whisper_amd.kvcache import PagedKVCache

pytestmark = pytest.mark.gpu


def make(L=2, H=3, D=64, PS=16, pages=40, seqs=8, width=6, dtype=torch.float32, seed=0):
    cache = PagedKVCache.allocate(L, H, D, pages, seqs, width, page_size=PS, dtype=dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    cache.k.copy_(torch.randn(cache.k.shape, generator=g, device="cuda"))
    cache.v.copy_(torch.randn(cache.v.shape, generator=g, device="cuda"))
    model = PageModel(pages, seqs, width, PS, cache.k.float().cpu().numpy().copy(), cache.v.float().cpu().numpy().copy())
    return cache, model


def same(cache, model):
    for name, want in model.state().items():
        np.testing.assert_array_equal(getattr(cache, name).cpu().numpy(), want, err_msg=name)
    np.testing.assert_array_equal(cache.k.float().cpu().numpy(), model.k)
    np.testing.assert_array_equal(cache.v.float().cpu().numpy(), model.v)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def status(t):
    return t.cpu().tolist()


def grow(cache, model, lens):
    """slots 0.. get lens committed tokens (an identity path over freshly reserved rows)"""
    ids = list(range(len(lens)))
    most = max(max(lens), 1)
    assert status(cache.reserve(i32(ids), i32(lens))) == model.reserve(ids, lens)
    path = np.tile(np.arange(most, dtype=np.int32), (len(lens), 1))
    assert status(cache.commit(i32(ids), i32(path), i32(lens))) == model.commit(ids, path, lens)


@pytest.mark.parametrize("PS,D,dtype", [(16, 64, torch.float32), (32, 128, torch.bfloat16), (256, 64, torch.bfloat16)])
def test_life_of_a_few_sequences(PS, D, dtype):
    cache, model = make(PS=PS, D=D, dtype=dtype)
    grow(cache, model, [PS * 2 + 5, 1, PS, 0])
    same(cache, model)
    # two children of 0, one of 2 and one of the empty 3; 1 becomes a child too and gives its page up
    dst, src = [4, 5, 6, 7, 1], [0, 0, 2, 3, 0]
    assert status(cache.fork(i32(dst), i32(src))) == model.fork(dst, src) == [OK] * 5
    same(cache, model)
    # the shared, partly filled last page is copied for everyone who asks, the parent among them; full pages stay shared
    ids = [5, 0, 4, 2, 7]
    assert status(cache.reserve(i32(ids), 3)) == model.reserve(ids, 3) == [OK] * 5
    same(cache, model)
    rng = np.random.RandomState(1)
    k = rng.randn(2, 5, 3, 3, D).astype(np.float32)
    v = rng.randn(2, 5, 3, 3, D).astype(np.float32)
    tk, tv = torch.tensor(k).cuda().to(dtype), torch.tensor(v).cuda().to(dtype)
    counts = [3, 0, 2, 1, 3]
    cache.append(i32(ids), tk, tv, counts=i32(counts))
    model.append(ids, tk.float().cpu().numpy(), tv.float().cpu().numpy(), counts, [0, 1])
    same(cache, model)
    path = [[0, 2, -1], [-1, -1, -1], [1, -1, -1], [0, -1, -1], [0, 1, 2]]
    taken = [2, 0, 1, 1, 3]
    assert status(cache.commit(i32(ids), i32(path), i32(taken))) == model.commit(ids, path, taken) == [OK] * 5
    same(cache, model)
    assert status(cache.truncate(i32([5, 6, 0]), i32([PS * 2, 1, 0]))) == model.truncate([5, 6, 0], [PS * 2, 1, 0])
    same(cache, model)
    assert int(cache.compact().item()) == model.compact()
    same(cache, model)
    assert status(cache.free(i32(list(range(8))))) == model.truncate(list(range(8)))
    same(cache, model)
    assert int(cache.refs.abs().sum().item()) == 0


def test_truncated_into_a_shared_page():
    """a page that two slots hold, cut short by one of them: its next token goes to a copy"""
    cache, model = make()
    grow(cache, model, [32])
    assert status(cache.fork(i32([1, 2]), i32([0, 0]))) == model.fork([1, 2], [0, 0])
    assert status(cache.truncate(i32([1]), i32([20]))) == model.truncate([1], [20])
    row = torch.randn(2, 1, 1, 3, 64, device="cuda")
    cache.append(i32([1]), row, row)                                   # not reserved: left out
    same(cache, model)
    assert status(cache.commit(i32([1]), i32([[0]]), i32([1]))) == model.commit([1], [[0]], [1]) == [INVALID]
    assert status(cache.reserve(i32([1]), 1)) == model.reserve([1], 1) == [OK]
    cache.append(i32([1]), row, row)
    model.append([1], row.cpu().numpy(), row.cpu().numpy(), None, [0, 1])
    same(cache, model)


def test_in_place_reorder_with_repeats():
    cache, model = make()
    grow(cache, model, [20, 33, 5, 16])
    for _ in range(3):
        dst, src = [0, 1, 2, 3], [2, 2, 1, 3]
        assert status(cache.fork(i32(dst), i32(src))) == model.fork(dst, src)
        same(cache, model)
        assert status(cache.reserve(i32(dst), 2)) == model.reserve(dst, 2)
        same(cache, model)
        path = np.tile(np.arange(2, dtype=np.int32), (4, 1))
        assert status(cache.commit(i32(dst), i32(path), i32([2] * 4))) == model.commit(dst, path, [2] * 4)
        same(cache, model)


@pytest.mark.parametrize("L,H", [(3, 2), (5, 16)])
def test_long_paths(L, H):
    """paths of hundreds of rows: some stay all along, some part early, late or behind the first 256, some are not paths behind the first 256"""
    N, n, PS = 700, 6, 64
    cache, model = make(L=L, H=H, PS=PS, pages=n * 12 + 1, seqs=n, width=12, dtype=torch.bfloat16)
    grow(cache, model, [3, 0, 17, 60, 1, 9])
    ids = list(range(n))
    assert status(cache.reserve(i32(ids), N)) == model.reserve(ids, N) == [OK] * n
    rows = torch.randn(L, n, N, H, 64, device="cuda").bfloat16()
    counts = [N, N, 690, N, N, 301]
    cache.append(i32(ids), rows, rows.flip(2), counts=i32(counts))
    model.append(ids, rows.float().cpu().numpy(), rows.flip(2).float().cpu().numpy(), counts, list(range(L)))
    same(cache, model)
    rng = np.random.RandomState(0)
    path = np.full((n, N), -1, np.int32)
    path[0] = np.arange(N)
    for i, stay in ((1, 0), (2, 200), (3, 256), (4, 400)):
        take = np.concatenate([np.arange(stay), np.sort(rng.choice(np.arange(stay, 690), 280, replace=False))])
        path[i, :len(take)] = take
    path[5, :300] = np.arange(300)
    path[5, 290] = 289
    taken = [N, 280, 480, 536, 680, 300]
    want = model.commit(ids, path, taken)
    assert status(cache.commit(i32(ids), i32(path), i32(taken))) == want == [OK] * 5 + [INVALID]
    same(cache, model)


def test_refused_entries_change_nothing():
    cache, model = make(pages=7)
    grow(cache, model, [17, 16])
    for call, args in [("truncate", ([0, 0, 9, -1, 1], [17, 0, 0, 0, 17])), ("fork", ([3, 3, 8, 4, 5], [0, 1, 0, 8, -2])),
                       ("reserve", ([0, 0, -1, 8], [1, 1, 1, 1])), ("reserve", ([0, 1], [-1, 1 << 30])), ("reserve", ([1, 0, 2, 3], [48, 60, 1, 0])),
                       ("commit", ([0, 0, 9], [[0], [0], [0]], [0, 0, 0])), ("commit", ([0, 1], [[0, 1], [1, 1]], [3, 2])),
                       ("commit", ([0], [[-1, 0]], [2])), ("commit", ([0], [[0, 1 << 30]], [2])), ("commit", ([0], [[0, 15]], [2])),
                       ("commit", ([0], [[0, 1]], [-1]))]:
        got = status(getattr(cache, call)(*[i32(a) for a in args]))
        assert got == getattr(model, call)(*args), (call, args, got)
        same(cache, model)


def test_pages_run_out_in_list_order():
    cache, model = make(pages=6, seqs=8)
    ids, extra = [3, 1, 5, 0, 2], [40, 16, 40, 0, 1]                    # 3 + 1 fit, 3 more do not, 0 need nothing, 1 comes too late
    got = status(cache.reserve(i32(ids), i32(extra)))
    assert got == model.reserve(ids, extra) == [OK, OK, NOMEM, OK, NOMEM]
    same(cache, model)
    assert status(cache.reserve(i32([2]), 17)) == model.reserve([2], 17) == [OK]
    same(cache, model)


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_random_traffic(seed):
    """many calls of every kind on a small pool, against the model after each"""
    rng = np.random.RandomState(seed)
    pages, seqs, width, PS = 61, 12, 9, 16
    cache, model = make(L=1, H=2, pages=pages, seqs=seqs, width=width, PS=PS, dtype=torch.bfloat16, seed=seed)
    for _ in range(60):
        ids = rng.permutation(seqs)[:rng.randint(1, seqs + 1)].tolist()
        kind = rng.randint(6)
        if kind == 0:
            lens = [int(rng.randint(0, model.lens[s] + 1)) for s in ids]
            assert status(cache.truncate(i32(ids), i32(lens))) == model.truncate(ids, lens)
        elif kind == 1:
            src = rng.randint(0, seqs, len(ids)).tolist()
            assert status(cache.fork(i32(ids), i32(src))) == model.fork(ids, src)
        elif kind == 2:
            assert int(cache.compact().item()) == model.compact()
        else:
            N = int(rng.randint(1, 20))
            extra = rng.randint(0, N + 1, len(ids)).tolist()
            assert status(cache.reserve(i32(ids), i32(extra))) == model.reserve(ids, extra)
            k = torch.randn(1, len(ids), N, 2, 64, device="cuda").bfloat16()
            v = torch.randn(1, len(ids), N, 2, 64, device="cuda").bfloat16()
            counts = rng.randint(0, N + 1, len(ids)).tolist()
            cache.append(i32(ids), k, v, counts=i32(counts))
            model.append(ids, k.float().cpu().numpy(), v.float().cpu().numpy(), counts, [0])
            path = np.full((len(ids), N), -1, np.int32)
            for i, c in enumerate(counts):
                way = np.sort(rng.permutation(max(1, c))[:rng.randint(0, max(1, c) + 1)])
                path[i, :len(way)] = way
                counts[i] = len(way)
            assert status(cache.commit(i32(ids), i32(path), i32(counts))) == model.commit(ids, path, counts)
        same(cache, model)


def test_a_pool_of_many_pages_and_slots():
    """more slots than a workgroup has threads, more pages than one scan step"""
    pages, seqs = 9000, 1500
    cache = PagedKVCache.allocate(1, 1, 64, pages, seqs, 8, dtype=torch.float32)
    model = PageModel(pages, seqs, 8, 16, cache.k.cpu().numpy().copy(), cache.v.cpu().numpy().copy())
    rng = np.random.RandomState(0)
    ids = rng.permutation(seqs).tolist()
    extra = rng.randint(0, 100, seqs).tolist()
    assert status(cache.reserve(i32(ids), i32(extra))) == model.reserve(ids, extra)
    path = np.tile(np.arange(100, dtype=np.int32), (seqs, 1))
    assert status(cache.commit(i32(ids), i32(path), i32(extra))) == model.commit(ids, path, extra)
    gone = ids[::3]
    assert status(cache.free(i32(gone))) == model.truncate(gone)
    dst, src = gone[:200], ids[1:400:2]
    assert status(cache.fork(i32(dst), i32(src))) == model.fork(dst, src)
    for name, want in model.state().items():
        np.testing.assert_array_equal(getattr(cache, name).cpu().numpy(), want, err_msg=name)
    assert int(cache.compact().item()) == model.compact()
    assert status(cache.reserve(i32(dst), 9)) == model.reserve(dst, 9)
    for name, want in model.state().items():
        np.testing.assert_array_equal(getattr(cache, name).cpu().numpy(), want, err_msg=name)


def test_strided_rows_one_layer():
    cache, model = make(dtype=torch.bfloat16, D=128)
    ids = [2, 0]
    cache.reserve(i32(ids), 5); model.reserve(ids, 5)
    base = torch.randn(2, 5, 9, 3, 128, device="cuda").bfloat16()          # [n, nodes, parts, heads, dim] as a fused projection leaves it
    k, v = base[:, :, 4], base[:, :, 7]
    assert not k.is_contiguous()
    cache.append(i32(ids), k, v, layer=1)
    model.append(ids, k.float().cpu().numpy()[None], v.float().cpu().numpy()[None], None, [1])
    same(cache, model)


def test_captured_and_replayed_cycle():
    """fork, reserve, append, commit in one graph, replayed with eager work between, against the model each time"""
    cache, model = make(pages=64)
    grow(cache, model, [20, 33])
    dst, src, ids = i32([2, 3]), i32([0, 1]), [2, 3]
    k = torch.randn(2, 2, 4, 3, 64, device="cuda")
    v = torch.randn(2, 2, 4, 3, 64, device="cuda")
    path, taken = i32([[0, 2, -1, -1], [1, 2, 3, -1]]), i32([2, 3])

    def cycle():
        cache.free(dst)
        cache.fork(dst, src)
        cache.reserve(dst, 4)
        cache.append(dst, k, v)
        return cache.commit(dst, path, taken)

    def model_cycle():
        model.truncate(ids)
        model.fork(ids, [0, 1])
        model.reserve(ids, 4)
        model.append(ids, k.cpu().numpy(), v.cpu().numpy(), None, [0, 1])
        return model.commit(ids, path.cpu().numpy(), [2, 3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cycle()
    torch.cuda.current_stream().wait_stream(side)
    model_cycle()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cycle()
    for i in range(4):
        k.copy_(torch.randn_like(k)); v.copy_(torch.randn_like(v))
        graph.replay()
        assert model_cycle() == status(out) == [OK, OK]
        same(cache, model)
        assert status(cache.truncate(i32([0]), i32([20 - i]))) == model.truncate([0], [20 - i])


def test_python_refusals():
    cache, _ = make()
    f = torch.zeros
    with pytest.raises(ValueError):
        cache.free(f(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        cache.free(f(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        cache.fork(i32([1, 2]), i32([0]))
    with pytest.raises(ValueError):
        cache.append(i32([0]), f(2, 1, 1, 3, 32, device="cuda"), f(2, 1, 1, 3, 32, device="cuda"))
    with pytest.raises(ValueError):
        cache.append(i32([0]), f(2, 1, 1, 3, 64, device="cuda").half(), f(2, 1, 1, 3, 64, device="cuda").half())
    with pytest.raises(ValueError):
        cache.commit(i32([0]), i32([0]), i32([1]))
    with pytest.raises(ValueError):
        PagedKVCache(cache.k, cache.v, cache.table, cache.refs[:-1].contiguous(), cache.lens, cache.held)
    with pytest.raises(ValueError):
        PagedKVCache(cache.k.half(), cache.v.half(), cache.table, cache.refs, cache.lens, cache.held)
    with pytest.raises(Exception, match="page_size"):
        PagedKVCache.allocate(1, 1, 64, 4, 2, 2, page_size=24)
