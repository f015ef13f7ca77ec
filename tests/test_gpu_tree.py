"""Tree attention over the paged cache and greedy verification of drafts (whisper_amd/kvcache.py, whisper_amd/draft.py) against 64-bit
plain forms (tests/kv_model.py), and a whole drafted step of them together."""
import numpy as np
import pytest
import torch

import kv_model as km
from whisper_amd.draft import verify_tree
from whisper_amd.kvcache import PagedKVCache

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def trees(rng, n, N):
    par = np.full((n, N), -1, np.int32)
    for i in range(n):
        for j in range(1, N):
            par[i, j] = rng.randint(-1, j) if rng.rand() < 0.5 else j - 1
    return par


class Case:
    """a cache whose every row is NaN but for committed (and, where asked, drafted) tokens, with those tokens on the host"""

    def __init__(self, lens, N, heads, kv_heads, D, PS, dtype, append=True, layers=2, layer=1, seed=0, counts=None):
        rng = np.random.RandomState(seed)
        self.n, self.N, self.heads, self.H, self.D, self.dtype, self.layer, self.append = len(lens), N, heads, kv_heads, D, dtype, layer, append
        self.lens, self.counts = np.asarray(lens), np.full(len(lens), N) if counts is None else np.asarray(counts)
        room = [-(-(int(l) + N) // PS) for l in lens]
        pages = sum(room) + 3
        self.cache = PagedKVCache.allocate(layers, kv_heads, D, pages, self.n + 1, max(room), page_size=PS, dtype=dtype)
        self.cache.k.fill_(float("nan")); self.cache.v.fill_(float("nan"))
        order = rng.permutation(pages).tolist()
        table, refs = np.full((self.n + 1, max(room)), -1, np.int32), np.zeros(pages, np.int32)
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *shape: torch.randn(shape, generator=g).to(dtype)  # noqa: E731
        self.q, self.kn, self.vn = rnd(self.n, N, heads, D), rnd(self.n, N, kv_heads, D), rnd(self.n, N, kv_heads, D)
        self.par = trees(rng, self.n, N)
        self.pre = []
        k, v = self.cache.k.cpu(), self.cache.v.cpu()
        self.slots = rng.permutation(self.n + 1)[:self.n]
        lens_dev, held = np.zeros(self.n + 1, np.int32), np.zeros(self.n + 1, np.int32)
        for i, s in enumerate(self.slots):
            own = [order.pop() for _ in range(room[i])]
            table[s, :room[i]] = own
            refs[own] = 1
            lens_dev[s], held[s] = lens[i], room[i]
            K, V = rnd(int(lens[i]), kv_heads, D), rnd(int(lens[i]), kv_heads, D)
            self.pre.append((K, V))
            for t in range(int(lens[i]) + (0 if append else int(self.counts[i]))):
                src = (K, V, t) if t < lens[i] else (self.kn[i], self.vn[i], t - int(lens[i]))
                k[layer, own[t // PS], :, t % PS], v[layer, own[t // PS], :, t % PS] = src[0][src[2]], src[1][src[2]]
        self.cache.k.copy_(k); self.cache.v.copy_(v)
        self.cache.table.copy_(torch.from_numpy(table)); self.cache.refs.copy_(torch.from_numpy(refs))
        self.cache.lens.copy_(torch.from_numpy(lens_dev)); self.cache.held.copy_(torch.from_numpy(held))

    def run(self, **kw):
        args = dict(parents=i32(self.par), counts=i32(self.counts))
        if self.append:
            args.update(k=self.kn.cuda(), v=self.vn.cuda())
        args.update(kw)
        return self.cache.attend(self.layer, i32(self.slots), args.pop("q", self.q.cuda()), **args)

    def check(self, out, scale=None, par=None):
        scale = self.D ** -0.5 if scale is None else scale
        par = self.par if par is None else par
        out = out.float().cpu().numpy().astype(np.float64)
        for i in range(self.n):
            c = int(self.counts[i])
            assert not out[i, c:].any(), "rows that are not there are 0"
            if c == 0:
                continue
            K, V = self.pre[i]
            K, V = torch.cat([K, self.kn[i, :c]]).float().numpy(), torch.cat([V, self.vn[i, :c]]).float().numpy()
            o, mass, reach = km.tree_attention(self.q[i, :c].float().numpy(), K, V, par[i, :c], scale)
            bound = km.attention_bound(o, mass, reach, self.D, len(K), self.dtype == BF16)
            off = np.abs(out[i, :c] - o)
            assert (off <= bound).all(), (i, float((off / bound).max()))


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("lens,N,heads,kv_heads,D,PS", [
    ([0], 1, 1, 1, 64, 16), ([1], 1, 2, 1, 64, 16), ([0, 5], 3, 2, 2, 64, 16), ([15, 16, 17], 7, 6, 6, 64, 16), ([31, 64, 65, 100], 16, 4, 2, 64, 32),
    ([300, 1, 77], 24, 20, 20, 64, 16), ([447] * 3, 1, 20, 20, 64, 16), ([200, 513], 64, 8, 2, 128, 64), ([129], 33, 16, 1, 128, 16),
    ([1000, 63], 17, 6, 2, 128, 128), ([700], 5, 12, 4, 64, 256), ([2500, 3], 2, 3, 3, 128, 16),
    # every kernel and both of its ways of cutting the work: rows of a key / value head x head size x short and long contexts
    ([90, 200], 24, 3, 3, 64, 16), ([1500, 20, 900], 24, 3, 3, 64, 16), ([100], 60, 2, 1, 64, 32), ([1400, 700], 60, 2, 1, 64, 32),
    ([33, 129], 50, 8, 2, 64, 16), ([1300, 40], 50, 8, 2, 64, 16), ([60, 5], 20, 4, 4, 128, 16), ([1100, 64], 20, 4, 4, 128, 16),
    ([65, 200], 40, 8, 2, 128, 32), ([4000], 40, 8, 2, 128, 32), ([130], 64, 16, 2, 128, 16), ([900, 2000], 64, 16, 2, 128, 64), ([50], 64, 16, 1, 64, 16)])
@pytest.mark.parametrize("append", [True, False])
def test_against_64_bits(dtype, lens, N, heads, kv_heads, D, PS, append):
    c = Case(lens, N, heads, kv_heads, D, PS, dtype, append=append, seed=N + len(lens))
    out = c.run()
    c.check(out)
    if append:                                                     # the rows lie in the cache now, and reading them there gives the same
        c.append = False
        assert torch.equal(c.run(), out)


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("n,N,heads,kv_heads,D,longest", [(130, 1, 8, 8, 64, 500), (129, 5, 24, 8, 64, 90), (66, 16, 16, 16, 128, 140), (1100, 1, 4, 1, 64, 33), (35, 2, 60, 30, 128, 508),
                                                          (70, 3, 24, 12, 128, 60), (50, 20, 32, 8, 64, 60), (48, 24, 20, 20, 64, 400), (400, 33, 2, 1, 64, 20)])
def test_many_short_sequences(dtype, n, N, heads, kv_heads, D, longest):
    """more sequences x heads than waves fit at once, short enough for a wave each: ragged, some empty, some padding, some refused"""
    rng = np.random.RandomState(n + N)
    c = Case(rng.randint(0, longest + 1, n), N, heads, kv_heads, D, 16, dtype, seed=n, counts=rng.randint(0, N + 1, n))
    c.check(c.run())
    c.append = False
    before = c.run()
    c.check(before)
    slots = c.slots.copy()
    slots[[3, 20]] = -1, n + 5
    c.cache.refs[c.cache.table[int(slots[7]), 0]] = 2                          # (a page that is shared does not matter to a call that appends nothing)
    got = c.cache.attend(c.layer, i32(slots), c.q.cuda(), parents=i32(c.par), counts=i32(c.counts))
    assert not got[3].any() and torch.isnan(got[20]).all()
    rest = [i for i in range(n) if i not in (3, 20)]
    assert torch.equal(got[rest], before[rest])
    # appending: a slot named twice and one whose page is shared are NaN, and leave the cache as it was
    slots[30] = slots[31]
    held = int(c.lens[7]) // 16
    c.cache.refs[c.cache.table[int(slots[7]), held]] = 2
    was = c.cache.k.clone()
    kn, vn = torch.randn_like(c.kn).cuda(), torch.randn_like(c.vn).cuda()
    got = c.cache.attend(c.layer, i32(slots), c.q.cuda(), parents=i32(c.par), counts=i32(c.counts), k=kn, v=vn)
    for i in (7, 31):
        assert torch.isnan(got[i]).all() if c.counts[i] > 0 else True
        own = c.cache.table[int(c.slots[i]), :-(-(int(c.lens[i]) + N) // 16)].long()
        if i == 7:
            assert torch.equal(c.cache.k[:, own].nan_to_num(9.0), was[:, own].nan_to_num(9.0))
    i = next(x for x in range(40, n) if c.counts[x] > 0) if n > 40 else 34
    if c.counts[i] > 0:
        page, row = int(c.cache.table[int(slots[i]), int(c.lens[i]) // 16]), int(c.lens[i]) % 16
        assert torch.equal(c.cache.k[c.layer, page, :, row], kn[i, 0])


@pytest.mark.parametrize("dtype,D,longest", [(torch.float32, 64, 300), (torch.float32, 64, 440), (BF16, 128, 300), (BF16, 128, 470)])
def test_very_many_sequences(dtype, D, longest):
    lens = np.random.RandomState(longest).randint(0, 21, 2001)
    lens[[0, 1000, 2000]] = longest
    c = Case(lens, 2, 2, 1, D, 16, dtype, seed=longest)
    c.check(c.run())
    c.append = False
    c.check(c.run())


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("n,N,heads,kv_heads,D,longest", [(1, 3, 1, 1, 64, 5000), (3, 2, 2, 1, 128, 3000), (8, 64, 8, 4, 64, 700), (17, 64, 8, 4, 64, 640), (33, 64, 8, 8, 64, 560),
                                                          (9, 33, 8, 4, 128, 700), (24, 33, 16, 8, 128, 530)])
def test_many_pieces_and_many_rows(dtype, n, N, heads, kv_heads, D, longest):
    """a merge with one row a workgroup (all threads on its pieces), with some, and with as many as it holds"""
    lens = np.random.RandomState(n).randint(0, longest + 1, n)
    lens[-1] = longest
    c = Case(lens, N, heads, kv_heads, D, 16, dtype, seed=n)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_ragged_counts_padding_and_chain(dtype):
    c = Case([40, 3, 0, 100], 12, 4, 2, 64, 16, dtype, counts=[12, 0, 5, 1])
    c.check(c.run())
    chain = np.tile(np.arange(-1, 11, dtype=np.int32), (4, 1))
    c.check(c.run(parents=None), par=chain)
    # a padded batch: entries of slot -1 are 0, the others unchanged
    pad = c.cache.attend(c.layer, torch.cat([i32([-1]), i32(c.slots), i32([-1])]), torch.cat([c.q[:1], c.q, c.q[:1]]).cuda(),
                         parents=i32(np.concatenate([c.par[:1], c.par, c.par[:1]])), counts=i32([12, *c.counts, 12]))
    assert not pad[0].any() and not pad[5].any()
    c.check(pad[1:5])


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_infinities_and_nan_in_masked_rows(dtype, D):
    """a drafted row that a node does not attend has no effect on it, whatever it holds; those that attend it get what IEEE gives"""
    c = Case([50, 7], 10, 4, 2, D, 16, dtype)
    c.par[:] = np.array([-1, 0, 0, 1, 1, 2, -1, 6, 5, 3])
    clean = c.run()
    bad = 2                                                        # 5 and 8 descend from it
    hit = np.zeros(10, bool)
    hit[[2, 5, 8]] = True
    for what in (float("nan"), float("inf"), -float("inf")):
        for which in ("kn", "vn"):
            rows = getattr(c, which).clone()
            rows[:, bad] = what
            out = c.run(**{"k" if which == "kn" else "v": rows.cuda()})
            assert torch.equal(out[:, ~hit], clean[:, ~hit]), (what, which)
            if which == "vn":
                assert not torch.isfinite(out[:, hit]).any()
    c.check(c.run())


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_large_scores_and_lowest_values(dtype):
    """scores of thousands, and keys that all give the type's lowest value: a softmax over equal scores"""
    c = Case([70], 6, 2, 2, 64, 16, dtype, seed=3)
    c.q *= 60
    c.check(c.run())
    c.q[:] = 0
    c.check(c.run())


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_strided_tensors_and_out(dtype):
    c = Case([33, 90], 6, 4, 4, 64, 16, dtype, seed=5)
    qkv = torch.stack([c.q, c.kn, c.vn], 2).cuda()                  # [n, N, 3, heads, D]
    out = torch.full((2, 8, 6, 64), 7.0, dtype=dtype, device="cuda").transpose(1, 2)     # [n, 6, 8, D]: heads outermost, 4 of 8 used
    got = c.cache.attend(c.layer, i32(c.slots), qkv[:, :, 0], parents=i32(c.par), k=qkv[:, :, 1], v=qkv[:, :, 2], out=out[:, :, 2:6])
    c.check(got)
    assert (out[:, :, :2] == 7).all() and (out[:, :, 6:] == 7).all()


def test_scale_and_split():
    c = Case([1500, 10, 600], 8, 4, 2, 64, 16, BF16, seed=6)
    c.check(c.run(scale=0.3), scale=0.3)
    for split in (64, 100, 512, 1 << 20):
        c.check(c.run(split_tokens=split))
    # with pieces of a fixed length a sequence's result does not depend on its neighbours
    both = c.run(split_tokens=128)
    c.append = False
    for i in range(3):
        one = c.cache.attend(c.layer, i32(c.slots[i:i + 1]), c.q[i:i + 1].cuda(), parents=i32(c.par[i:i + 1]), split_tokens=128)
        assert torch.equal(one[0], both[i])


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_refused_entries_give_nan_and_append_nothing(dtype):
    c = Case([40, 20, 30], 4, 2, 2, 64, 16, dtype, seed=7)
    before = c.cache.k.clone()
    ok = c.run()
    c.cache.k.copy_(before)
    slots = c.slots.copy()
    c.cache.held[int(slots[1])] = 1                                 # 16 rows held, 20 committed
    out = c.run()
    assert torch.equal(out[0], ok[0]) and torch.equal(out[2], ok[2]) and torch.isnan(out[1]).all()
    c.cache.held[int(slots[1])] = 2
    c.cache.table[int(slots[1]), 0] = 10 ** 6                       # a page that is none
    out = c.run()
    assert torch.equal(out[0], ok[0]) and torch.isnan(out[1]).all()
    c.cache.k.copy_(before)
    page = int(c.cache.table[int(slots[2]), 1].item())
    c.cache.refs[page] = 2                                          # the page of the draft is someone else's too
    out = c.run()
    assert torch.equal(out[0], ok[0]) and torch.isnan(out[2]).all()
    p2 = c.cache.k[:, page].clone()
    assert torch.equal(p2.nan_to_num(9), before[:, page].nan_to_num(9))
    c.cache.refs[page] = 1
    # the same slot twice: only its first entry appends
    twice = i32([slots[0], slots[0], 99])
    out = c.cache.attend(c.layer, twice, c.q.cuda(), parents=i32(c.par), k=c.kn[[0, 1, 2]].cuda(), v=c.vn[[0, 1, 2]].cuda())
    assert torch.equal(out[0], ok[0]) and torch.isnan(out[1:]).all()
    # twice, reading only, is allowed
    out = c.cache.attend(c.layer, i32([slots[0]] * 3), c.q[[0, 0, 0]].cuda(), parents=i32(c.par[[0, 0, 0]]))
    assert torch.equal(out[0], out[2]) and torch.equal(out[0], ok[0])
    # parents that are not before their node, and what hangs on them
    par = c.par.copy()
    par[0] = [-1, 2, 0, 1]
    out = c.cache.attend(c.layer, i32(slots[:1]), c.q[:1].cuda(), parents=i32(par[:1]))[0]
    assert torch.isfinite(out[[0, 2]]).all() and torch.isnan(out[[1, 3]]).all()


def test_other_stream_and_replayed_graph():
    c = Case([200, 31], 8, 4, 2, 64, 16, BF16, seed=8)
    want = c.run()
    q, k, v, par, cnt, slots = c.q.cuda(), c.kn.cuda(), c.vn.cuda(), i32(c.par), i32(c.counts), i32(c.slots)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.cache.attend(c.layer, slots, q, parents=par, k=k, v=v, counts=cnt)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.cache.attend(c.layer, slots, q, parents=par, k=k, v=v, counts=cnt)
    for i in range(4):
        new = torch.randn(c.q.shape, generator=torch.Generator().manual_seed(i)).to(BF16)
        q.copy_(new)
        eager = c.cache.attend(c.layer, slots, q, parents=par, k=k, v=v, counts=cnt)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_a_fixed_cut_does_not_see_the_batch():
    """32-bit results of long sequences in pieces of a fixed length, alone and among many: the pieces are merged in the same order"""
    lens = np.random.RandomState(3).randint(0, 3000, 40)
    lens[5], lens[7] = 3000, 2999
    c = Case(lens, 16, 8, 2, 64, 16, torch.float32, seed=8)
    both = c.run(split_tokens=64)
    c.check(both)
    c.append = False
    for i in (5, 7, 39):
        one = c.cache.attend(c.layer, i32(c.slots[i:i + 1]), c.q[i:i + 1].cuda(), parents=i32(c.par[i:i + 1]), split_tokens=64)
        assert torch.equal(one[0], both[i])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [2000, 16384])
def test_one_long_piece_in_32_bits(D, L):
    """one workgroup takes the whole sequence: the root mean square of the error, against that of the result.  A wave adds up a quarter of the
    keys; every addition is off by half a step, 2^-24, of a sum that grows as a random walk does: 2^-24 sqrt(L / 4 / 2) of the result.  Scores
    and exponentials add a few steps that do not grow with L."""
    H, pages = 2, L // 16 + 1
    g = torch.Generator().manual_seed(L + D)
    c = PagedKVCache.allocate(1, H, D, pages, 1, pages, dtype=torch.float32)
    k, v = (torch.randn(pages, H, 16, D, generator=g) for _ in range(2))
    c.k[0], c.v[0] = k.cuda(), v.cuda()
    c.table.copy_(i32([range(pages)])); c.refs.fill_(1); c.held.fill_(pages); c.lens.fill_(L - 1)
    q = torch.randn(1, 1, 3 * H, D, generator=g)
    got = c.attend(0, i32([0]), q.cuda(), split_tokens=1 << 20)[0, 0].cpu().double()
    K, V = (x.permute(1, 0, 2, 3).reshape(H, -1, D)[:, :L].double() for x in (k, v))
    want = (torch.softmax(q[0, 0].view(H, 3, D).double() @ K.transpose(1, 2) * D ** -0.5, -1) @ V).reshape(3 * H, D)
    assert float(((got - want) ** 2).sum().sqrt() / (want ** 2).sum().sqrt()) <= 2.0 ** -24 * ((L / 8) ** 0.5 + 16)


def test_the_output_may_be_the_queries():
    c = Case([700, 3, 90, 0], 9, 6, 2, 64, 16, BF16, seed=9)
    q = c.q.cuda()
    assert c.run(q=q, out=q) is q
    c.check(q)


def test_offsets_past_32_bits():
    """the last layer and the last pages of pools of 9 GB: the same results as in a small pool, and pages copied, appended to and moved there"""
    H, D, PS, L, P = 8, 128, 64, 3, 24000
    big = PagedKVCache.allocate(L, H, D, P, 3, 20, page_size=PS, dtype=BF16)
    small = PagedKVCache.allocate(1, H, D, 8, 3, 20, page_size=PS, dtype=BF16)
    assert big.k.numel() > 2 ** 32
    big.refs.fill_(1)
    big.refs[P - 8:] = 0
    ids = i32([0])
    kv = torch.randn(2, 1, 1, 200, H, D, device="cuda").to(BF16)
    q = torch.randn(1, 1, 4 * H, D, device="cuda").to(BF16)
    outs = []
    for cache, layer in ((big, 2), (small, 0)):
        assert cache.reserve(ids, 200).tolist() == [0]
        cache.append(ids, kv[0, 0], kv[1, 0], layer=layer)
        cache.commit(ids, i32([list(range(0, 150)) + [199] + [-1] * 49]), i32([151]))
        assert cache.fork(i32([1]), ids).tolist() == [0] and cache.reserve(i32([1]), 5).tolist() == [0]
        new = kv[:, 0, :, 7:12]
        outs.append(cache.attend(layer, i32([1]), q.expand(1, 5, 4 * H, D), k=new[0], v=new[1]))
    assert big.table[1, 0] >= P - 8 and torch.equal(outs[0], outs[1])
    for t in (0, 1):
        rows = int(small.lens[t].item())
        for pos in (0, 63, 64, 150, rows - 1):
            a = big.k[2, int(big.table[t, pos // PS]), :, pos % PS]
            assert torch.equal(a, small.k[0, int(small.table[t, pos // PS]), :, pos % PS])


def test_attend_refusals():
    c = Case([4], 2, 2, 2, 64, 16, BF16)
    s = i32(c.slots)
    with pytest.raises(ValueError):
        c.cache.attend(0, s, c.q.cuda().float())
    with pytest.raises(ValueError):
        c.cache.attend(0, s, c.q.cuda(), k=c.kn.cuda())
    with pytest.raises(ValueError):
        c.cache.attend(0, s, c.q.cuda(), parents=i32([[0]]))
    with pytest.raises(ValueError):
        c.cache.attend(0, s, c.q.cuda().requires_grad_())
    with pytest.raises(Exception, match="layer"):
        c.cache.attend(2, s, c.q.cuda())
    with pytest.raises(Exception, match="n_nodes"):
        c.cache.attend(0, s, torch.zeros(1, 65, 2, 64, dtype=BF16, device="cuda"))
    assert c.cache.attend(0, i32([]), c.q.cuda()[:0]).shape == (0, 2, 2, 64)


# ---- verification ---------------------------------------------------------------------------------------------------------------------

def verify_case(rng, n, N, V, dtype):
    logits = torch.tensor(rng.randn(n, N, V) * 3, dtype=torch.float32).to(dtype)
    par, tokens = trees(rng, n, N), rng.randint(0, V, (n, N))
    for b in range(n):
        for j in range(1, N):
            if par[b, j] >= 0 and rng.rand() < 0.7:
                logits[b, par[b, j], tokens[b, j]] = 20.0
    suppress = (rng.rand(V) < 0.05).astype(np.uint8)
    suppress[tokens.ravel()] = 0
    if suppress.all():
        suppress[0] = 0
    return logits, tokens.astype(np.int32), par, suppress


def verify_check(logits, tokens, par, counts, suppress, got, V):
    pick, lp, path, taken, nxt = km.verify(logits.float().numpy(), tokens, par, counts, suppress)
    np.testing.assert_array_equal(got["pick"].cpu().numpy(), pick)
    np.testing.assert_array_equal(got["path"].cpu().numpy(), path)
    np.testing.assert_array_equal(got["n_accept"].cpu().numpy(), taken)
    np.testing.assert_array_equal(got["next"].cpu().numpy(), nxt)
    have = got["logprob"].cpu().numpy()
    np.testing.assert_array_equal(np.isfinite(have), np.isfinite(lp))
    ok = np.isfinite(lp)
    # every term e^x has the error of its argument's rounding (|x| u, x up to ~50 where it still counts) and of the hardware exp2 (2 u),
    # the sum at most one half step per partial sum on a path of V / 256 + 16 of them, and the logarithm 2 u of its value
    bound = (60 + V / 256 + 16) * 2.0 ** -24 + 4 * 2.0 ** -24 * np.abs(lp)
    assert (np.abs(have - lp)[ok] <= bound[ok]).all()


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("n,N,V", [(1, 1, 1), (1, 1, 7), (2, 5, 33), (3, 64, 1000), (1, 8, 51865), (5, 16, 5003), (40, 3, 777)])
def test_verify(dtype, n, N, V):
    rng = np.random.RandomState(V + N)
    logits, tokens, par, suppress = verify_case(rng, n, N, V, dtype)
    counts = rng.randint(0, N + 1, n)
    counts[0] = N
    got = verify_tree(logits.cuda(), i32(tokens), i32(par), counts=i32(counts), suppress=torch.from_numpy(suppress).cuda())
    verify_check(logits, tokens, par, counts, suppress, got, V)
    # rows that lie apart and do not start on 16 bytes; a chain; no mask
    wide = torch.full((n, N, V + 3), 99.0, dtype=dtype)
    wide[..., 1:V + 1] = logits
    chain = np.tile(np.arange(-1, N - 1, dtype=np.int32), (n, 1))
    got = verify_tree(wide.cuda()[..., 1:V + 1], i32(tokens))
    verify_check(logits, tokens, chain, np.full(n, N), np.zeros(V, np.uint8), got, V)


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("V", [40, 9001])
def test_verify_ties_and_values_that_are_no_numbers(dtype, V):
    nan, inf = float("nan"), float("inf")
    x = torch.zeros(1, 10, V, dtype=dtype)
    x[0, 0] = -5; x[0, 0, [30, 7, 39]] = 2                          # ties: the lowest id
    x[0, 1] = nan                                                   # nothing left
    x[0, 2] = -inf
    x[0, 3, ::2] = nan; x[0, 3, 11] = 1
    x[0, 4, [9, 12]] = inf                                          # two infinite logits share the probability
    x[0, 5] = -inf; x[0, 5, 33] = -1e30                             # one id, however low
    x[0, 6] = torch.finfo(dtype).min                                # all of the type's lowest value: equal
    x[0, 7, 5] = 3; x[0, 8, 5] = 3; x[0, 9] = inf
    sup = np.zeros(V, np.uint8)
    sup[5] = 1
    tokens = np.zeros((1, 10), np.int32)
    par = np.full((1, 10), -1, np.int32)
    got = verify_tree(x.cuda(), i32(tokens), i32(par), suppress=torch.from_numpy(sup).cuda())
    verify_check(x, tokens, par, np.array([10]), sup, got, V)
    every = np.ones(V, np.uint8)
    got = verify_tree(x.cuda(), i32(tokens), i32(par), suppress=torch.from_numpy(every).cuda())
    assert (got["pick"] == -1).all() and (got["logprob"] == -inf).all() and int(got["n_accept"]) == 1 and int(got["next"]) == -1


def test_verify_twins_and_odd_parents():
    """of siblings with one token the first is taken; a parent that is not before its node is never reached"""
    x = torch.zeros(1, 6, 50)
    x[0, 0, 3] = x[0, 1, 4] = x[0, 2, 4] = 5
    tokens = np.array([[9, 3, 3, 4, 4, 3]], np.int32)
    par = np.array([[-1, 0, 0, 2, 1, 5]], np.int32)
    got = verify_tree(x.cuda(), i32(tokens), i32(par))
    assert got["path"].tolist() == [[0, 1, 4, -1, -1, -1]] and got["n_accept"].tolist() == [3]
    with pytest.raises(ValueError):
        verify_tree(x.cuda(), i32(tokens)[:, :5], i32(par))
    with pytest.raises(ValueError):
        verify_tree(x.cuda().half(), i32(tokens), i32(par))
    with pytest.raises(ValueError):
        verify_tree(x.cuda(), i32(tokens), i32(par), suppress=torch.zeros(49, dtype=torch.uint8, device="cuda"))


# ---- together ---------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_a_drafted_step_equals_single_tokens(dtype):
    """fork, reserve, attend (appending), verify and commit as a drafted decode uses them: the cache then holds what one-token steps of the
    accepted tokens leave, and the next token attends it alike"""
    rng = np.random.RandomState(4)
    L, H, D, N, n, V = 2, 4, 64, 9, 3, 500
    emb = torch.tensor(rng.randn(V, 3, L, H, D), dtype=torch.float32).to(dtype).cuda()      # a token's q, k, v in every layer
    cache = PagedKVCache.allocate(L, H, D, 64, 12, 8, dtype=dtype)
    base = i32([0, 1, 2])
    lens = [20, 5, 33]
    cache.reserve(base, i32(lens))
    first = i32(rng.randint(0, V, (n, 33)))
    e = emb[first.long()]                                                                # [n, 33, 3, L, H, D]
    cache.append(base, e[:, :, 1].permute(2, 0, 1, 3, 4), e[:, :, 2].permute(2, 0, 1, 3, 4), counts=i32(lens))
    cache.commit(base, i32(np.tile(np.arange(33), (n, 1))), i32(lens))
    tree, single = i32([3, 4, 5]), i32([6, 7, 8])
    assert cache.fork(i32([3, 4, 5, 6, 7, 8]), i32([0, 1, 2, 0, 1, 2])).tolist() == [0] * 6
    par, tokens = trees(rng, n, N), rng.randint(0, V, (n, N)).astype(np.int32)
    logits = torch.randn(n, N, V, device="cuda")
    for b in range(n):
        for j in range(1, N):
            if par[b, j] >= 0 and rng.rand() < 0.8:
                logits[b, par[b, j], tokens[b, j]] = 30.0
    assert cache.reserve(tree, N).tolist() == [0] * 3
    e = emb[torch.tensor(tokens).long().cuda()]
    outs = [cache.attend(l, tree, e[:, :, 0, l], parents=i32(par), k=e[:, :, 1, l], v=e[:, :, 2, l], split_tokens=64) for l in range(L)]
    r = verify_tree(logits, i32(tokens), i32(par))
    assert cache.commit(tree, r["path"], r["n_accept"]).tolist() == [0] * 3
    path, taken = r["path"].cpu().numpy(), r["n_accept"].cpu().numpy()
    for step in range(int(taken.max())):
        live = [b for b in range(n) if step < taken[b]]
        ids = i32([6 + b for b in live])
        assert cache.reserve(ids, 1).tolist() == [0] * len(live)
        node = [int(path[b, step]) for b in live]
        e1 = emb[torch.tensor([[int(tokens[b, j])] for b, j in zip(live, node)]).cuda()]
        for l in range(L):
            o = cache.attend(l, ids, e1[:, :, 0, l], k=e1[:, :, 1, l], v=e1[:, :, 2, l], split_tokens=64)
            for at, (b, j) in enumerate(zip(live, node)):
                # the same keys, but grouped differently in the sums: the two roundings of each side (half a step of bf16 twice, or fp32 sums)
                tol = 2 ** -6 if dtype == BF16 else 1e-5
                torch.testing.assert_close(o[at, 0].float(), outs[l][b, j].float(), rtol=tol, atol=tol)
        cache.commit(ids, i32([[0]] * len(live)), i32([1] * len(live)))
    assert cache.lens[3:6].tolist() == cache.lens[6:9].tolist() == [l + int(t) for l, t in zip(lens, taken)]
    for b in range(n):
        total = int(cache.lens[3 + b])
        for pool in (cache.k, cache.v):
            rows = [torch.stack([pool[:, int(cache.table[s, t // 16]), :, t % 16] for t in range(total)]) for s in (3 + b, 6 + b)]
            assert torch.equal(rows[0], rows[1])
    q = torch.randn(n, 1, H, D, device="cuda").to(dtype)
    assert torch.equal(cache.attend(0, tree, q, counts=i32([0] * n)), torch.zeros_like(q))
    kv = torch.randn(n, 1, H, D, device="cuda").to(dtype)
    cache.reserve(i32([3, 4, 5, 6, 7, 8]), 1)
    assert torch.equal(cache.attend(0, tree, q, k=kv, v=kv, split_tokens=64), cache.attend(0, single, q, k=kv, v=kv, split_tokens=64))
