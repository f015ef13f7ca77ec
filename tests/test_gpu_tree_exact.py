"""Tree attention of bf16 caches held to what the rounding of its result alone allows: probabilities keep their bits, and no key is lost
wherever it stands."""
import numpy as np
import pytest
import torch

import kv_model as km
from test_gpu_tree import BF16, Case, i32, trees
from whisper_amd.kvcache import PagedKVCache

pytestmark = pytest.mark.gpu


def tight_bound(o, mass, reach, D, tokens):
    """kv_model.attention_bound for 32 bits (scores, exponentials and sums; a probability enters as two bf16 terms, so there are twice as many
    additions), 2^-14 of every probability for what two bf16 terms leave out (half a step, 2^-8, of a second term of at most 2^-7 + 2^-8 of it), and
    half a step, 2^-8, of the result."""
    u = 2.0 ** -24
    rel = 2 * (D + 4) * u * reach + (4 * tokens + 64) * u + 2.0 ** -14
    return rel * mass * (1 + 2.0 ** -7) + 2.0 ** -8 * np.abs(o) + 1e-30


def check(c, out, scale=None):
    scale = c.D ** -0.5 if scale is None else scale
    out = out.float().cpu().numpy().astype(np.float64)
    for i in range(c.n):
        K, V = torch.cat([c.pre[i][0], c.kn[i]]).float().numpy(), torch.cat([c.pre[i][1], c.vn[i]]).float().numpy()
        o, mass, reach = km.tree_attention(c.q[i].float().numpy(), K, V, c.par[i], scale)
        off, bound = np.abs(out[i] - o), tight_bound(o, mass, reach, c.D, len(K))
        assert (off <= bound).all(), (i, float((off / bound).max()), int((off > bound).sum()))


# every kernel for bf16 caches: the waves share the keys (16 or 32 rows; a whole sequence or pieces), a wave alone, the waves share the rows
@pytest.mark.parametrize("lens,N,heads,kv_heads,D,PS", [
    ([30, 100], 5, 4, 2, 64, 16), ([90, 200], 24, 3, 3, 64, 16), ([64, 9], 6, 4, 2, 128, 16), ([700, 20], 5, 4, 2, 64, 16), ([700, 90], 24, 3, 3, 64, 16),
    ([600, 31], 6, 4, 2, 128, 32), (list(range(0, 130)), 1, 8, 8, 64, 16), (list(range(3, 100)), 2, 16, 8, 128, 16), (list(range(1, 65)), 20, 12, 12, 64, 16),
    ([50, 129], 40, 2, 2, 128, 16), ([65, 200], 40, 8, 2, 128, 32), ([900], 20, 4, 4, 128, 32), ([1000, 30], 64, 8, 2, 128, 64), ([40], 64, 16, 4, 64, 16), ([800, 3], 64, 6, 2, 64, 16)])
def test_probabilities_keep_their_bits(lens, N, heads, kv_heads, D, PS):
    c = Case(lens, N, heads, kv_heads, D, PS, BF16, seed=len(lens) + N)
    c.q *= 3                                                       # the weight on few tokens, whose roundings do not average out
    check(c, c.run())


FORMS = [([30, 100], 5, 4, 2, 64, 16), ([90, 200], 24, 3, 3, 64, 16), ([64, 9], 6, 4, 2, 128, 16), ([700, 200], 5, 4, 2, 64, 16), ([700, 90], 24, 3, 3, 64, 16),
         (list(range(20, 150)), 1, 8, 8, 64, 16), (list(range(20, 100)), 20, 12, 12, 64, 16), ([50, 129], 40, 2, 2, 128, 16), ([1000, 300], 64, 8, 2, 128, 64),
         ([800, 30], 64, 6, 2, 64, 16)]


@pytest.mark.parametrize("lens,N,heads,kv_heads,D,PS", FORMS)
def test_infinite_values_of_committed_tokens(lens, N, heads, kv_heads, D, PS):
    """every row attends them, so its column is infinite, with their sign; NaN where both signs meet, and nothing else changes"""
    c = Case(lens, N, heads, kv_heads, D, PS, BF16, seed=1)
    c.q *= 0.25                                                    # no probability is 0
    clean = c.run().float().cpu()
    for s in range(c.n):
        for token, col, what in ((0, 3, float("inf")), (int(c.lens[s]) - 1, 17, -float("inf")), (int(c.lens[s]) // 2, 40, float("inf")), (1, 40, -float("inf"))):
            page = int(c.cache.table[int(c.slots[s]), token // PS])
            c.cache.v[c.layer, page, :, token % PS, col] = what
    out = c.run().float().cpu()
    assert (out[..., 3] == float("inf")).all() and (out[..., 17] == -float("inf")).all() and torch.isnan(out[..., 40]).all()
    rest = [x for x in range(D) if x not in (3, 17, 40)]
    assert torch.equal(out[..., rest], clean[..., rest])


@pytest.mark.parametrize("lens,N,heads,kv_heads,D,PS", [
    ([0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65], 24, 6, 2, 64, 16), ([447, 448, 129, 127], 64, 8, 1, 64, 16), ([511, 513, 640, 1000], 24, 16, 1, 64, 16),
    ([128, 127, 129, 400], 12, 16, 2, 128, 32), ([575, 576, 577], 12, 16, 1, 128, 16), ([0, 1, 63, 64, 65, 127, 200], 17, 32, 2, 128, 16),
    ([512, 511, 640, 2000], 64, 16, 1, 128, 64), ([700, 1023, 1025], 64, 15, 1, 64, 128), (list(range(100)), 3, 32, 8, 64, 16)])
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("split", [0, 64, 200])
def test_no_key_is_lost(dtype, lens, N, heads, kv_heads, D, PS, split):
    """every row points at one token, its own among those it attends, so that almost all of its weight is there: first, last and every other one of
    the committed tokens (ends of tiles, pages, pieces and shares) in turn, and the node itself"""
    c = Case(lens, N, heads, kv_heads, D, PS, dtype, seed=3)
    G = heads // kv_heads
    for s in range(c.n):
        length = int(c.lens[s])
        for node in range(N):
            for h in range(heads):
                at = (node * G + h % G) * max(1, -(-length // (N * G))) if length else 0
                at = length - 1 - at if (node + h) % 2 else at     # from both ends
                key = c.kn[s, node, h // G] if at < 0 or at >= length or (node + 3 * h) % 11 == 0 else c.pre[s][0][at, h // G]
                c.q[s, node, h] = (4 * key.float()).to(dtype)
    if dtype == torch.float32:
        c.check(c.run(split_tokens=split))
    else:
        check(c, c.run(split_tokens=split))


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("lens,N,heads,kv_heads,D,PS", FORMS + [([1500, 700, 900], 24, 3, 3, 64, 16), ([3000, 1100], 6, 4, 2, 128, 16)])
@pytest.mark.parametrize("split", [0, 128])
def test_every_row_of_a_refused_entry_is_nan(dtype, lens, N, heads, kv_heads, D, PS, split):
    """in whole sequences and in pieces, nodes that are not there included; all other entries stay as they are"""
    n = len(lens)
    c = Case(lens, N, heads, kv_heads, D, PS, dtype, seed=5, counts=[max(1, N - 2)] * n)
    c.append = False
    kn, vn = c.kn.cuda(), c.vn.cuda()
    run = lambda slots, **kw: c.cache.attend(c.layer, i32(slots), c.q.cuda(), parents=i32(c.par), counts=i32(c.counts), split_tokens=split, **kw)  # noqa: E731
    c.cache.append(i32(c.slots), c.kn.cuda(), c.vn.cuda(), counts=i32(c.counts), layer=c.layer)
    good = run(c.slots)
    assert torch.isfinite(good).all() and not good[:, max(1, N - 2):].any()

    def alike(out, rest, slots):
        if split or np.array_equal(slots, c.slots):
            assert torch.equal(out[rest], good[rest])
        else:                                                      # another batch is cut elsewhere: each side's rounding (bf16: half a step each) and its sums in 32 bits
            torch.testing.assert_close(out[rest], good[rest], rtol=2.0 ** -7 if dtype == BF16 else 0, atol=1e-3)

    def refused(at, slots=c.slots, **kw):
        out = run(slots, **kw)
        assert torch.isnan(out[at]).all(), (at, int(torch.isnan(out[at]).sum()), out[at].numel())
        alike(out, [i for i in range(n) if i != at], slots)
    table, held, refs = c.cache.table, c.cache.held, c.cache.refs
    for at in (0, n - 1):
        s = int(c.slots[at])
        other = c.slots.copy()
        for bad in (n + 1, -2, 10 ** 6):
            other[at] = bad
            refused(at, other)
        was = int(held[s])
        held[s] = max(0, -(-(int(c.lens[at]) + max(1, N - 2)) // PS) - 1)
        refused(at)
        held[s] = was
        for page in (0, int(c.lens[at]) // PS):                    # the first piece's, the last's
            was = int(table[s, page])
            for bad in (-1, 10 ** 8):
                table[s, page] = bad
                refused(at)
            table[s, page] = was
        page = int(table[s, int(c.lens[at]) // PS])
        refs[page] = 2
        refused(at, k=kn, v=vn)
        refs[page] = 1
    if n > 1:
        twice = c.slots.copy()
        twice[n - 1] = twice[0]
        refused(n - 1, twice, k=kn, v=vn)
    pad = c.slots.copy()
    pad[0] = -1
    out = run(pad)
    assert not out[0].any()
    alike(out, range(1, n), pad)


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("G,kv_heads,D", [(1, 2, 64), (3, 2, 64), (8, 1, 64), (16, 1, 64), (1, 2, 128), (2, 4, 128), (4, 2, 128), (16, 1, 128)])
@pytest.mark.parametrize("longest,split", [(100, 64), (3000, 64), (3000, 300), (3000, 1 << 20), (20000, 64)])
def test_a_fixed_cut_does_not_see_the_width_of_the_batch(dtype, G, kv_heads, D, longest, split):
    """a sequence of three nodes, alone and among sequences that pad the batch to more nodes: the same bits"""
    n, W, PS = 3, 64, 64
    H, g = G * kv_heads, torch.Generator().manual_seed(G)
    lens = [longest, longest // 3, 7]
    pages = [-(-(x + W) // PS) for x in lens]
    c = PagedKVCache.allocate(1, kv_heads, D, sum(pages), n, max(pages), page_size=PS, dtype=dtype)
    c.k.copy_(torch.randn(c.k.shape, generator=g).to(dtype)); c.v.copy_(torch.randn(c.v.shape, generator=g).to(dtype))
    c.lens.copy_(i32([0] * n))
    assert not c.reserve(i32(range(n)), i32([x + W for x in lens])).any()
    c.lens.copy_(i32(lens))
    q = torch.randn(n, W, H, D, generator=g).to(dtype).cuda()
    par = i32(trees(np.random.RandomState(1), n, W))
    want = None
    for width in (3, 4, 5, 8, 9, 16, 17, 32, 33, 43, 64):
        counts = i32([3, width, max(1, width - 2)])
        out = c.attend(0, i32([0, 1, 2]), q[:, :width].contiguous(), parents=par[:, :width].contiguous(), counts=counts, split_tokens=split)[0, :3]
        want = out if want is None else want
        assert torch.equal(out, want), (width, float((out - want).abs().max()))
    for width in (3, 17, 64):
        alone = c.attend(0, i32([0]), q[:1, :width].contiguous(), parents=par[:1, :width].contiguous(), counts=i32([3]), split_tokens=split)[0, :3]
        assert torch.equal(alone, want)
