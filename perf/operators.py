"""The operators of drafted (speculative) decoding over a paged key/value cache, as a user of whisper_amd meets them, and their plain forms.

attend   tree attention: the drafted nodes of every sequence attend the sequence's cached prefix and their own ancestors; the nodes' keys
         and values are appended behind the prefix (``append``) or lie there already.  One node a sequence is the single-token form.
verify   the arg-max of every drafted node's logits, its log-probability, and the longest drafted path that agrees with it.
fork     pages: the children of the last step are freed, forked anew from their parents (pages shared), and given room for the next
         tokens, which copies the shared, partly filled last page of each child.
commit   pages: roll back to the committed length, make room for a draft, append its rows in every layer, and move the accepted path's
         rows together behind the prefix.
compact  pages: the live pages of a fragmented pool move to its lowest places.

The page-structure of a case (lengths, trees, accepted paths) follows from the case, the values and the page numbers from the seed.
"""
import math
import zlib

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
DEVICE = "cuda"


def listed():
    return [
        # one window of the smallest model with a short draft: launch latency
        dict(name="attend_tiny_f32", kind="attend", type="f32", seqs=1, nodes=5, heads=6, kv_heads=6, dim=64, page=16, shortest=60, longest=60, append=True),
        # 16 windows of large-v3, draft trees of up to 24 nodes, anywhere in the 448-position context
        dict(name="attend_large_tree24", kind="attend", type="bf16", seqs=16, nodes=24, heads=20, kv_heads=20, dim=64, page=16, shortest=30, longest=420, append=True),
        # 64 windows of large-v3, one token each: the plain decode step
        dict(name="attend_64_single", kind="attend", type="bf16", seqs=64, nodes=1, heads=20, kv_heads=20, dim=64, page=16, shortest=200, longest=447, append=True),
        # long contexts, shared key/value heads, full trees whose rows are in the cache already
        dict(name="attend_long_shared_heads", kind="attend", type="bf16", seqs=8, nodes=64, heads=32, kv_heads=8, dim=128, page=64, shortest=40000, longest=131072, append=False),
        # one window, a short draft over the multilingual vocabulary
        dict(name="verify_one", kind="verify", type="f32", seqs=1, nodes=8, vocab=51865),
        # 64 windows, 16 nodes each, the large-v3 vocabulary
        dict(name="verify_64", kind="verify", type="f32", seqs=64, nodes=16, vocab=51866),
        # 3 windows of the smallest model in 5 branches each
        dict(name="fork_tiny", kind="fork", type="f32", layers=4, kv_heads=6, dim=64, page=16, parents=3, width=5, longest=200, extra=1),
        # 12 windows of large-v3 in 5 branches each
        dict(name="fork_large", kind="fork", type="bf16", layers=32, kv_heads=20, dim=64, page=16, parents=12, width=5, longest=440, extra=1),
        # 16 windows of large-v3-turbo (4 decoder layers), drafts of 24 nodes
        dict(name="commit_turbo", kind="commit", type="bf16", layers=4, kv_heads=20, dim=64, page=16, seqs=16, nodes=24, longest=420),
        # 64 windows of large-v3, drafts of 16 nodes
        dict(name="commit_large", kind="commit", type="bf16", layers=32, kv_heads=20, dim=64, page=16, seqs=64, nodes=16, longest=420),
        # a pool of the smallest model in use to two fifths
        dict(name="compact_tiny", kind="compact", type="f32", layers=4, kv_heads=6, dim=64, page=16, pages=256, seqs=9, longest=200),
        # a pool of large-v3 in use to a half
        dict(name="compact_large", kind="compact", type="bf16", layers=32, kv_heads=20, dim=64, page=16, pages=1024, seqs=36, longest=440),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "verify", "verify", "fork", "commit", "compact"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "verify":
        seqs, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        return dict(kind=kind, type=dtype, seqs=seqs, nodes=min(nodes, max(1, 2048 // seqs)), vocab=_log_int(rng, 1000, 140000))
    kv_heads, dim, page = rng.choice([1, 2, 4, 6, 8, 12, 16, 20]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    if kind == "attend":
        heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv_heads <= 64])
        seqs, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        longest = _log_int(rng, 1, 65536)
        longest = max(1, min(longest, (1 << 28) // (seqs * kv_heads * dim), (1 << 29) // (seqs * heads * nodes)))
        return dict(kind=kind, type=dtype, seqs=seqs, nodes=nodes, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    shortest=rng.randrange(longest + 1), longest=longest, append=rng.random() < 0.7)
    layers, longest = _log_int(rng, 1, 32), _log_int(rng, 20, 2000)
    row = layers * kv_heads * dim
    if kind == "fork":
        parents, width = _log_int(rng, 1, 24), rng.randrange(1, 9)
        longest = max(1, min(longest, (1 << 28) // (row * parents)))
        return dict(kind=kind, type=dtype, layers=layers, kv_heads=kv_heads, dim=dim, page=page, parents=parents, width=width, longest=longest,
                    extra=_log_int(rng, 1, 40))
    if kind == "commit":
        seqs, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        longest = max(1, min(longest, (1 << 28) // (row * seqs)))
        return dict(kind=kind, type=dtype, layers=layers, kv_heads=kv_heads, dim=dim, page=page, seqs=seqs, nodes=nodes, longest=longest)
    pages = max(4, min(_log_int(rng, 32, 2000), (1 << 28) // (row * page)))
    return dict(kind=kind, type=dtype, layers=layers, kv_heads=kv_heads, dim=dim, page=page, pages=pages, seqs=_log_int(rng, 2, 64), longest=max(page, min(longest, pages * page // 2)))


# ---- the structure of a case ---------------------------------------------------------------------------------------------------

def _case_rng(case):
    return np.random.RandomState(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))


def _lengths(r, n, lo, hi):
    out = r.randint(lo, hi + 1, n)
    out[r.randint(n)] = hi
    return out.astype(np.int32)


def _trees(r, n, nodes):
    """parents [n][nodes] (node 0 is the root, every other node's parent stands before it, most often close), counts [n]"""
    par = np.full((n, nodes), -1, np.int32)
    for j in range(1, nodes):
        par[:, j] = r.randint(np.maximum(0, j - 1 - r.randint(0, 6, n)), j)
    counts = r.randint(max(1, nodes // 2), nodes + 1, n).astype(np.int32)
    counts[r.randint(n)] = nodes
    return par, counts


def _paths(r, par, counts):
    """one root-to-node path of every tree, as an accepted draft leaves it: path [n][nodes] padded with -1, its length [n]"""
    n, nodes = par.shape
    path, taken = np.full((n, nodes), -1, np.int32), np.zeros(n, np.int32)
    for s in range(n):
        j, chain = int(r.randint(counts[s])), []
        while j >= 0:
            chain.append(j)
            j = int(par[s, j])
        path[s, :len(chain)] = chain[::-1]
        taken[s] = len(chain)
    return path, taken


def _structure(case):
    r, kind = _case_rng(case), case["kind"]
    if kind == "attend":
        lens = _lengths(r, case["seqs"], case["shortest"], case["longest"])
        par, counts = _trees(r, case["seqs"], case["nodes"])
        return dict(lens=lens, par=par, counts=counts)
    if kind == "verify":
        par, counts = _trees(r, case["seqs"], case["nodes"])
        return dict(par=par, counts=counts)
    if kind == "fork":
        return dict(lens=_lengths(r, case["parents"], max(1, case["longest"] // 3), case["longest"]))
    if kind == "commit":
        lens = _lengths(r, case["seqs"], case["longest"] // 4, case["longest"])
        par, counts = _trees(r, case["seqs"], case["nodes"])
        path, taken = _paths(r, par, counts)
        return dict(lens=lens, par=par, counts=counts, path=path, taken=taken)
    # compact: as many sequences as fit half the pool, on pages picked anywhere in it
    lens = _lengths(r, case["seqs"], 1, case["longest"])
    need = -(-lens // case["page"])
    lens[np.cumsum(need) > max(1, case["pages"] // 2)] = 0
    return dict(lens=lens, order=r.permutation(case["pages"]).astype(np.int32))


def _pool(case, lens, max_pages, n_pages, order, layers, g):
    """pools with values in every row, tables over the page numbers of `order`, counts of users, lengths and held pages"""
    n, page = len(lens), case["page"]
    need = -(-lens // page)
    table, at = np.full((n, max_pages), -1, np.int32), 0
    for s in range(n):
        table[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
    refs = np.zeros(n_pages, np.int32)
    refs[order[:at]] = 1
    shape = (layers, n_pages, case["kv_heads"], page, case["dim"])
    dtype = DTYPES[case["type"]]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE)  # noqa: E731
    return dict(k=torch.randn(shape, generator=g, device=DEVICE, dtype=dtype), v=torch.randn(shape, generator=g, device=DEVICE, dtype=dtype),
                table=dev(table), refs=dev(refs), lens=dev(lens.astype(np.int32)), held=dev(need.astype(np.int32)))


def _make(case, seed):
    c, r = case, np.random.RandomState(seed % (1 << 32))
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    st, kind = _structure(case), case["kind"]
    dtype = DTYPES[c["type"]]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE)  # noqa: E731
    s = dict(kind=kind)
    if kind == "verify":
        n, N, V = c["seqs"], c["nodes"], c["vocab"]
        tokens = r.randint(0, V, (n, N)).astype(np.int32)
        # rows as the vocabulary projection leaves them: padded to a multiple of 16
        logits = torch.randn((n, N, -(-V // 16) * 16), generator=g, device=DEVICE) * 3.0
        hit = (r.rand(n, N) < 0.6) & (st["par"] >= 0)
        at, node = np.nonzero(hit)
        suppress = np.zeros(V, np.uint8)
        suppress[r.randint(0, V, min(90, V // 4))] = 1
        suppress[tokens.reshape(-1)] = 0
        logits[dev(at), dev(st["par"][at, node].astype(np.int64)), dev(tokens[at, node].astype(np.int64))] = 24.0
        s.update(logits=logits.to(dtype)[..., :V], tokens=dev(tokens), parents=dev(st["par"]), counts=dev(st["counts"]), suppress=dev(suppress))
        return s
    page, need = c["page"], -(-st["lens"] // c["page"])
    if kind == "attend":
        lens, N = st["lens"], c["nodes"]
        room = -(-(lens + N) // page)                     # the nodes' rows have their pages
        n_pages = int(room.sum()) + 1 + int(room.sum()) // 32
        s.update(_pool(c, room * page, int(room.max()), n_pages, r.permutation(n_pages).astype(np.int32), 1, g))
        s["lens"] = dev(lens)
        rnd = lambda h: torch.randn((c["seqs"], N, h, c["dim"]), generator=g, device=DEVICE, dtype=dtype)  # noqa: E731
        s.update(seqs=torch.arange(c["seqs"], device=DEVICE, dtype=torch.int32), q=rnd(c["heads"]), parents=dev(st["par"]), counts=dev(st["counts"]),
                 kn=rnd(c["kv_heads"]) if c["append"] else None, vn=rnd(c["kv_heads"]) if c["append"] else None, scale=c["dim"] ** -0.5)
    elif kind == "fork":
        W, kids = c["parents"], c["parents"] * c["width"]
        lens = np.concatenate([st["lens"], np.zeros(kids, np.int32)])
        most = -(-(c["longest"] + c["extra"]) // page)
        n_pages = int(need.sum()) + kids * (1 + -(-c["extra"] // page)) + 5
        s.update(_pool(c, lens, most, n_pages, r.permutation(n_pages).astype(np.int32), c["layers"], g))
        s.update(dst=dev(np.arange(W, W + kids, dtype=np.int32)), src=dev(np.repeat(np.arange(W, dtype=np.int32), c["width"])), extra=c["extra"])
    elif kind == "commit":
        lens, N = st["lens"], c["nodes"]
        most = -(-(c["longest"] + N) // page)
        n_pages = int((-(-(lens + N) // page)).sum()) + 3
        s.update(_pool(c, lens, most, n_pages, r.permutation(n_pages).astype(np.int32), c["layers"], g))
        rnd = lambda: torch.randn((c["layers"], c["seqs"], N, c["kv_heads"], c["dim"]), generator=g, device=DEVICE, dtype=dtype)  # noqa: E731
        s.update(seqs=torch.arange(c["seqs"], device=DEVICE, dtype=torch.int32), base=dev(lens), nodes=N, kn=rnd(), vn=rnd(), counts=dev(st["counts"]),
                 path=dev(st["path"]), taken=dev(st["taken"]))
    else:
        most = -(-c["longest"] // page)
        s.update(_pool(c, st["lens"], most, c["pages"], st["order"], c["layers"], g))
        s.update(was={n: s[n].clone() for n in ("table", "refs")})
    return s


def prepare(case, seed):
    s = _make(case, seed)
    if own and s["kind"] != "verify":
        from whisper_amd.kvcache import PagedKVCache
        s["cache"] = PagedKVCache(s["k"], s["v"], s["table"], s["refs"], s["lens"], s["held"])
    return s


def run(s):
    return (_own if own else _plain)[s["kind"]](s)


# ---- the framework's calls ---------------------------------------------------------------------------------------------------------

def _state(s, *names):
    return {n: s[n] for n in names}


def _own_attend(s):
    out = s["cache"].attend(0, s["seqs"], s["q"], s["parents"], k=s["kn"], v=s["vn"], counts=s["counts"], scale=s["scale"])
    return dict(out=out, **(_state(s, "k", "v") if s["kn"] is not None else {}))


def _own_verify(s):
    from whisper_amd.draft import verify_tree
    return verify_tree(s["logits"], s["tokens"], s["parents"], counts=s["counts"], suppress=s["suppress"])


def _own_fork(s):
    cache = s["cache"]
    cache.truncate(s["dst"])
    cache.fork(s["dst"], s["src"])
    status = cache.reserve(s["dst"], s["extra"])
    return dict(status=status, **_state(s, "k", "v", "table", "refs", "lens", "held"))


def _own_commit(s):
    cache = s["cache"]
    cache.truncate(s["seqs"], s["base"])
    cache.reserve(s["seqs"], s["nodes"])
    cache.append(s["seqs"], s["kn"], s["vn"], counts=s["counts"])
    status = cache.commit(s["seqs"], s["path"], s["taken"])
    return dict(status=status, **_state(s, "k", "v", "table", "refs", "lens", "held"))


def _own_compact(s):
    s["table"].copy_(s["was"]["table"])
    s["refs"].copy_(s["was"]["refs"])
    live = s["cache"].compact()
    return dict(live=live, **_state(s, "k", "v", "table", "refs", "lens", "held"))


_own = dict(attend=_own_attend, verify=_own_verify, fork=_own_fork, commit=_own_commit, compact=_own_compact)


# ---- the plain forms -------------------------------------------------------------------------------------------------------------

def _ancestors(parents):
    """[n, N, N]: whether node j is node i or one of its ancestors (powers of the parent relation)"""
    n, N = parents.shape
    step = (parents[..., None] == torch.arange(N, device=parents.device)).float() + torch.eye(N, device=parents.device)
    return torch.linalg.matrix_power(step, N) > 0


def _rows(s, seqs, N):
    """page and slot of the rows at lens + 0 .. N-1 of every listed sequence"""
    page = s["k"].shape[3]
    pos = s["lens"][seqs.long()].long()[:, None] + torch.arange(N, device=seqs.device)
    pages = s["table"][seqs.long()].long().gather(1, (pos // page).clamp(max=s["table"].shape[1] - 1))
    return pages.clamp(min=0), pos % page


def _put(pool, pages, slots, rows, active):
    """pool [L][P][H][page][D]: rows [L][n][N][H][D] to their places, where active"""
    was = pool[:, pages, :, slots]                               # [n, N, L, H, D]
    pool[:, pages, :, slots] = torch.where(active[..., None, None, None], rows.permute(1, 2, 0, 3, 4), was)


def _plain_attend(s):
    q, seqs, N = s["q"].float(), s["seqs"], s["q"].shape[1]
    n, _, heads, D = q.shape
    H, page = s["k"].shape[2], s["k"].shape[3]
    active = torch.arange(N, device=q.device) < s["counts"][:, None]
    if s["kn"] is not None:
        pages, slots = _rows(s, seqs, N)
        _put(s["k"], pages, slots, s["kn"][None], active)
        _put(s["v"], pages, slots, s["vn"][None], active)
    table = s["table"][seqs.long()].long()
    T = table.shape[1] * page
    keys = s["k"][0][table.clamp(min=0)].permute(0, 2, 1, 3, 4).reshape(n, H, T, D).float()
    vals = s["v"][0][table.clamp(min=0)].permute(0, 2, 1, 3, 4).reshape(n, H, T, D).float()
    lens = s["lens"][seqs.long()].long()
    node = torch.arange(T, device=q.device) - lens[:, None]      # < 0: the prefix; 0 ..: the drafted node's own row
    seen = _ancestors(s["parents"])
    seen = seen.gather(2, node.clamp(0, N - 1)[:, None].expand(n, N, T)) & (node >= 0)[:, None] & (node < N)[:, None] | (node < 0)[:, None]
    seen = seen & active[..., None]
    qg = q.reshape(n, N, H, heads // H, D).permute(0, 2, 3, 1, 4).reshape(n, H, -1, D)
    score = (qg @ keys.transpose(2, 3)).reshape(n, H, heads // H, N, T) * s["scale"]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    out = (p.reshape(n, H, -1, T) @ vals).reshape(n, H, heads // H, N, D) / total.clamp(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, N, heads, D).to(s["q"].dtype)
    return dict(out=out, **(_state(s, "k", "v") if s["kn"] is not None else {}))


def _plain_verify(s):
    x, tokens, parents = s["logits"].float(), s["tokens"], s["parents"].long()
    n, N, V = x.shape
    at = torch.arange(N, device=x.device)
    active = at < s["counts"][:, None]
    x = x.masked_fill(s["suppress"].bool(), -math.inf)
    top = x.amax(-1, keepdim=True)
    pick = torch.where(x == top, torch.arange(V, device=x.device), V).amin(-1)
    logprob = -(x - top).exp().sum(-1).log()
    # a node is reached where its token is its parent's pick; of siblings with one token the first counts
    agrees = (pick.gather(1, parents.clamp(min=0)) == tokens) & (parents >= 0)
    twin = (parents[:, :, None] == parents[:, None, :]) & (tokens[:, :, None] == tokens[:, None, :]) & (at[None, :] < at[:, None])
    good = active & ((agrees & ~twin.any(-1)) | (at == 0))
    reached = ~(_ancestors(s["parents"]) & ~good[:, None, :]).any(-1)
    path = torch.where(reached, at, N).sort(-1).values
    taken = reached.sum(-1)
    last = path.gather(1, (taken - 1).clamp(min=0)[:, None]).clamp(max=N - 1)
    follow = pick.gather(1, last)[:, 0]
    return dict(pick=torch.where(active, pick, -1).int(), logprob=torch.where(active, logprob, 0.0), path=torch.where(path < N, path, -1).int(), n_accept=taken.int(),
                next=torch.where(taken > 0, follow, -1).int())


def _truncate(s, seqs, lens):
    i, page = seqs.long(), s["k"].shape[3]
    new = torch.zeros_like(s["lens"][i]) if lens is None else lens
    keep = (new + page - 1) // page
    rows = s["table"][i]
    drop = (rows >= 0) & (torch.arange(rows.shape[1], device=rows.device) >= keep[:, None])
    s["refs"].scatter_add_(0, rows.clamp(min=0).long().reshape(-1), -drop.int().reshape(-1))
    s["table"][i] = torch.where(drop, -1, rows)
    s["held"][i] = torch.minimum(s["held"][i], keep)
    s["lens"][i] = new


def _fork(s, dst, src):
    page = s["k"].shape[3]
    lens = s["lens"][src.long()]
    keep = (lens + page - 1) // page
    rows = s["table"][src.long()]
    rows = torch.where(torch.arange(rows.shape[1], device=rows.device) < keep[:, None], rows, -1)
    s["refs"].scatter_add_(0, rows.clamp(min=0).long().reshape(-1), (rows >= 0).int().reshape(-1))
    s["table"][dst.long()], s["lens"][dst.long()], s["held"][dst.long()] = rows, lens, keep


def _reserve(s, seqs, extra):
    """room for `extra` more rows in private pages: the lowest free pages, in the order of the list; a shared last page is copied"""
    i, page = seqs.long(), s["k"].shape[3]
    lens, held, rows, refs = s["lens"][i], s["held"][i], s["table"][i], s["refs"]
    want = (lens + extra + page - 1) // page
    tail, fill = lens // page, lens % page
    old = rows.gather(1, tail.clamp(max=rows.shape[1] - 1).long()[:, None])[:, 0]
    copies = (fill > 0) & (refs[old.clamp(min=0).long()] > 1)
    need = copies.int() + (want - held).clamp(min=0)
    after = need.cumsum(0)
    served = (need == 0) | (after <= (refs == 0).sum())
    free = torch.argsort((refs > 0).int(), stable=True)
    first = after - need
    col = torch.arange(rows.shape[1], device=rows.device)
    rank = torch.where((col == tail[:, None]) & copies[:, None], first[:, None], first[:, None] + copies[:, None].int() + col - held[:, None])
    fresh = (((col == tail[:, None]) & copies[:, None]) | ((col >= held[:, None]) & (col < want[:, None]))) & served[:, None]
    page_of = free[rank.clamp(0, refs.shape[0] - 1).long()]
    s["table"][i] = torch.where(fresh, page_of.int(), rows)
    s["held"][i] = torch.where(served, torch.maximum(held, want), held)
    refs.scatter_add_(0, page_of.reshape(-1), fresh.int().reshape(-1))
    moved = copies & served
    refs.scatter_add_(0, old.clamp(min=0).long(), -moved.int())
    a, b = old[moved].long(), free[first[moved].long()]
    filled = (torch.arange(page, device=rows.device) < fill[moved][:, None])[None, :, None, :, None]
    s["k"][:, b] = torch.where(filled, s["k"][:, a], s["k"][:, b])
    s["v"][:, b] = torch.where(filled, s["v"][:, a], s["v"][:, b])
    return torch.where(served, 0, -3).int()


def _plain_fork(s):
    _truncate(s, s["dst"], None)
    _fork(s, s["dst"], s["src"])
    status = _reserve(s, s["dst"], s["extra"])
    return dict(status=status, **_state(s, "k", "v", "table", "refs", "lens", "held"))


def _plain_commit(s):
    _truncate(s, s["seqs"], s["base"])
    _reserve(s, s["seqs"], s["nodes"])
    pages, slots = _rows(s, s["seqs"], s["nodes"])
    at = torch.arange(s["nodes"], device=pages.device)
    active = at < s["counts"][:, None]
    _put(s["k"], pages, slots, s["kn"], active)
    _put(s["v"], pages, slots, s["vn"], active)
    taken = at < s["taken"][:, None]
    path = s["path"].clamp(min=0).long()
    fp, fs = pages.gather(1, path), slots.gather(1, path)
    _put(s["k"], pages, slots, s["k"][:, fp, :, fs].permute(2, 0, 1, 3, 4), taken)
    _put(s["v"], pages, slots, s["v"][:, fp, :, fs].permute(2, 0, 1, 3, 4), taken)
    s["lens"][s["seqs"].long()] += s["taken"]
    return dict(status=torch.zeros_like(s["taken"]), **_state(s, "k", "v", "table", "refs", "lens", "held"))


def _plain_compact(s):
    s["table"].copy_(s["was"]["table"])
    s["refs"].copy_(s["was"]["refs"])
    live = s["refs"] > 0
    n = live.sum()
    at = torch.arange(live.shape[0], device=live.device)
    moves, holes = live & (at >= n), ~live & (at < n)
    src, dst = at[moves], at[holes]                                # the i-th page to move goes to the i-th hole
    to = at.clone()
    to[src] = dst
    s["k"][:, dst], s["v"][:, dst] = s["k"][:, src], s["v"][:, src]
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    s["table"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].int(), -1))
    return dict(live=n.int().reshape(1), **_state(s, "k", "v", "table", "refs", "lens", "held"))


_plain = dict(attend=_plain_attend, verify=_plain_verify, fork=_plain_fork, commit=_plain_commit, compact=_plain_compact)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------

def work(case):
    c, st, kind = case, _structure(case), case["kind"]
    es = 4 if c["type"] == "f32" else 2
    if kind == "verify":
        rows = int(st["counts"].sum())
        return dict(bytes=rows * c["vocab"] * es + c["vocab"] + c["seqs"] * c["nodes"] * 20, flops=3 * rows * c["vocab"])
    row = 2 * c["kv_heads"] * c["dim"] * es                       # keys and values of one token in one layer
    if kind == "attend":
        lens, counts = st["lens"].astype(np.int64), st["counts"].astype(np.int64)
        depth = np.zeros_like(st["par"], dtype=np.int64)
        for j in range(c["nodes"]):
            depth[:, j] = np.where(st["par"][:, j] >= 0, depth[np.arange(len(lens)), np.maximum(st["par"][:, j], 0)], 0) + 1
        pairs = int((lens * counts).sum() + (depth * (np.arange(c["nodes"]) < counts[:, None])).sum())
        seen = int(((lens + counts) * (counts > 0)).sum())
        moved = seen * row + (int(counts.sum()) * row if c["append"] else 0)
        return dict(bytes=moved + (int(counts.sum()) + c["seqs"] * c["nodes"]) * c["heads"] * c["dim"] * es, flops=4 * c["heads"] * c["dim"] * pairs)
    if kind == "fork":
        fill = st["lens"].astype(np.int64) % c["page"]
        held = -(-st["lens"].astype(np.int64) // c["page"])
        return dict(bytes=int(fill.sum()) * c["width"] * row * c["layers"] * 2 + int(held.sum()) * (1 + c["width"]) * 8, flops=0)
    if kind == "commit":
        moved = int(((st["path"] != np.arange(c["nodes"])) & (st["path"] >= 0)).sum())
        return dict(bytes=2 * c["layers"] * row * (int(st["counts"].sum()) + moved), flops=0)
    need = int((-(-st["lens"] // c["page"])).sum())
    moved = int((st["order"][:need] >= need).sum())
    return dict(bytes=2 * moved * c["page"] * row * c["layers"] + 8 * c["pages"], flops=0)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] not in ("attend", "verify"):
        return None                                               # rows and page numbers move; nothing is computed
    s = _make(case, seed)
    st = _structure(case)
    if case["kind"] == "verify":
        n, N = st["par"].shape
        pick, logprob = np.full((n, N), -1, np.int32), np.zeros((n, N))
        path, taken, follow = np.full((n, N), -1, np.int32), np.zeros(n, np.int32), np.full(n, -1, np.int32)
        allowed = torch.nonzero(s["suppress"] == 0)[:, 0]
        tokens = s["tokens"].cpu().numpy()
        for b in range(n):
            count = int(st["counts"][b])
            x = s["logits"][b, :count].double()[:, allowed].cpu().numpy()
            best = x.argmax(-1)                                   # the first of equals
            pick[b, :count] = allowed.cpu().numpy()[best]
            logprob[b, :count] = x.max(-1) - (x.max(-1) + np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1)))
            cur, k = 0, 0
            while cur is not None:
                path[b, k] = cur
                k, follow[b] = k + 1, pick[b, cur]
                cur = next((j for j in range(cur + 1, count) if st["par"][b, j] == cur and tokens[b, j] == pick[b, cur]), None)
            taken[b] = k
        return dict(pick=pick, logprob=logprob, path=path, n_accept=taken, next=follow)
    n, N, heads, D = s["q"].shape
    H, page = s["k"].shape[2], s["k"].shape[3]
    out = torch.zeros((n, N, heads, D), dtype=torch.float64, device=DEVICE)
    for b in range(n):
        length, count = int(st["lens"][b]), int(st["counts"][b])
        pages = s["table"][b, :-(-(length + count) // page)].long()
        flat = lambda pool: pool[0, pages].transpose(0, 1).reshape(H, -1, D)[:, :length + count].double()  # noqa: E731
        K, V = flat(s["k"]), flat(s["v"])
        if s["kn"] is not None:
            K = torch.cat([K[:, :length], s["kn"][b, :count].double().transpose(0, 1)], 1)
            V = torch.cat([V[:, :length], s["vn"][b, :count].double().transpose(0, 1)], 1)
        hidden = torch.ones((count, length + count), dtype=torch.bool)
        hidden[:, :length] = False
        for i in range(count):
            j = i
            while j >= 0:
                hidden[i, length + j] = False
                j = int(st["par"][b, j])
        for h in range(heads):
            score = s["q"][b, :count, h].double() @ K[h // (heads // H)].T * s["scale"]
            out[b, :count, h] = torch.softmax(score.masked_fill(hidden.to(DEVICE), -math.inf), -1) @ V[h // (heads // H)]
    return dict(out=out, **(dict(k=None, v=None) if s["kn"] is not None else {}))
