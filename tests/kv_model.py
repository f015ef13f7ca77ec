"""Plain models of the paged cache, tree attention and draft verification (whisper_amd/kvcache.py, whisper_amd/draft.py): numpy, one
entry after the other, 64 bits."""
import numpy as np

OK, INVALID, NOMEM = 0, -1, -3


class PageModel:
    """tables and counts of a cache, and (optionally) pools of token rows, entry by entry as include/whisper_amd.h says"""

    def __init__(self, n_pages, max_seqs, max_pages, page_size, k=None, v=None):
        self.PS, self.max_pages = page_size, max_pages
        self.table = np.full((max_seqs, max_pages), -1, np.int32)
        self.refs = np.zeros(n_pages, np.int32)
        self.lens = np.zeros(max_seqs, np.int32)
        self.held = np.zeros(max_seqs, np.int32)
        self.k, self.v = k, v                                  # [L, P, H, PS, D]

    def state(self):
        return dict(table=self.table, refs=self.refs, lens=self.lens, held=self.held)

    def _ok(self, seqs, i):
        return 0 <= seqs[i] < len(self.lens) and seqs[i] not in seqs[:i]

    def truncate(self, seqs, lens=None):
        out = []
        for i, s in enumerate(seqs):
            want = 0 if lens is None else int(lens[i])
            if not self._ok(seqs, i) or not 0 <= want <= self.lens[s]:
                out.append(INVALID)
                continue
            keep = -(-want // self.PS)
            for p in range(keep, self.held[s]):
                self.refs[self.table[s, p]] -= 1
                self.table[s, p] = -1
            self.lens[s], self.held[s] = want, min(self.held[s], keep)
            out.append(OK)
        return out

    def fork(self, dst, src):
        was = [(self.table[s].copy(), int(self.lens[s])) if 0 <= s < len(self.lens) else None for s in src]
        out = []
        for i, d in enumerate(dst):
            if not self._ok(dst, i) or was[i] is None:
                out.append(INVALID)
                continue
            for p in range(self.held[d]):
                self.refs[self.table[d, p]] -= 1
            row, n = was[i]
            keep = -(-n // self.PS)
            self.table[d] = -1
            self.table[d, :keep] = row[:keep]
            for p in row[:keep]:
                self.refs[p] += 1
            self.lens[d], self.held[d] = n, keep
            out.append(OK)
        return out

    def reserve(self, seqs, extra):
        refs = self.refs.copy()                                # what the call finds
        free = [p for p in range(len(refs)) if refs[p] == 0]
        out, taken = [], 0
        for i, s in enumerate(seqs):
            e = int(extra[i]) if np.ndim(extra) else int(extra)
            if not self._ok(seqs, i) or e < 0:
                out.append(INVALID)
                continue
            n, held = int(self.lens[s]), int(self.held[s])
            want = -(-(n + e) // self.PS)
            if want > self.max_pages:
                out.append(NOMEM)
                continue
            copy = e > 0 and n % self.PS != 0 and refs[self.table[s, n // self.PS]] > 1
            need = int(copy) + max(0, want - held)
            if need and taken + need > len(free):
                taken = len(free) + 1                          # every later entry that needs a page is refused too
                out.append(NOMEM)
                continue
            pages = free[taken:taken + need]
            taken += need
            if copy:
                a, b = self.table[s, n // self.PS], pages.pop(0)
                self.table[s, n // self.PS] = b
                self.refs[a] -= 1
                self.refs[b] = 1
                for pool in (self.k, self.v):
                    if pool is not None:
                        pool[:, b, :, :n % self.PS] = pool[:, a, :, :n % self.PS]
            for j, p in enumerate(pages):
                self.table[s, held + j] = p
                self.refs[p] = 1
            self.held[s] = max(held, want)
            out.append(OK)
        return out

    def places(self, s, upto):
        return [(int(self.table[s, t // self.PS]), t % self.PS) for t in range(self.lens[s], self.lens[s] + upto)]

    def _private(self, s, upto):
        if self.lens[s] + upto > self.held[s] * self.PS:
            return False
        return all(0 <= p < len(self.refs) and self.refs[p] == 1 for p, _ in self.places(s, upto))

    def append(self, seqs, k, v, counts, layers):
        for i, s in enumerate(seqs):
            n = k.shape[2] if counts is None else min(int(counts[i]), k.shape[2])
            if not self._ok(seqs, i) or n <= 0 or not self._private(s, n):
                continue
            for j, (p, t) in enumerate(self.places(s, n)):
                for at, layer in enumerate(layers):
                    self.k[layer, p, :, t] = k[at, i, j]
                    self.v[layer, p, :, t] = v[at, i, j]

    def commit(self, seqs, path, counts):
        out = []
        for i, s in enumerate(seqs):
            n = int(counts[i])
            way = [int(x) for x in path[i][:max(0, n)]]
            if not self._ok(seqs, i) or not 0 <= n <= len(path[i]) or any(x < 0 for x in way) or any(b <= a for a, b in zip(way, way[1:])) or \
                    (n and not self._private(s, way[-1] + 1)):
                out.append(INVALID)
                continue
            spot = self.places(s, way[-1] + 1 if n else 0)
            for pool in (self.k, self.v):
                if pool is not None:
                    for to, frm in enumerate(way):
                        pool[:, spot[to][0], :, spot[to][1]] = pool[:, spot[frm][0], :, spot[frm][1]]
            self.lens[s] += n
            out.append(OK)
        return out

    def compact(self):
        live = np.nonzero(self.refs > 0)[0]
        n = len(live)
        moves = [int(p) for p in live if p >= n]
        holes = [p for p in range(n) if self.refs[p] == 0]
        to = {a: b for a, b in zip(moves, holes)}
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            for pool in (self.k, self.v):
                if pool is not None:
                    pool[:, b] = pool[:, a]
        for s in range(len(self.lens)):
            for p in range(self.max_pages):
                self.table[s, p] = to.get(int(self.table[s, p]), self.table[s, p])
        return n


def ancestors(parents):
    """[N][N] booleans: j is i or an ancestor of i"""
    N = len(parents)
    seen = np.zeros((N, N), bool)
    for i in range(N):
        j = i
        while j >= 0:
            seen[i, j] = True
            j = int(parents[j])
    return seen


def tree_attention(q, K, V, parents, scale):
    """one sequence, one layer, 64 bits: q [N, heads, D]; K, V [tokens + N, kv_heads, D]; returns o [N, heads, D] and, for tolerances,
    sum_j p_j |v_j| and the largest scale * sum |q| |k|.  Masked rows are left out of every sum, not multiplied by 0."""
    N, heads, D = q.shape
    seen = ancestors(parents)
    n_prefix = len(K) - N
    o, mass, reach = np.zeros((N, heads, D)), np.zeros((N, heads, D)), 0.0
    for i in range(N):
        rows = np.concatenate([np.arange(n_prefix), n_prefix + np.nonzero(seen[i])[0]])
        for h in range(heads):
            kh = h // (heads // K.shape[1])
            k, v = K[rows, kh].astype(np.float64), V[rows, kh].astype(np.float64)
            s = scale * (k @ q[i, h].astype(np.float64))
            p = np.exp(s - s.max())
            p /= p.sum()
            o[i, h] = p @ v
            mass[i, h] = p @ np.abs(v)
            reach = max(reach, float((abs(scale) * (np.abs(k) @ np.abs(q[i, h].astype(np.float64)))).max()))
    return o, mass, reach


def attention_bound(o, mass, reach, D, tokens, bf16):
    """How far a kernel may be from the 64-bit result, element by element.  fp32: a score of D products is off by at most D + 2 half
    steps of sum |q||k| scale, the exponent's argument by two more; a probability moves by that much relatively, numerator and
    denominator each, and the sums over the tokens (in any order) and the merges add a half step per term: all times sum p |v|.
    bf16 caches: every probability and the result are rounded to bf16 as well, half a step each."""
    u = 2.0 ** -24
    rel = 2 * (D + 4) * u * reach + (2 * tokens + 64) * u
    if bf16:
        return (rel + 2.0 ** -8) * mass * (1 + 2.0 ** -7) + 2.0 ** -8 * np.abs(o) + 1e-30
    return rel * mass + 1e-30


def verify(logits, tokens, parents, counts, suppress):
    n, N, V = logits.shape
    pick, lp = np.full((n, N), -1, np.int32), np.zeros((n, N))
    path, taken, nxt = np.full((n, N), -1, np.int32), np.zeros(n, np.int32), np.full(n, -1, np.int32)
    for b in range(n):
        for j in range(int(counts[b])):
            x = logits[b, j].astype(np.float64)
            ok = ~np.isnan(x) & (x > -np.inf) & (suppress == 0)
            if not ok.any():
                lp[b, j] = -np.inf
                continue
            ids = np.nonzero(ok)[0]
            pick[b, j] = ids[x[ids].argmax()]
            top = x[ids].max()
            lp[b, j] = -np.log(np.where(x[ids] == top, 1.0, np.exp(np.minimum(x[ids] - (top if np.isfinite(top) else 0), 0) if np.isfinite(top) else -np.inf)).sum())
        cur, k = (0 if counts[b] > 0 else None), 0
        while cur is not None:
            path[b, k] = cur
            k, nxt[b] = k + 1, pick[b, cur]
            cur = next((j for j in range(cur + 1, int(counts[b])) if parents[b, j] == cur and tokens[b, j] == pick[b, cur] and pick[b, cur] >= 0), None)
        taken[b] = k
    return pick, lp, path, taken, nxt
