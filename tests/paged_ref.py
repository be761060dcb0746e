"""A paged KV cache on the host, in plain Python: the books that fork, grow and
compact keep, and attention over them in 64 bits."""
import numpy as np

NONE = 0xffffffff
U = 2.0 ** -24  # half a step of f32, relative


class Books:
    def __init__(self, n_pages, page_len, n_seqs, max_pages):
        self.P, self.pl, self.S, self.M = n_pages, page_len, n_seqs, max_pages
        self.table = np.full((n_seqs, max_pages), NONE, np.uint32)
        self.lens = np.zeros(n_seqs, np.uint32)
        self.refs = np.zeros(n_pages, np.uint32)

    def used(self, n):
        return -(-int(n) // self.pl)

    def fork(self, frm, keep=None):
        old_t, old_l = self.table.copy(), self.lens.copy()
        self.table[:], self.lens[:], self.refs[:] = NONE, 0, 0
        for s, f in enumerate(frm):
            if f >= self.S:
                continue
            n = min(int(old_l[f]), self.M * self.pl)
            n = n if keep is None else min(n, int(keep[s]))
            self.lens[s] = n
            for i in range(self.used(n)):
                self.table[s, i] = old_t[f, i]
                if old_t[f, i] < self.P:
                    self.refs[old_t[f, i]] += 1

    def grow(self, g):
        """(status, copies): copies = [(source page, destination page, rows)]."""
        status, copies = np.zeros(self.S, np.uint32), []
        left, out = sorted(int(p) for p in np.nonzero(self.refs == 0)[0]), False
        for s in range(self.S):
            n, more = int(self.lens[s]), int(g[s])
            if not more:
                continue
            if n + more > self.M * self.pl:
                status[s] = 2
                continue
            last = int(self.table[s, self.used(n) - 1]) if n % self.pl else NONE
            cow = last < self.P and self.refs[last] > 1
            extra = self.used(n + more) - self.used(n)
            if out or cow + extra > len(left):
                status[s], out = 1, True
                continue
            if cow:
                d = left.pop(0)
                copies.append((last, d, n % self.pl))
                self.refs[last] -= 1
                self.refs[d] = 1
                self.table[s, self.used(n) - 1] = d
            for i in range(extra):
                d = left.pop(0)
                self.refs[d] = 1
                self.table[s, self.used(n) + i] = d
            self.lens[s] = n + more
        return status, copies

    def compact(self):
        """(live pages, moves): moves = [(from id, to id)]."""
        live = [int(p) for p in np.nonzero(self.refs)[0]]
        L = len(live)
        moves = list(zip([p for p in live if p >= L], [p for p in range(L) if not self.refs[p]]))
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        new = dict(moves)
        for s in range(self.S):
            for i in range(self.M):
                self.table[s, i] = new.get(int(self.table[s, i]), self.table[s, i])
        return L, moves


def apply(pool, copies=(), moves=(), page=None):
    """The copies and moves on a pool [layers, pages, page, width], all read before they are written."""
    old = pool.copy()
    for a, b, rows in copies:
        pool[:, b, :rows] = old[:, a, :rows]
    for a, b in moves:
        pool[:, b] = old[:, a]


def positions(books, s, prefix=None):
    """The (page, row) of every position sequence s holds that has a page, and their numbers."""
    n = min(int(books.lens[s]), books.M * books.pl)
    pre = [] if prefix is None else list(prefix)
    ids = np.array([pre[i] if i < len(pre) else books.table[s, i] for i in range(books.used(n))], np.int64)
    pos = np.arange(n)
    page = ids[pos // books.pl] if n else np.zeros(0, np.int64)
    ok = page < books.P
    return page[ok], (pos % books.pl)[ok], pos[ok]


def attn(q, k, v, books, layer, heads, kv_heads, prefix=None):
    """q [S, n, heads * hd] over pools k, v [layers, pages, page, width]: (o, tolerance), f64.

    The tolerance, elementwise: a score is a sum of hd f32 products, off by at
    most (hd + 2) u sum|q k| scale and, in the exponent, 4 roundings of its own
    size (|s| + |max|) u; a weight by twice that relative to the others, and 4 u
    of the exponential; sums over N keys by N u in any order; the quotient
    and what a split joins, 16 u. All of it of sum_x p_x |v_x|."""
    S, n, W = q.shape
    hd, G = W // heads, heads // kv_heads
    out, tol = np.zeros((S, n, heads, hd)), np.zeros((S, n, heads, hd))
    for s in range(S):
        page, row, pos = positions(books, s, prefix)
        K = k[layer, page, row].astype(np.float64).reshape(-1, kv_heads, hd)
        V = v[layer, page, row].astype(np.float64).reshape(-1, kv_heads, hd)
        end = min(int(books.lens[s]), books.M * books.pl)
        for j in range(n):
            m = int(np.searchsorted(pos, end - n + j, side="right")) if end - n + j >= 0 else 0
            if not m:
                continue
            for h in range(heads):
                x = q[s, j, h * hd:(h + 1) * hd].astype(np.float64)
                sc = K[:m, h // G] @ x / np.sqrt(hd)
                size = np.abs(K[:m, h // G]) @ np.abs(x) / np.sqrt(hd)
                e = np.exp(sc - sc.max())
                p = e / e.sum()
                out[s, j, h] = p @ V[:m, h // G]
                d = (hd + 2) * size.max() + 4 * 2 * np.abs(sc).max() + 4
                tol[s, j, h] = (2 * d + m + 16) * U * (p @ np.abs(V[:m, h // G])) + 1e-37
    return out.reshape(q.shape), tol.reshape(q.shape)
