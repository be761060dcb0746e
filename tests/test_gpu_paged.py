"""GPU: the paged KV cache of a batch (fork, grow, compact, the rotated write)
against its plain bookkeeping, bit for bit, and attention over it against 64
bits, at the sizes, lengths and tables where they can go wrong."""
import numpy as np
import pytest

import paged_ref as ref
from mdma_amd.backend import (ACT_F32, ACT_F32_CPU, ACT_I8, AttnSpec, BackendError, Gfx950Backend, KvPages, KvView,
                              NotImplemented as NotImpl, RopeSpec, ShapeMismatch)  # noqa: F401

pytestmark = pytest.mark.gpu
CANARY = np.float32(123456.25)


def buf(be, a):
    a = np.ascontiguousarray(a)
    b = be.alloc(a.nbytes)
    if a.nbytes:
        be.upload(b, 0, a)
    return b


def u32(be, b, n):
    return be.download(b, 0, 4 * n).view(np.uint32)


class Cache:
    """A KvPages with its host copy."""

    def __init__(self, be, books, layers, width, seed, k=None, v=None):
        self.be, self.books = be, books
        r = np.random.default_rng(seed)
        shape = (layers, books.P, books.pl, width)
        self.k = r.standard_normal(shape, np.float32).astype(np.float16) if k is None else k
        self.v = r.standard_normal(shape, np.float32).astype(np.float16) if v is None else v
        self.dev = KvPages(buf(be, self.k), buf(be, self.v), buf(be, books.table), buf(be, books.lens),
                           buf(be, books.refs), layers, books.P, books.pl, width, books.S, books.M)

    def check(self, what=""):
        b, be, d = self.books, self.be, self.dev
        assert np.array_equal(u32(be, d.lens, b.S), b.lens), what
        assert np.array_equal(u32(be, d.table, b.S * b.M).reshape(b.S, b.M), b.table), what
        assert np.array_equal(u32(be, d.refs, b.P), b.refs), what
        for host, dev in ((self.k, d.k), (self.v, d.v)):
            got = be.download(dev, 0, host.nbytes).view(np.uint16).reshape(host.shape)
            assert np.array_equal(got, host.view(np.uint16)), what


def filled(lens, page_len, seed, slack=3, prefix_pages=0, n_seqs=None, max_pages=None):
    """Books of sequences with these lengths, pages scattered; the first prefix_pages of each shared."""
    S = len(lens)
    probe = ref.Books(1, page_len, S, 1)
    own = [max(0, probe.used(n) - prefix_pages) for n in lens]
    P = prefix_pages + sum(own) + slack
    M = max_pages or max([probe.used(n) for n in lens] + [prefix_pages, 1]) + 1
    b = ref.Books(P, page_len, S, M)
    ids = np.random.default_rng(seed).permutation(P)
    pre, at = ids[:prefix_pages], prefix_pages
    for s, n in enumerate(lens):
        b.lens[s] = n
        u = b.used(n)
        for i in range(u):
            if i < prefix_pages:
                b.table[s, i] = pre[i]
            else:
                b.table[s, i] = ids[at]
                at += 1
            b.refs[b.table[s, i]] += 1
    return b, pre.astype(np.uint32)


# ---- books ----

@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("S,P,pl,M,layers,width", [(1, 5, 16, 4, 1, 8), (8, 60, 16, 9, 3, 48), (33, 300, 32, 12, 2, 64),
                                                   (5, 3000, 16, 700, 1, 8), (200, 1500, 64, 6, 1, 16)])
def test_random_forks_grows_compactions(backend, S, P, pl, M, layers, width, seed):
    r = np.random.default_rng(seed)
    c = Cache(backend, ref.Books(P, pl, S, M), layers, width, seed)
    b = c.books
    frm, keep, grow, status, live = (backend.alloc(4 * S) for _ in range(5))
    for step in range(6):
        g = r.integers(0, pl * 3, S).astype(np.uint32) * (r.random(S) < 0.8)
        if r.random() < 0.2:
            g[r.integers(0, S)] = 0xffffffff  # far past max_pages
        backend.upload(grow, 0, g.astype(np.uint32))
        backend.kv_pages_grow(c.dev, grow, status)
        want, copies = b.grow(g)
        for pool in (c.k, c.v):
            ref.apply(pool, copies=copies)
        assert np.array_equal(u32(backend, status, S), want), (step, "status")
        c.check((step, "grow"))
        f = np.where(r.random(S) < 0.5, np.arange(S), r.integers(0, S + 1, S)).astype(np.uint32)
        f[f == S] = ref.NONE
        kp = r.integers(0, M * pl, S).astype(np.uint32) if r.random() < 0.6 else None
        backend.upload(frm, 0, f)
        if kp is not None:
            backend.upload(keep, 0, kp)
        backend.kv_pages_fork(c.dev, frm, keep if kp is not None else None)
        b.fork(f, kp)
        c.check((step, "fork"))
        backend.kv_pages_compact(c.dev, live if step % 2 else None)
        L, moves = b.compact()
        for pool in (c.k, c.v):
            ref.apply(pool, moves=moves)
        if step % 2:
            assert u32(backend, live, 1)[0] == L
        c.check((step, "compact"))


def test_shared_last_page_copies_all_but_one(backend):
    """Four beams on one partly filled page: three copies, and the last goes on in place; where one of them does not
    grow, all that grow copy."""
    for growing in ([1, 1, 1, 1], [1, 0, 1, 1]):
        b = ref.Books(20, 16, 4, 4)
        b.table[0, :2], b.lens[0], b.refs[[7, 3]] = (7, 3), 21, 1
        c = Cache(backend, b, 2, 16, 1)
        backend.kv_pages_fork(c.dev, buf(backend, np.zeros(4, np.uint32)))
        b.fork([0, 0, 0, 0])
        g, status = buf(backend, np.array(growing, np.uint32)), backend.alloc(16)
        backend.kv_pages_grow(c.dev, g, status)
        _, copies = b.grow(growing)
        assert len(copies) == 3
        for pool in (c.k, c.v):
            ref.apply(pool, copies=copies)
        c.check(growing)


def test_largest_batch_of_sequences(backend):
    S = 1024
    b, _ = filled([17] * S, 16, 3, slack=S + 5)
    c = Cache(backend, b, 1, 8, 2)
    g, status = buf(backend, np.full(S, 16, np.uint32)), backend.alloc(4 * S)
    backend.kv_pages_grow(c.dev, g, status)
    want, _ = b.grow(np.full(S, 16))
    assert np.array_equal(u32(backend, status, S), want) and not want.any()
    backend.kv_pages_fork(c.dev, buf(backend, np.full(S, 1023, np.uint32)))
    b.fork(np.full(S, 1023))
    backend.kv_pages_compact(c.dev)
    _, moves = b.compact()
    for pool in (c.k, c.v):
        ref.apply(pool, moves=moves)
    c.check()


@pytest.mark.parametrize("S,P,M", [(64, 8192, 128), (64, 8193, 64), (65, 8191, 127), (3, 24583, 2731), (1024, 8200, 8)])
def test_books_of_many_pages(backend, S, P, M):
    """Tables and counts about and past what one workgroup holds (8192 entries, 8192 pages); scattered live pages."""
    r = np.random.default_rng(S)
    c = Cache(backend, ref.Books(P, 16, S, M), 1, 8, S)
    b = c.books
    ids, at = r.permutation(P), 0
    for s in range(S):
        b.lens[s] = r.integers(0, min(M, P // S - 1) * 16 - 20)
        u = b.used(b.lens[s])
        b.table[s, :u] = ids[at:at + u]
        b.refs[ids[at:at + u]] += 1
        at += u
    for dev, host in ((c.dev.table, b.table), (c.dev.lens, b.lens), (c.dev.refs, b.refs)):
        backend.upload(dev, 0, host)
    status, live = backend.alloc(4 * S), backend.alloc(4)
    for step in range(2):
        f = np.where(r.random(S) < 0.6, np.arange(S), r.integers(0, S, S)).astype(np.uint32)
        backend.kv_pages_fork(c.dev, buf(backend, f))
        b.fork(f)
        c.check((step, "fork"))
        g = r.integers(0, 20, S).astype(np.uint32)
        backend.kv_pages_grow(c.dev, buf(backend, g), status)
        want, copies = b.grow(g)
        assert np.array_equal(u32(backend, status, S), want)
        for pool in (c.k, c.v):
            ref.apply(pool, copies=copies)
        c.check((step, "grow"))
        backend.kv_pages_compact(c.dev, live)
        L, moves = b.compact()
        for pool in (c.k, c.v):
            ref.apply(pool, moves=moves)
        assert u32(backend, live, 1)[0] == L
        c.check((step, "compact"))


def test_ids_outside_the_pool_are_skipped(backend):
    b, _ = filled([40, 33], 16, 5)
    b.table[0, 1] = b.P  # one past the last page
    b.table[1, 2] = 0x80000000  # the partly filled last page
    b.lens[:] = 40, 33
    c = Cache(backend, b, 2, 16, 4)
    backend.kv_pages_fork(c.dev, buf(backend, np.array([1, 0], np.uint32)))
    b.fork([1, 0])
    c.check("fork")
    g, status = buf(backend, np.array([5, 9], np.uint32)), backend.alloc(8)
    backend.kv_pages_grow(c.dev, g, status)
    _, copies = b.grow([5, 9])
    assert not copies
    c.check("grow")
    backend.kv_pages_compact(c.dev)
    _, moves = b.compact()
    for pool in (c.k, c.v):
        ref.apply(pool, moves=moves)
    c.check("compact")


# ---- the rotated write ----

def angles(pos, hd, theta):
    f = np.array([np.float32(float(np.float32(theta)) ** float(np.float32(-2.0 * i / hd))) for i in range(hd // 2)],
                 np.float32)
    return (np.float32(pos) * f).astype(np.float64)


@pytest.mark.parametrize("lens,new,page,heads,kv_heads,hd", [
    ([1], 1, 16, 1, 1, 8), ([0, 300, 17], 1, 16, 6, 6, 48), ([5, 0, 33, 64], 7, 32, 8, 2, 128),
    ([200, 130], 129, 64, 4, 4, 64), ([1000], 1000, 256, 28, 4, 128), ([40, 41], 2, 16, 16, 1, 256)])
def test_rope_kv_write_paged(backend, lens, new, page, heads, kv_heads, hd):
    b, _ = filled(lens, page, 7)
    S, W, H = len(lens), kv_heads * hd, heads * hd
    if S > 2:
        b.table[2, 0] = b.P + 3  # no page: that position is not stored
    c = Cache(backend, b, 2, W, 3)
    r = np.random.default_rng(9)
    q, k, v = (r.standard_normal((S, new, w)).astype(np.float32) for w in (H, W, W))
    qb, kb, vb = (buf(backend, x) for x in (q, k, v))
    theta = 500000.0
    backend.rope_kv_write_paged(qb, kb, vb, c.dev, 1, RopeSpec(hd, theta))
    want_q = q.astype(np.float64)
    old = c.k.copy()
    for s in range(S):
        for j in range(new):
            p = int(b.lens[s]) - new + j
            if p < 0:
                continue
            z = np.exp(1j * angles(p, hd, theta))
            rows = []
            for x in (q[s, j], k[s, j]):
                w = x.astype(np.float64).reshape(-1, hd // 2, 2) @ np.array([1, 1j]) * z
                rows.append(np.stack([w.real, w.imag], -1).reshape(-1))
            want_q[s, j] = rows[0]
            pg = int(b.table[s, p // page])
            if pg < b.P:
                c.v[1, pg, p % page] = v[s, j].astype(np.float16)  # one rounding
                old[1, pg, p % page] = rows[1].astype(np.float16)
    # q: a pair's products and their sum in f32 with cos and sin each off by 2 u at most: 6 u of |x| + |y|.
    got = backend.download_f32(qb).reshape(q.shape)
    size = np.abs(q).reshape(S, new, -1, 2).sum(-1).repeat(2, -1).reshape(q.shape)
    assert np.all(np.abs(got - want_q) <= 6 * ref.U * size)
    assert np.array_equal(backend.download(vb, 0, v.nbytes).view(np.float32).reshape(v.shape), v)
    assert np.array_equal(backend.download_f32(kb).reshape(k.shape), k)
    gv = backend.download(c.dev.v, 0, c.v.nbytes).view(np.uint16).reshape(c.v.shape)
    assert np.array_equal(gv, c.v.view(np.uint16))
    # k: the same in f32, then one rounding to f16, half a step: 2^-11 relative (2^-25 near zero).
    gk = backend.download(c.dev.k, 0, c.k.nbytes).view(np.float16).reshape(c.k.shape).astype(np.float64)
    sk = np.zeros_like(gk)
    for s in range(S):
        for j in range(new):
            p = int(b.lens[s]) - new + j
            if p >= 0 and b.table[s, p // page] < b.P:
                sk[1, b.table[s, p // page], p % page] = np.abs(k[s, j]).reshape(-1, 2).sum(-1).repeat(2)
    want = old.astype(np.float64)
    assert np.all(np.abs(gk - want) <= (2 * 2.0 ** -11 * np.abs(want) + 2.0 ** -24 + 6 * ref.U * sk) * (sk > 0))


def test_rope_kv_write_paged_same_bits_as_contiguous(backend):
    """One sequence in pages and in a contiguous cache: the same q, k and v bits."""
    hd, heads, kv_heads, n, pos = 64, 8, 2, 5, 37
    b, _ = filled([pos + n], 16, 1)
    c = Cache(backend, b, 1, kv_heads * hd, 2)
    r = np.random.default_rng(2)
    q, k, v = (r.standard_normal((n, w * hd)).astype(np.float32) for w in (heads, kv_heads, kv_heads))
    q1, q2, kb, vb = buf(backend, q), buf(backend, q), buf(backend, k), buf(backend, v)
    kc, vc = (backend.alloc((pos + n) * kv_heads * hd * 2) for _ in range(2))
    backend.rope_kv_write(q1, kb, vb, kc, vc, pos * kv_heads * hd, pos, n, RopeSpec(hd, 1e4), n * kv_heads * hd)
    backend.rope_kv_write_paged(q2, kb, vb, c.dev, 0, RopeSpec(hd, 1e4))
    assert np.array_equal(backend.download(q1, 0, q.nbytes), backend.download(q2, 0, q.nbytes))
    for cont, paged in ((kc, c.dev.k), (vc, c.dev.v)):
        a = backend.download(cont, 0, cont.len).view(np.uint16).reshape(-1, kv_heads * hd)[pos:]
        g = backend.download(paged, 0, c.k.nbytes).view(np.uint16).reshape(c.k.shape)
        page, row, _ = ref.positions(b, 0)
        assert np.array_equal(g[0, page, row][pos:], a)


# ---- attention ----

def run_attn(be, c, q, heads, kv_heads, layer=0, prefix=None, fill=None):
    hd = q.shape[-1] // heads
    qb = buf(be, q)
    ob = be.f32_buf(np.full(q.size + 64, CANARY, np.float32))
    pb = buf(be, prefix) if prefix is not None else None
    be.attn_paged(qb, c.dev, layer, pb, AttnSpec(hd, heads, kv_heads), ob)
    o = be.download_f32(ob)
    assert np.all(o[q.size:] == CANARY)
    return o[:q.size].reshape(q.shape)


def check_attn(be, lens, new, page, heads, kv_heads, hd, prefix_pages=0, seed=1, qscale=1.5, mutate=None):
    b, pre = filled(lens, page, seed, prefix_pages=prefix_pages)
    c = Cache(be, b, 2, kv_heads * hd, seed + 1)
    r = np.random.default_rng(seed + 2)
    q = (r.standard_normal((len(lens), new, heads * hd)) * qscale).astype(np.float32)
    if mutate:
        mutate(b, c, q)
        c = Cache(be, b, 2, kv_heads * hd, seed + 1, c.k, c.v)
    pre = pre if prefix_pages else None
    want, tol = ref.attn(q, c.k, c.v, b, 1, heads, kv_heads, pre)
    got = run_attn(be, c, q, heads, kv_heads, 1, pre)
    assert np.all(np.isfinite(got))
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
    # On the whole: rounding errors of random sign, u sqrt(keys) in the sums, u sqrt(hd) of a score's size.
    err, size = np.linalg.norm(got - want), np.linalg.norm(want)
    n = max(max(lens), 1)
    assert err <= 4 * ref.U * (np.sqrt(n) + 4 * np.sqrt(hd) * max(qscale, 1) + 4) * size + 1e-30, (err, size)
    return got


HEADS = [(1, 1, 8), (6, 6, 48), (8, 2, 64), (28, 4, 128), (16, 1, 256), (24, 8, 80), (40, 8, 128), (3, 3, 16),
         (34, 2, 72)]


@pytest.mark.parametrize("heads,kv_heads,hd", HEADS)
@pytest.mark.parametrize("lens,new,page,prefix_pages", [
    ([1], 1, 16, 0), ([0, 70, 1, 16, 17], 1, 16, 0), ([129, 300, 64], 5, 32, 0), ([400, 0, 131, 260], 1, 64, 2),
    ([90, 200, 70], 3, 16, 4), ([65], 65, 16, 0), ([515, 513], 2, 256, 2)])
def test_attn_paged(backend, heads, kv_heads, hd, lens, new, page, prefix_pages):
    check_attn(backend, lens, new, page, heads, kv_heads, hd, prefix_pages)


@pytest.mark.parametrize("lens,new,page,heads,kv_heads,hd,prefix_pages", [
    ([3000], 1, 16, 8, 2, 128, 0), ([2500, 2100], 1, 32, 4, 4, 64, 60), ([1700] * 9, 1, 16, 8, 2, 64, 100),
    ([700, 650, 800], 40, 64, 4, 1, 128, 9), ([1300, 1, 5], 9, 128, 2, 1, 256, 8), ([2048] * 3, 1, 256, 8, 8, 128, 7),
    ([1100] * 70, 1, 64, 8, 1, 64, 16), ([4100, 40], 2, 16, 14, 2, 64, 1)])
def test_attn_paged_long(backend, lens, new, page, heads, kv_heads, hd, prefix_pages):
    check_attn(backend, lens, new, page, heads, kv_heads, hd, prefix_pages, seed=5)


@pytest.mark.parametrize("page,prefix_pages", [(16, 17), (16, 21), (16, 30), (32, 9), (32, 13), (64, 5), (128, 3)])
@pytest.mark.parametrize("S,new,heads,kv_heads,hd", [(2, 1, 4, 2, 64), (5, 3, 8, 2, 96), (9, 2, 16, 2, 128),
                                                     (3, 40, 4, 2, 128), (6, 3, 8, 1, 256)])
def test_attn_paged_prefix_that_ends_inside_a_tile(backend, page, prefix_pages, S, new, heads, kv_heads, hd):
    """A shared prefix of any number of pages, few query rows and many: no key behind it counts twice. Tails of one
    position to a few pages, and sequences that end in the prefix."""
    pre = page * prefix_pages
    lens = [pre + new + i * 17 % 70 for i in range(S)]
    lens[-1] = pre - 5 if S > 2 else pre + new
    check_attn(backend, lens, new, page, heads, kv_heads, hd, prefix_pages)


# (prefixes long enough to be read once for the batch)
LONG_PREFIX = [(16, 64), (16, 65), (16, 67), (16, 70), (32, 33), (64, 17), (128, 9), (256, 5)]


@pytest.mark.parametrize("page,prefix_pages", LONG_PREFIX)
@pytest.mark.parametrize("S,new,heads,kv_heads,hd", [(2, 1, 4, 2, 64), (3, 3, 8, 2, 96), (9, 2, 16, 2, 128),
                                                     (3, 40, 2, 1, 128), (6, 3, 8, 1, 256), (5, 2, 6, 6, 48)])
def test_attn_paged_long_prefix(backend, page, prefix_pages, S, new, heads, kv_heads, hd):
    pre = page * prefix_pages
    lens = [pre + new + i * 17 % 70 for i in range(S)]
    lens[-1] = pre - 5 if S > 2 else pre + new
    if S > 3:
        lens[1], lens[2] = 0, 500
    check_attn(backend, lens, new, page, heads, kv_heads, hd, prefix_pages)


@pytest.mark.parametrize("page,prefix_pages", LONG_PREFIX)
@pytest.mark.parametrize("S,new,heads,kv_heads", [(3, 1, 8, 2), (24, 3, 8, 2)])
def test_attn_paged_long_prefix_beside_anything(backend, page, prefix_pages, S, new, heads, kv_heads):
    """NaN in pages of no one, behind every sequence's end and in the other layer, infinities where a prefix list
    names no page: none of it is read into a row."""
    pre = page * prefix_pages
    lens = [pre + new + i * 5 % 37 for i in range(S)]
    lens[1] = pre - page - 3

    def mutate(b, c, q):
        held = np.zeros((b.P, b.pl), bool)
        for s in range(b.S):
            p, row, _ = ref.positions(b, s)
            held[p, row] = True
        for pool in (c.k, c.v):
            pool[:, ~held] = np.nan
            pool[0] = np.inf
    check_attn(backend, lens, new, page, heads, kv_heads, 64, prefix_pages, mutate=mutate)
    # Pages of the prefix that are not there: page 0, of no one, holds NaN.
    b, ids = filled(lens, page, 3, prefix_pages=prefix_pages)
    c = Cache(backend, b, 1, kv_heads * 64, 4)
    ids = ids.copy()
    gone = [0, 3, prefix_pages - 1]
    c.k[0, ids[gone]], c.v[0, ids[gone]] = np.nan, -np.inf
    c = Cache(backend, b, 1, kv_heads * 64, 4, c.k, c.v)
    ids[gone] = [b.P, ref.NONE, 0x80000000]
    q = np.random.default_rng(5).standard_normal((S, new, heads * 64)).astype(np.float32)
    want, tol = ref.attn(q, c.k, c.v, b, 0, heads, kv_heads, ids)
    assert np.all(np.abs(run_attn(backend, c, q, heads, kv_heads, 0, ids) - want) <= tol)


@pytest.mark.parametrize("S", [2, 40])
def test_attn_paged_long_prefix_values_that_are_not_finite(backend, S):
    """An infinite value in the shared prefix makes its dim infinite for every row that sees it, a NaN key the row NaN;
    a sequence that ends before them has neither."""
    page, pages = 32, 40
    for k_bad in (False, True):
        lens = [page * pages + 1 + i % 7 for i in range(S - 1)] + [1100]
        b, ids = filled(lens, page, 3, prefix_pages=pages)
        c = Cache(backend, b, 1, 64, 4)
        if k_bad:
            c.k[0, ids[37], 9, 3] = np.nan
        else:
            c.v[0, ids[37], 9, 7] = np.inf
        c = Cache(backend, b, 1, 64, 4, c.k, c.v)
        q = np.random.default_rng(6).standard_normal((S, 1, 128)).astype(np.float32)
        got = run_attn(backend, c, q, 2, 1, 0, ids)
        (c.k if k_bad else c.v)[0, ids[37], 9] = np.where(np.isfinite((c.k if k_bad else c.v)[0, ids[37], 9]),
                                                          (c.k if k_bad else c.v)[0, ids[37], 9], 0)
        want, tol = ref.attn(q, c.k, c.v, b, 0, 2, 1, ids)
        assert np.all(np.abs(got - want)[-1] <= tol[-1])
        if k_bad:
            assert np.all(np.isnan(got[:-1]))
        else:
            got = got.reshape(S, 2, 64)
            assert np.all(got[:-1, :, 7] == np.inf)
            assert np.all(np.isfinite(np.delete(got[:-1], 7, -1)))
            other = np.abs(got - want.reshape(got.shape))[:-1] <= tol.reshape(got.shape)[:-1]
            assert np.all(np.delete(other, 7, -1))


@pytest.mark.parametrize("seed", range(40))
def test_attn_paged_any_sizes(backend, seed):
    """Sizes, lengths (around the prefix's end, below new, 0) and prefixes drawn at random."""
    r = np.random.default_rng(1000 + seed)
    heads, kv_heads, hd = [(2, 1, 8), (6, 6, 48), (8, 2, 64), (7, 1, 128), (4, 1, 256), (6, 2, 80), (12, 2, 24),
                           (34, 2, 72)][r.integers(8)]
    page, new = int(2 ** r.integers(4, 9)), int(r.choice([1, 1, 2, 3, 9, 33]))
    S = int(r.integers(1, 1 + (12 if new < 4 else 4)))
    prefix_pages = int(r.choice([0, r.integers(1, 300 // page + 2), r.integers(1024 // page, 1500 // page + 2)]))
    pre = prefix_pages * page
    lens = [int(pre + r.choice([0, 1, new, r.integers(1, 40), r.integers(1, 700)])) for _ in range(S)]
    for s in range(S):
        if r.random() < 0.2:
            lens[s] = int(r.choice([0, 1, max(0, new - 1), max(0, pre - 1), r.integers(0, pre + 1)]))
    check_attn(backend, lens, new, page, heads, kv_heads, hd, prefix_pages, seed=seed)


def test_attn_paged_wide_scores(backend):
    """Queries forty times larger: a few keys take all the weight."""
    check_attn(backend, [700, 33, 290], 2, 16, 8, 2, 64, 1, qscale=40.0)


@pytest.mark.parametrize("scale", [1e-30, 1e-8, 1e8, 1e30])
def test_attn_paged_any_query_size(backend, scale):
    """Queries far from 1, with values over many binades in a row."""
    def mutate(b, c, q):
        q *= np.float32(scale)
        q[..., ::3] *= np.float32(2.0 ** -9)
        if scale > 1:  # (scores of a size that keeps the softmax finite and the bound meaningful)
            c.k[:] = (c.k.astype(np.float32) * 0).astype(np.float16)
            c.k[..., 0] = np.float16(6e-8) if scale == 1e8 else 0
    check_attn(backend, [300, 20], 1, 16, 4, 2, 64, qscale=1.0, mutate=mutate)


@pytest.mark.parametrize("prefix_pages", [0, 3])
def test_attn_paged_masked_places_may_hold_anything(backend, prefix_pages):
    """NaN and infinities past a sequence's length, in pages of no one, and (K and V) at keys after a query."""
    def mutate(b, c, q):
        held = np.zeros((b.P, b.pl), bool)
        for s in range(b.S):
            page, row, _ = ref.positions(b, s)
            held[page, row] = True
        for pool in (c.k, c.v):
            pool[:, ~held] = np.nan
            pool[0] = np.inf  # the other layer
    check_attn(backend, [70, 0, 1, 95, 49], 1, 16, 8, 2, 64, prefix_pages, mutate=mutate)
    # The last of three new tokens' key and value are not finite: only that token's row is.
    b, pre = filled([90, 52], 16, 3, prefix_pages=prefix_pages)
    c = Cache(backend, b, 1, 128, 4)
    for s in range(2):
        p = int(b.lens[s]) - 1
        c.k[0, b.table[s, p // 16], p % 16] = np.nan
        c.v[0, b.table[s, p // 16], p % 16] = np.inf
    c = Cache(backend, b, 1, 128, 4, c.k, c.v)
    q = np.random.default_rng(5).standard_normal((2, 3, 512)).astype(np.float32)
    pre = pre if prefix_pages else None
    got = run_attn(backend, c, q, 8, 2, 0, pre)
    for s in range(2):
        p = int(b.lens[s]) - 1
        c.k[0, b.table[s, p // 16], p % 16] = 0
        c.v[0, b.table[s, p // 16], p % 16] = 0
    want, tol = ref.attn(q, c.k, c.v, b, 0, 8, 2, pre)
    assert np.all(np.abs(got - want)[:, :2] <= tol[:, :2])
    assert np.all(np.isnan(got[:, 2]))


def test_attn_paged_values_that_are_not_finite(backend):
    """As the formula has them: a key at score -inf has no weight, one at +inf or NaN makes the row NaN, an infinite
    value its dim infinite, an infinite query the row NaN."""
    b, _ = filled([100] * 5, 16, 3)
    c = Cache(backend, b, 1, 64, 4)
    q = np.random.default_rng(6).standard_normal((5, 1, 64)).astype(np.float32)
    q[:3, 0, 0] = 1.0
    at = [(int(b.table[s, 1]), 5) for s in range(5)]
    c.k[0, at[0][0], 5, 0] = -np.inf
    c.k[0, at[1][0], 5, 0] = np.inf
    c.v[0, at[2][0], 5, 7] = -np.inf
    q[3, 0, 9] = np.inf
    q[4, 0, 9] = np.nan
    c = Cache(backend, b, 1, 64, 4, c.k, c.v)
    got = run_attn(backend, c, q, 1, 1)
    k0 = c.k.astype(np.float64)
    with np.errstate(invalid="ignore"):
        for s in range(5):
            page, row, _ = ref.positions(b, s)
            sc = k0[0, page, row] @ q[s, 0].astype(np.float64) / 8
            p = np.exp(sc - sc.max())
            want = (p / p.sum()) @ c.v[0, page, row].astype(np.float64)
            g = got[s, 0]
            assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(np.isinf(g), np.isinf(want)), s
            fin = np.isfinite(want)
            # scores of at most 40 with 64 terms, 100 keys: the bound of ref.attn at these sizes
            assert np.all(np.abs(g[fin] - want[fin]) <= (2 * (66 * 40 + 8 * 40) + 116) * ref.U * 4), s


def test_attn_paged_pages_that_are_not_there(backend):
    def mutate(b, c, q):
        b.table[0, 1] = b.P
        b.table[1, :] = ref.NONE
        b.table[2, 3] = 0xfffffffe
        b.lens[3] = 0xffffffff  # read as the table's end, entries past its pages naming none
    got = check_attn(backend, [70, 40, 64, 30], 1, 16, 8, 2, 64, mutate=mutate)
    assert not got[1].any()


@pytest.mark.parametrize("S,new,lens", [(1, 1025, [1900]), (2, 1025, [1900, 1100]), (1, 2100, [2200])])
def test_attn_paged_more_rows_than_parts_have_room_for(backend, S, new, lens):
    """Rows whose parts would take hundreds of MB: fewer parts, in the end none, and the prefix read by each sequence.
    Some rows of each wave against 64 bits."""
    heads, hd, page, prefix_pages = 64, 256, 64, 8
    b, pre = filled(lens, page, 5, prefix_pages=prefix_pages)
    c = Cache(backend, b, 1, hd, 6)
    r = np.random.default_rng(7)
    q = r.standard_normal((S, new, heads * hd), np.float32)
    ob = backend.alloc(q.nbytes)
    backend.attn_paged(buf(backend, q), c.dev, 0, buf(backend, pre), AttnSpec(hd, heads, 1), ob)
    o = backend.download_f32(ob).reshape(S, new, heads, hd)
    assert np.isfinite(o).all()
    q = q.reshape(o.shape)
    for s in range(S):
        for j in [0, 1, 2, 15, 16, new // 2, new - 2, new - 1]:
            # (one query of a shorter sequence: the same keys)
            one, at = ref.Books(b.P, page, 1, b.M), int(b.lens[s]) - new + j + 1
            one.table[0], one.lens[0] = b.table[s], at
            h = r.integers(0, heads, 3)
            want, tol = ref.attn(q[s, j, h].reshape(1, 1, -1), c.k, c.v, one, 0, 3, 1)
            assert np.all(np.abs(o[s, j, h].reshape(1, 1, -1) - want) <= tol), (s, j, h)


def test_attn_paged_no_prefix_equals_prefix(backend):
    """The same cache with its shared pages named and not: within the bound of either."""
    b, pre = filled([300, 280, 1, 500], 16, 8, prefix_pages=10)
    b.lens[2], b.refs[:] = 37, 9  # shorter than the prefix
    b.table[2, :3] = pre[:3]
    c = Cache(backend, b, 1, 128, 3)
    q = np.random.default_rng(1).standard_normal((4, 2, 512)).astype(np.float32)
    want, tol = ref.attn(q, c.k, c.v, b, 0, 8, 2)
    for p in (None, pre, pre[:1], np.zeros(0, np.uint32)):
        got = run_attn(backend, c, q, 8, 2, 0, p)
        assert np.all(np.abs(got - want) <= tol)


def test_attn_paged_prefix_as_a_view_of_a_table_row(backend):
    b, pre = filled([100, 90], 16, 8, prefix_pages=4)
    c = Cache(backend, b, 1, 64, 3)
    q = np.random.default_rng(1).standard_normal((2, 1, 128)).astype(np.float32)
    view = backend.view(c.dev.table, b.M * 4, 16)  # row 1, four pages
    ob = backend.alloc(q.nbytes)
    backend.attn_paged(buf(backend, q), c.dev, 0, view, AttnSpec(64, 2, 1), ob)
    want, tol = ref.attn(q, c.k, c.v, b, 0, 2, 1)
    assert np.all(np.abs(backend.download_f32(ob).reshape(q.shape) - want) <= tol)


def test_attn_paged_matches_contiguous_attention(backend):
    """The same sequence in pages and in a contiguous cache: both within the bound."""
    b, _ = filled([333], 16, 2)
    c = Cache(backend, b, 1, 256, 5)
    page, row, _ = ref.positions(b, 0)
    kc, vc = buf(backend, c.k[0, page, row]), buf(backend, c.v[0, page, row])
    q = np.random.default_rng(3).standard_normal((1, 4, 8 * 128)).astype(np.float32)
    o = backend.alloc(q.nbytes)
    backend.attn(buf(backend, q), KvView(kc, vc, 333), AttnSpec(128, 8, 2), o)
    want, tol = ref.attn(q, c.k, c.v, b, 0, 8, 2)
    for got in (run_attn(backend, c, q, 8, 2), backend.download_f32(o).reshape(q.shape)):
        assert np.all(np.abs(got - want) <= tol)


def test_attn_paged_same_call_same_bits(backend):
    b, pre = filled([900, 700, 811], 16, 2, prefix_pages=30)
    c = Cache(backend, b, 1, 256, 5)
    q = np.random.default_rng(3).standard_normal((3, 1, 8 * 128)).astype(np.float32)
    first = run_attn(backend, c, q, 8, 2, 0, pre)
    for mode in (ACT_F32, ACT_I8, ACT_F32_CPU, ACT_F32):
        backend.set_act_mode(mode)
        try:
            assert np.array_equal(run_attn(backend, c, q, 8, 2, 0, pre), first)
        finally:
            backend.set_act_mode(ACT_F32)


def test_paged_cache_past_32_bit_offsets(backend):
    """Pages whose elements lie past 2^32 in a pool of 9 GB, attended to, written, copied and moved."""
    pl, W, hd = 256, 1024, 128
    P = (1 << 32) // (pl * W) + 40
    k, v = (backend.alloc(P * pl * W * 2) for _ in range(2))
    try:
        r = np.random.default_rng(1)
        far = [P - 1, P - 7, P - 30]
        data = {}
        for p in far + [2]:
            for n, pool in (("k", k), ("v", v)):
                data[n, p] = r.standard_normal((pl, W), np.float32).astype(np.float16)
                backend.upload(pool, p * pl * W * 2, data[n, p])
        b = ref.Books(P, pl, 2, 4)
        b.table[0, :3], b.lens[0] = far, 700
        b.refs[far] = 1
        dev = KvPages(k, v, buf(backend, b.table), buf(backend, b.lens), buf(backend, b.refs), 1, P, pl, W, 2, 4)

        def attend():
            q = r.standard_normal((2, 1, 8 * hd)).astype(np.float32)
            o = backend.alloc(q.nbytes)
            backend.attn_paged(buf(backend, q), dev, 0, None, AttnSpec(hd, 8, 8), o)
            small = ref.Books(4, pl, 2, 4)
            small.lens[:] = b.lens
            small.table[:] = b.table
            ids = sorted({int(x) for x in b.table[b.table != ref.NONE]})
            for i, p in enumerate(ids):
                small.table[b.table == p] = i
            small.P = len(ids)
            pools = [np.stack([backend.download(x, p * pl * W * 2, pl * W * 2).view(np.float16).reshape(pl, W)
                               for p in ids])[None] for x in (k, v)]
            want, tol = ref.attn(q, *pools, small, 0, 8, 8)
            assert np.all(np.abs(backend.download_f32(o).reshape(q.shape) - want) <= tol)

        attend()
        frm = buf(backend, np.zeros(2, np.uint32))
        backend.kv_pages_fork(dev, frm)
        b.fork([0, 0])
        g, status = buf(backend, np.array([3, 4], np.uint32)), backend.alloc(8)
        backend.kv_pages_grow(dev, g, status)  # one copy of the far last page into page 0
        _, copies = b.grow([3, 4])
        assert [(a, d) for a, d, _ in copies] == [(far[2], 0)]
        for n, pool in (("k", k), ("v", v)):
            got = backend.download(pool, 0, copies[0][2] * W * 2).view(np.float16).reshape(-1, W)
            assert np.array_equal(got.view(np.uint16), data[n, far[2]][:copies[0][2]].view(np.uint16))
        q, nk, nv = (r.standard_normal((2, 3, W)).astype(np.float32) for _ in range(3))
        backend.rope_kv_write_paged(buf(backend, q), buf(backend, nk), buf(backend, nv), dev, 0, RopeSpec(hd, 1e4))
        last = int(b.lens[1]) - 1
        got = backend.download(v, (int(b.table[1, last // pl]) * pl + last % pl) * W * 2, W * 2).view(np.uint16)
        assert np.array_equal(got, nv[1, 2].astype(np.float16).view(np.uint16))
        attend()
        backend.kv_pages_compact(dev)
        L, moves = b.compact()
        assert L == 4 and len(moves) == 3
        assert np.array_equal(u32(backend, dev.table, 8).reshape(2, 4), b.table)
        attend()
    finally:
        k.close()
        v.close()


def test_captured_decode_steps_replay(backend):
    """grow, write and attend captured once; every replay is the next step, with eager work between the replays."""
    S, hd, heads, kvh, page = 3, 64, 8, 2, 16
    W, H = kvh * hd, heads * hd
    b, pre = filled([40, 0, 63], page, 2, slack=30, prefix_pages=2, max_pages=12)
    b.lens[1], b.refs[pre] = 35, 3
    b.table[1, :2] = pre
    b.table[1, 2] = [p for p in range(b.P) if not b.refs[p]][0]
    b.refs[b.table[1, 2]] = 1
    c = Cache(backend, b, 2, W, 3)
    r = np.random.default_rng(4)
    qb, kb, vb, ob = (backend.alloc(S * n * 4) for n in (H, W, W, H))
    g, status, pb = buf(backend, np.ones(S, np.uint32)), backend.alloc(4 * S), buf(backend, pre)

    def step():
        backend.kv_pages_grow(c.dev, g, status)
        backend.rope_kv_write_paged(qb, kb, vb, c.dev, 1, RopeSpec(hd, 1e4))
        backend.attn_paged(qb, c.dev, 1, pb, AttnSpec(hd, heads, kvh), ob)

    def inputs():
        x = [r.standard_normal((S, 1, n)).astype(np.float32) for n in (H, W, W)]
        for dst, a in zip((qb, kb, vb), x):
            backend.upload(dst, 0, a)

    backend.reserve_scratch(32 << 20)  # (eager calls between the replays must not grow it)
    inputs()
    step()
    b.grow(np.ones(S))
    backend.join_execution()
    graphs = [backend.capture(step), backend.capture(step)]  # two, sharing the context's workspace
    for i in range(40):
        inputs()
        graphs[i % 2].launch()
        b.grow(np.ones(S))
        if i % 3 == 0:  # eager work of the same kind in between, and its answer
            backend.join_execution()
            check_attn(backend, [200, 31], 1, 16, 4, 2, 64, 2, seed=i)
        assert np.array_equal(u32(backend, c.dev.lens, S), b.lens)
        k, v = (backend.download(x, 0, c.k.nbytes).view(np.float16).reshape(c.k.shape) for x in (c.dev.k, c.dev.v))
        q = backend.download_f32(qb).reshape(S, 1, H)
        want, tol = ref.attn(q, k, v, b, 1, heads, kvh, pre)
        assert np.all(np.abs(backend.download_f32(ob).reshape(S, 1, H) - want) <= tol), i
    assert np.array_equal(u32(backend, c.dev.table, b.S * b.M).reshape(b.S, b.M), b.table)
    for x in graphs:
        x.close()


def test_refusals_reach_the_caller(backend):
    b, pre = filled([20, 20], 16, 1)
    c = Cache(backend, b, 1, 64, 1)
    q, o = backend.alloc(2 * 128 * 4), backend.alloc(2 * 128 * 4)
    with pytest.raises(ShapeMismatch):
        backend.attn_paged(q, c.dev, 1, None, AttnSpec(64, 2, 1), o)
    with pytest.raises(ShapeMismatch):
        backend.attn_paged(q, c.dev, 0, None, AttnSpec(64, 2, 1), q)
    other = Gfx950Backend(0)
    try:
        with pytest.raises(ShapeMismatch):
            other.attn_paged(q, c.dev, 0, None, AttnSpec(64, 2, 1), o)
        with pytest.raises(ShapeMismatch):
            other.kv_pages_compact(c.dev)
    finally:
        other.close()
    assert np.array_equal(u32(backend, c.dev.lens, 2), b.lens)
