"""GPU: a batch of requests decoded with all of its operators together, as a
server would: fork, grow, projections with adapters, the rotated write,
attention behind a shared prefix and compact, step after step on one cache,
eager and as a captured graph. The cache has to stay what its plain
bookkeeping says bit for bit, and each operator's output near 64 bits of what
it read."""
import numpy as np
import pytest

import paged_ref as ref
from test_gpu_lora import Set
from test_gpu_paged import Cache, angles, buf, filled, u32
from mdma_amd import synth
from mdma_amd.backend import GGML_F16, GGML_Q8_0, AttnSpec, RopeSpec

pytestmark = pytest.mark.gpu
LAYERS, D, HEADS, KV_HEADS, HD, PAGE, THETA = 2, 96, 4, 2, 32, 16, 1e4
H, W = HEADS * HD, KV_HEADS * HD


class Step:
    """The buffers and launches of one decode step of S sequences."""

    def __init__(self, be, S, new, prefix_pages, cache, seed):
        self.be, self.cache, self.S, self.new = be, cache, S, new
        T = S * new
        self.w = [{n: be.upload_weight(synth.weight(GGML_Q8_0, r, c, seed + 8 * i + j), GGML_Q8_0, (r, c))
                   for j, (n, r, c) in enumerate((("q", H, D), ("k", W, D), ("v", W, D), ("o", D, H)))}
                  for i in range(LAYERS)]
        self.lq = [Set(be, GGML_F16, D, H, 32, [4, 0, 32], seed + i) for i in range(LAYERS)]
        self.lo = [Set(be, GGML_F16, H, D, 32, [4, 0, 32], seed + 5 + i) for i in range(LAYERS)]
        self.b = [{n: be.alloc(4 * T * c) for n, c in (("x", D), ("q0", H), ("q", H), ("k", W), ("v", W), ("o", H),
                                                       ("y0", D), ("y", D))} for _ in range(LAYERS)]
        self.out = be.alloc(4 * T * D)
        self.ids, self.frm, self.keep, self.grow, self.status, self.live = (
            be.alloc(4 * n) for n in (T, S, S, S, S, 1))
        # (the shared prefix's ids: sequence 0's row, so compact renumbers them too)
        self.prefix = be.view(cache.dev.table, 0, 4 * prefix_pages)

    def books(self):
        self.be.kv_pages_fork(self.cache.dev, self.frm, self.keep)
        self.be.kv_pages_grow(self.cache.dev, self.grow, self.status)

    def layers(self):
        be, dev = self.be, self.cache.dev
        for i, (w, b) in enumerate(zip(self.w, self.b)):
            be.qmatmul(w["q"], b["x"], b["q0"])
            be.lora_add(self.lq[i].dev, self.ids, b["x"], b["q0"], b["q"])
            be.qmatmul(w["k"], b["x"], b["k"])
            be.qmatmul(w["v"], b["x"], b["v"])
            be.rope_kv_write_paged(b["q"], b["k"], b["v"], dev, i, RopeSpec(HD, THETA))
            be.attn_paged(b["q"], dev, i, self.prefix, AttnSpec(HD, HEADS, KV_HEADS), b["o"])
            be.qmatmul(w["o"], b["o"], b["y0"])
            be.lora_add(self.lo[i].dev, self.ids, b["o"], b["y0"], b["y"])
            be.add(b["x"], b["y"], self.b[i + 1]["x"] if i + 1 < LAYERS else self.out)

    def compact(self):
        self.be.kv_pages_compact(self.cache.dev, self.live)

    def get(self, layer, name, width):
        return self.be.download_f32(self.b[layer][name]).reshape(self.S, self.new, width)


def rotated(x, pos, tol):
    """x [heads * HD] at pos in 64 bits, and its tolerance: x's own carried along, and the rotation's 6 u."""
    z = np.exp(1j * angles(pos, HD, THETA))
    w = x.astype(np.float64).reshape(-1, HD // 2, 2) @ np.array([1, 1j]) * z
    size = np.abs(x).reshape(-1, 2).sum(-1).repeat(2)
    t = np.broadcast_to(tol, x.shape).reshape(-1, 2).sum(-1).repeat(2)
    return np.stack([w.real, w.imag], -1).reshape(-1), t * (1 + 6 * ref.U) + 6 * ref.U * size


def check_step(be, st, ids, prefix_pages):
    c, b = st.cache, st.cache.books
    pre = b.table[0, :prefix_pages]
    for i in range(LAYERS):
        x, q0, kn, vn = (st.get(i, n, w) for n, w in (("x", D), ("q0", H), ("k", W), ("v", W)))
        want, tol = st.lq[i].want(ids, x.reshape(-1, D), q0.reshape(-1, H))
        want, tol = want.reshape(q0.shape), tol.reshape(q0.shape)
        got_q = st.get(i, "q", H)
        gk, gv = (be.download(p, 0, c.k.nbytes).view(np.float16).reshape(c.k.shape) for p in (c.dev.k, c.dev.v))
        for s in range(st.S):
            for j in range(st.new):
                p = int(b.lens[s]) - st.new + j
                if p < 0:
                    continue
                wq, tq = rotated(want[s, j], p, tol[s, j])
                assert np.all(np.abs(got_q[s, j] - wq) <= tq), (i, s, j)
                at = i, b.table[s, p // PAGE], p % PAGE
                wk, tk = rotated(kn[s, j], p, 0)
                # (one rounding to f16 of the f32 that tk is about)
                assert np.all(np.abs(gk[at] - wk) <= 2.0 ** -11 * np.abs(wk) + 2.0 ** -25 + 2 * tk), (i, s, j)
                c.k[at], c.v[at] = gk[at], vn[s, j].astype(np.float16)
        # every other position as it was, and v's rounding: bit for bit
        assert np.array_equal(gk[i].view(np.uint16), c.k[i].view(np.uint16))
        assert np.array_equal(gv[i].view(np.uint16), c.v[i].view(np.uint16))
        o = st.get(i, "o", H)
        wo, to = ref.attn(got_q, gk, gv, b, i, HEADS, KV_HEADS, pre)
        assert np.all(np.abs(o - wo) <= to), i
        y0, y = st.get(i, "y0", D).reshape(-1, D), st.get(i, "y", D).reshape(-1, D)
        wy, ty = st.lo[i].want(ids, o.reshape(-1, H), y0)
        assert np.all(np.abs(y - wy) <= ty), i


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("captured", [False, True])
def test_decode_steps(backend, captured, new):
    S, prefix_pages, start = 6, 2, 41
    books, _ = filled([start] * S, PAGE, 3, slack=40, prefix_pages=prefix_pages, max_pages=8)
    # One request's prompt, which the others continue: its third page is shared too, partly filled.
    books.fork([0] * S)
    c = Cache(backend, books, LAYERS, W, 4)
    st = Step(backend, S, new, prefix_pages, c, 11)
    r = np.random.default_rng(new)
    backend.reserve_scratch(32 << 20)  # (other calls between the replays must not grow it)
    graph = None

    def step():
        st.books()
        st.layers()

    def warm():  # (what a first call allocates, before the capture)
        backend.upload(st.frm, 0, np.arange(S, dtype=np.uint32))
        backend.upload(st.keep, 0, np.full(S, 0xffffffff, np.uint32))
        for x in (st.grow, st.ids):
            backend.upload(x, 0, np.zeros(x.len // 4, np.uint32))
        k, v = (backend.download(p, 0, p.len) for p in (c.dev.k, c.dev.v))
        step()
        st.compact()
        backend.join_execution()
        for p, old in ((c.dev.k, k), (c.dev.v, v), (c.dev.table, books.table), (c.dev.refs, books.refs)):
            backend.upload(p, 0, old)

    if captured:
        warm()
        graph = backend.capture(step)
        compact = backend.capture(st.compact)
    for i in range(14):
        # Sequence 0 goes on; the others take a place of any, now and then cut, or end.
        f = np.where(r.random(S) < 0.6, np.arange(S), r.integers(0, S, S)).astype(np.uint32)
        f[r.random(S) < 0.1] = ref.NONE
        f[0] = 0
        keep = np.full(S, 0xffffffff, np.uint32)
        for s in range(1, S):
            if f[s] < S and r.random() < 0.2:
                keep[s] = r.integers(prefix_pages * PAGE, 60)
        ended = [s for s in range(S) if f[s] >= S or not books.lens[f[s]]]
        for s in ended[:1]:  # a new request behind the shared prompt
            f[s], keep[s] = 0, start
            ended.remove(s)
        grow = np.full(S, new, np.uint32)
        grow[ended] = 0
        ids = r.choice([0, 1, 2, 3, ref.NONE], S * new).astype(np.uint32)
        x = r.standard_normal((S * new, D)).astype(np.float32)
        for dst, a in ((st.frm, f), (st.keep, keep), (st.grow, grow), (st.ids, ids), (st.b[0]["x"], x)):
            backend.upload(dst, 0, a)
        graph.launch() if captured else step()
        books.fork(f, keep)
        status, copies = books.grow(grow)
        for pool in (c.k, c.v):
            ref.apply(pool, copies=copies)
        assert np.array_equal(u32(backend, st.status, S), status) and not status.any()
        check_step(backend, st, ids, prefix_pages)
        c.check((i, "step"))
        if i % 3 == 2:
            compact.launch() if captured else st.compact()
            L, moves = books.compact()
            for pool in (c.k, c.v):
                ref.apply(pool, moves=moves)
            assert u32(backend, st.live, 1)[0] == L
            c.check((i, "compact"))
    if captured:
        graph.close()
        compact.close()


def test_prompts_of_a_batch_then_decode_same_bits_as_one_by_one(backend):
    """Sequences written and decoded as a batch hold the same cache bits as each of them alone in a cache of its own:
    neither pages nor neighbours change what is stored."""
    S, steps = 3, 5
    r = np.random.default_rng(8)
    x = r.standard_normal((steps, S, 3, W)).astype(np.float32)
    spec = RopeSpec(HD, THETA)
    whole = backend.kv_pages(1, 20, PAGE, W, S, 4)
    single = [backend.kv_pages(1, 6, PAGE, W, 1, 4) for _ in range(S)]
    status = backend.alloc(4 * S)
    for t in range(steps):
        backend.kv_pages_grow(whole, buf(backend, np.full(S, 3, np.uint32)), status)
        backend.rope_kv_write_paged(buf(backend, x[t]), buf(backend, x[t]), buf(backend, x[t]), whole, 0, spec)
        for s, c in enumerate(single):
            backend.kv_pages_grow(c, buf(backend, np.full(1, 3, np.uint32)), status)
            backend.rope_kv_write_paged(buf(backend, x[t, s]), buf(backend, x[t, s]), buf(backend, x[t, s]), c, 0, spec)

    def rows(c, s, n):
        table = u32(backend, c.table, c.n_seqs * c.max_pages).reshape(c.n_seqs, -1)[s]
        for pool in (c.k, c.v):
            p = backend.download(pool, 0, pool.len).view(np.uint16).reshape(c.n_pages, PAGE, W)
            yield p[table[:-(-n // PAGE)]].reshape(-1, W)[:n]

    for s, c in enumerate(single):
        for a, b in zip(rows(whole, s, 3 * steps), rows(c, 0, 3 * steps)):
            assert np.array_equal(a, b)
