"""GPU: low-rank adapters of many requests (lora_add) against 64 bits."""
import numpy as np
import pytest

from mdma_amd.backend import (ACT_F32, ACT_I8, DOMAIN_DEVICE, GGML_F16, GGML_F32, GGML_Q8_0, BackendError,
                              Gfx950Backend, ShapeMismatch, NotImplemented as NotImpl)
from paged_ref import NONE, U

pytestmark = pytest.mark.gpu
CANARY = np.float32(123456.25)


def buf(be, a):
    a = np.ascontiguousarray(a)
    b = be.alloc(a.nbytes)
    be.upload(b, 0, a)
    return b


class Set:
    """An adapter set with its host copy; ranks: per slot, 0 = left empty."""

    def __init__(self, be, dtype, n_in, n_out, max_rank, ranks, seed):
        r = np.random.default_rng(seed)
        t = np.float16 if dtype == GGML_F16 else np.float32
        self.dev = be.lora(dtype, n_in, n_out, max_rank, len(ranks))
        self.host = []
        for i, k in enumerate(ranks):
            a = (r.standard_normal((k, n_in)) * n_in ** -0.5).astype(t)
            b = (r.standard_normal((n_out, k)) * 0.1).astype(t)
            self.host.append((a, b, float(np.float32(r.uniform(0.5, 2)))))
            if k:
                self.dev.load(i, *self.host[-1])

    def want(self, ids, x, base):
        """(y, tolerance): u is a sum of n_in f32 products, off by n_in u of sum|a x| at most in any order, the
        second sum by another (rank + 2) u and the last step by 2 u of what it adds."""
        y, tol = base.astype(np.float64), np.zeros(base.shape)
        for t, i in enumerate(ids):
            if i >= len(self.host) or not len(self.host[i][0]):
                continue
            a, b, s = (np.asarray(v, np.float64) for v in self.host[i])
            X = x[t].astype(np.float64)
            y[t] += s * (b @ (a @ X))
            size = s * (np.abs(b) @ (np.abs(a) @ np.abs(X)))
            tol[t] = (x.shape[1] + a.shape[0] + 8) * U * size + 2 * U * (np.abs(base[t]) + np.abs(y[t]))
        return y, tol


def run(be, st, ids, x, base, in_place=False):
    n = base.size
    bb = buf(be, np.concatenate([base.reshape(-1), np.full(64, CANARY, np.float32)]))
    yb = bb if in_place else be.f32_buf(np.full(n + 64, CANARY, np.float32))
    be.lora_add(st.dev, buf(be, np.asarray(ids, np.uint32)), buf(be, x), bb, yb)
    y = be.download_f32(yb)
    assert np.all(y[n:] == CANARY)
    if not in_place:
        assert np.array_equal(be.download_f32(bb)[:n], base.reshape(-1))
    return y[:n].reshape(base.shape)


def check(be, dtype, n_in, n_out, max_rank, ranks, ids, seed=1, in_place=False):
    st = Set(be, dtype, n_in, n_out, max_rank, ranks, seed)
    r = np.random.default_rng(seed + 1)
    x = (r.standard_normal((len(ids), n_in)) * (1 + 14 * (r.random(n_in) < 0.01))).astype(np.float32)
    base = r.standard_normal((len(ids), n_out)).astype(np.float32)
    got = run(be, st, ids, x, base, in_place)
    want, tol = st.want(ids, x, base)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
    bare = [t for t, i in enumerate(ids) if i >= len(ranks) or not ranks[i]]
    assert np.array_equal(got[bare].view(np.uint32), base[bare].view(np.uint32))
    # On the whole: roundings of random sign, u sqrt(n_in) of the products' own size.
    d, dw = got.astype(np.float64) - base, want - base
    if len(bare) < len(ids):
        assert np.linalg.norm(d - dw) <= 4 * U * ((np.sqrt(n_in) + 8) * np.linalg.norm(dw) + np.linalg.norm(base) +
                                                  np.linalg.norm(want))
    return st, got


SHAPES = [(32, 8), (288, 288), (257, 33), (1, 1), (7, 130), (1024, 515), (4096, 1024), (640, 4096)]


@pytest.mark.parametrize("dtype", [GGML_F16, GGML_F32])
@pytest.mark.parametrize("n_in,n_out", SHAPES)
@pytest.mark.parametrize("tokens", [1, 2, 17, 64, 65, 130])
def test_lora_add(backend, dtype, n_in, n_out, tokens):
    ranks = [4, 0, 16, 13, 1, 33]
    r = np.random.default_rng(tokens)
    ids = r.choice([0, 1, 2, 3, 4, 5, 6, NONE], tokens)
    check(backend, dtype, n_in, n_out, 33, ranks, ids, seed=tokens, in_place=tokens % 2 == 0)


@pytest.mark.parametrize("dtype", [GGML_F16, GGML_F32])
@pytest.mark.parametrize("rank,max_rank", [(1, 1), (15, 16), (16, 16), (64, 64), (100, 256), (256, 256)])
def test_ranks(backend, dtype, rank, max_rank):
    check(backend, dtype, 512, 384, max_rank, [rank, rank], [0, 1, 0, NONE, 1])


@pytest.mark.parametrize("dtype", [GGML_F16, GGML_F32])
@pytest.mark.parametrize("tokens,pattern", [(1000, "one"), (1000, "runs"), (777, "mixed"), (300, "bare"), (64, "each"),
                                            (63, "each"), (100, "each"), (2049, "runs")])
def test_many_tokens(backend, dtype, tokens, pattern):
    slots = 100 if pattern == "each" else 4
    r = np.random.default_rng(3)
    ids = {"one": np.full(tokens, 2), "runs": np.arange(tokens) * slots // tokens,
           "mixed": r.integers(0, slots + 1, tokens), "bare": np.full(tokens, NONE),
           "each": r.permutation(slots)[:tokens]}[pattern]
    check(backend, dtype, 320, 200, 32, [8 + i % 25 for i in range(slots)], ids, seed=tokens)


@pytest.mark.parametrize("counts", [(17, 17, 1), (1, 1, 1), (16, 16, 16), (33, 1, 17), (81, 81, 81), (1, 0, 255),
                                    (49, 129, 65), (0, 256, 0)])
def test_groups_of_an_adapter_that_are_not_full(backend, counts):
    """Tokens of two adapters and of none, as many of each as these, in runs and mixed."""
    ids = np.repeat(np.array([0, 1, NONE], np.uint32), counts)
    check(backend, GGML_F16, 96, 130, 8, [8, 5], ids, seed=3)
    check(backend, GGML_F16, 96, 130, 8, [8, 5], np.random.default_rng(4).permutation(ids), seed=3)


@pytest.mark.parametrize("seed", range(30))
def test_any_sizes(backend, seed):
    """Sizes, ranks and who has which adapter drawn at random."""
    r = np.random.default_rng(2000 + seed)
    n_in, n_out = (int(np.exp(r.uniform(0, np.log(3000)))) for _ in range(2))
    tokens = int(np.exp(r.uniform(0, np.log(700))))
    top = int(r.choice([1, 7, 16, 17, 32, 33, 64, 65, 130, 256]))
    ranks = [int(k) for k in r.integers(0, top + 1, int(r.integers(1, 9)))]
    ids = r.choice(list(range(len(ranks) + 1)) + [NONE], tokens)
    if r.random() < 0.5:
        ids = np.sort(ids)
    check(backend, GGML_F16 if r.random() < 0.6 else GGML_F32, n_in, n_out, top, ranks, ids, seed=seed,
          in_place=bool(r.random() < 0.5))


@pytest.mark.parametrize("tokens", [256, 257, 300, 1000, 1023, 1024, 1025])
@pytest.mark.parametrize("slots", [1, 3, 40, 700])
def test_mixed_requests_same_call_same_bits(backend, tokens, slots):
    """Every token another request's, around the sizes at which groups are found another way."""
    r = np.random.default_rng(tokens + slots)
    ranks = [int(k) for k in r.integers(0, 9, slots)]
    ids = r.choice(list(range(slots)) + [NONE], tokens)
    st, got = check(backend, GGML_F16, 64, 70, 8, ranks, ids, seed=slots)
    x, base = r.standard_normal((tokens, 64), np.float32), r.standard_normal((tokens, 70), np.float32)
    a, b = (run(backend, st, ids, x, base) for _ in range(2))
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_most_tokens_of_a_call(backend):
    """2^19 tokens; one more is refused."""
    T, r = 1 << 19, np.random.default_rng(3)
    st = Set(backend, GGML_F16, 8, 8, 4, [4, 2, 0], 5)
    ids = r.choice([0, 1, 2, NONE], T).astype(np.uint32)
    x, base = (r.standard_normal((T, 8), np.float32) for _ in range(2))
    got = run(backend, st, ids, x, base)
    at = np.concatenate([np.arange(40), r.integers(0, T, 200), np.arange(T - 40, T)])
    want, tol = st.want(ids[at], x[at], base[at])
    assert np.all(np.abs(got[at] - want) <= tol)
    bare = ids >= 2
    assert np.array_equal(got[bare].view(np.uint32), base[bare].view(np.uint32))
    n = T + 1
    with pytest.raises(BackendError) as e:
        backend.lora_add(st.dev, backend.alloc(4 * n), backend.alloc(32 * n), backend.alloc(32 * n), backend.alloc(32 * n))
    assert "2^19" in str(e.value)


def test_token_alone_and_in_a_batch(backend):
    """A token's result in a batch of 40 against the same token alone: both within the bound, and the same call twice
    the same bits."""
    st, _ = check(backend, GGML_F16, 512, 256, 16, [16, 8], [0])
    r = np.random.default_rng(5)
    x, base = r.standard_normal((40, 512)).astype(np.float32), r.standard_normal((40, 256)).astype(np.float32)
    ids = r.integers(0, 2, 40)
    want, tol = st.want(ids, x, base)
    all_ = run(backend, st, ids, x, base)
    assert np.array_equal(all_, run(backend, st, ids, x, base))
    for mode in (ACT_I8, ACT_F32):
        backend.set_act_mode(mode)
        try:
            assert np.array_equal(all_, run(backend, st, ids, x, base))
        finally:
            backend.set_act_mode(ACT_F32)
    for t in (0, 17, 39):
        got = run(backend, st, ids[t:t + 1], x[t:t + 1], base[t:t + 1])
        assert np.all(np.abs(got - want[t:t + 1]) <= tol[t:t + 1])


@pytest.mark.parametrize("dtype", [GGML_F16, GGML_F32])
@pytest.mark.parametrize("tokens", [5, 90])
def test_values_that_are_not_finite_stay_in_their_token(backend, dtype, tokens):
    st, _ = check(backend, dtype, 100, 70, 8, [3, 8], [0])
    r = np.random.default_rng(5)
    x, base = r.standard_normal((tokens, 100)).astype(np.float32), r.standard_normal((tokens, 70)).astype(np.float32)
    ids = np.arange(tokens) % 2
    x[1, 3], x[2, 50], base[3, 7] = np.nan, np.inf, -np.inf
    got = run(backend, st, ids, x, base)
    with np.errstate(invalid="ignore"):
        want, tol = st.want(ids, x, base)
    for t in range(tokens):
        if t in (1, 2):
            assert not np.isfinite(got[t]).any() and np.array_equal(np.isnan(got[t]), np.isnan(want[t]))
        else:
            ok = np.isfinite(want[t])
            assert np.all(np.abs(got[t] - want[t])[ok] <= tol[t][ok])
            assert np.array_equal(got[t][~ok], want[t][~ok])


def test_slots_loaded_again_and_emptied(backend):
    st, _ = check(backend, GGML_F16, 96, 64, 32, [32, 5], [0, 1])
    r = np.random.default_rng(8)
    x, base = r.standard_normal((3, 96)).astype(np.float32), r.standard_normal((3, 64)).astype(np.float32)
    a, b = r.standard_normal((2, 96)).astype(np.float16), r.standard_normal((64, 2)).astype(np.float16)
    st.host[0] = (a, b, 0.5)
    st.dev.load(0, a, b, 0.5)
    want, tol = st.want([0, 1, 0], x, base)
    assert np.all(np.abs(run(backend, st, [0, 1, 0], x, base) - want) <= tol)
    st.dev.load(1, None, None)
    got = run(backend, st, [0, 1, 0], x, base)
    assert np.array_equal(got[1], base[1]) and np.all(np.abs(got - want)[[0, 2]] <= tol[[0, 2]])


def test_beside_the_shared_projection_captured(backend):
    """qmatmul and lora_add in place on its output, captured; the ids change between the replays."""
    from mdma_amd import synth

    n_in, n_out, T = 288, 96, 6
    w = backend.upload_weight(synth.weight(GGML_Q8_0, n_out, n_in, 1), GGML_Q8_0, (n_out, n_in))
    st, _ = check(backend, GGML_F16, n_in, n_out, 16, [16, 3, 8], [0])
    ids, x, y = backend.alloc(4 * T), backend.alloc(4 * T * n_in), backend.alloc(4 * T * n_out)

    def step():
        backend.qmatmul(w, x, y)
        backend.lora_add(st.dev, ids, x, y, y)

    r = np.random.default_rng(2)
    backend.upload(ids, 0, np.full(T, NONE, np.uint32))
    backend.upload(x, 0, r.standard_normal(T * n_in).astype(np.float32))
    step()
    backend.join_execution()
    g = backend.capture(step)
    for i in range(6):
        who, X = r.integers(0, 4, T).astype(np.uint32), r.standard_normal((T, n_in)).astype(np.float32)
        backend.upload(ids, 0, who)
        backend.upload(x, 0, X)
        g.launch()
        got = backend.download_f32(y).reshape(T, n_out)
        base = backend.alloc(4 * T * n_out)
        backend.qmatmul(w, x, base)
        base = backend.download_f32(base).reshape(T, n_out)
        want, tol = st.want(who, X, base)
        assert np.all(np.abs(got - want) <= tol), i
    g.close()


def test_refusals(backend):
    st, _ = check(backend, GGML_F16, 64, 32, 8, [8], [0])
    ids, x, y = backend.alloc(12), backend.alloc(3 * 64 * 4), backend.alloc(3 * 32 * 4)
    backend.upload(ids, 0, np.zeros(3, np.uint32))
    for bad in (lambda: backend.lora_add(st.dev, backend.alloc(8), x, y, y),
                lambda: backend.lora_add(st.dev, ids, backend.alloc(3 * 64 * 4 - 4), y, y),
                lambda: backend.lora_add(st.dev, ids, x, backend.alloc(8), y),
                lambda: backend.lora_add(st.dev, ids, x, y, backend.alloc(8)),
                lambda: backend.lora_add(st.dev, ids, x, y, x),
                lambda: st.dev.load(1, np.zeros((8, 64)), np.zeros((32, 8))),
                lambda: st.dev.load(0, np.zeros((9, 64)), np.zeros((32, 9))),
                lambda: st.dev.load(0, np.zeros((8, 63)), np.zeros((32, 8))),
                lambda: backend.lora(GGML_F16, 64, 32, 257, 1), lambda: backend.lora(GGML_F16, 0, 32, 8, 1)):
        with pytest.raises(ShapeMismatch):
            bad()
    with pytest.raises(NotImpl):
        backend.lora(GGML_Q8_0, 64, 32, 8, 1)
    other = Gfx950Backend(0)
    try:
        with pytest.raises(ShapeMismatch):
            other.lora_add(st.dev, ids, x, y, y)
    finally:
        other.close()


def test_set_is_charged_to_the_budget():
    be = Gfx950Backend(0)
    try:
        be.set_buffer_budget(device=64 << 10)
        with pytest.raises(BackendError) as e:
            be.lora(GGML_F16, 4096, 4096, 64, 4)
        assert e.value.code == 6 and be.buffer_usage(DOMAIN_DEVICE)[0] == 0
        st = be.lora(GGML_F32, 64, 64, 16, 2)
        assert be.buffer_usage(DOMAIN_DEVICE)[0] == 2 * 2 * 64 * 16 * 4 + 2 * 12
        st.close()
        assert be.buffer_usage(DOMAIN_DEVICE)[0] == 0
    finally:
        be.close()
