"""Performance cases of the operators that serve a batch of requests: attention over a paged KV cache with a shared
prefix (`Gfx950Backend.attn_paged`), the cache's writes (`rope_kv_write_paged`), its page tables (`kv_pages_fork`,
`kv_pages_grow`, `kv_pages_compact`) and the requests' low-rank adapters (`lora_add`).

Each case is one call (or two that belong together) as a decode or prompt step makes it. Where `own` is false the
same results come from elementary torch operations in 32 bits. Geometries are those of `mdma_amd.llama_synth`
(TinyStories-15M, Llama-3-8B) and generic ones between them.
"""
import math
import random

import numpy as np
import torch

own = False

NONE = -1  # a table entry that names no page, an id that names no sequence or adapter (0xffffffff)
LAYER = 1  # the layer that attention and writes use, of two


# ---- cases ----

def _attn(name, **c):
    return dict(dict(name=name) if name else {}, kind="attn", **c)


def _write(name, **c):
    return dict(dict(name=name) if name else {}, kind="write", **c)


def _fork(name, **c):
    return dict(dict(name=name) if name else {}, kind="fork", **c)


def _compact(name, **c):
    return dict(dict(name=name) if name else {}, kind="compact", **c)


def _lora(name, **c):
    return dict(dict(name=name) if name else {}, kind="lora", **c)


def listed():
    return [
        # The smallest step: three short chats on the TinyStories-15M geometry, nothing shared, one token each.
        _attn("attn_tiny", seqs=3, new=1, prefix=0, own_lo=17, own_hi=200, empty=0, page=16, heads=6, kv_heads=6,
              head_dim=48, pattern=1),
        # A long system prompt shared by 64 chats of a Llama-3-8B geometry, one token each: the largest.
        _attn("attn_shared_prompt", seqs=64, new=1, prefix=16384, own_lo=100, own_hi=1000, empty=0, page=64, heads=32,
              kv_heads=8, head_dim=128, pattern=2),
        # Five drafted tokens per sequence to verify, ragged contexts up to 4096, nothing shared, a padded batch
        # with two empty slots.
        _attn("attn_verify5_ragged", seqs=16, new=5, prefix=0, own_lo=5, own_hi=4096, empty=2, page=32, heads=32,
              kv_heads=8, head_dim=128, pattern=3),
        # One decode step's new rows of eight sequences at their own positions.
        _write("write_decode8", seqs=8, new=1, lo=40, hi=4000, empty=1, page=16, heads=32, kv_heads=8, head_dim=128,
               theta=500000.0, pattern=4),
        # Four prompts' new rows.
        _write("write_prompts", seqs=4, new=509, lo=509, hi=2048, empty=0, page=64, heads=32, kv_heads=8,
               head_dim=128, theta=500000.0, pattern=5),
        # A decode step's bookkeeping of eight unrelated sequences on a small cache: nothing forks, some get a page.
        _fork("grow_decode8", seqs=8, fan=1, keep_lo=50, keep_hi=500, new=1, layers=2, page=16, width=1024, pattern=6),
        # Beam search, 8 requests of 8 beams: every beam continues its request's first one, a new token each, so
        # shared last pages are copied in all layers.
        _fork("fork_beams8x8", seqs=64, fan=8, keep_lo=300, keep_hi=700, new=1, layers=8, page=16, width=1024,
              pattern=7),
        # A small cache after a few requests ended.
        _compact("compact_small", pages=200, live=0.6, seqs=8, layers=2, page=16, width=288, pattern=8),
        # A large cache after half of its requests ended.
        _compact("compact_large", pages=2048, live=0.5, seqs=32, layers=4, page=16, width=1024, pattern=9),
        # One token with one small f32 adapter on the TinyStories-15M width.
        _lora("lora_tiny", tokens=1, n_in=288, n_out=288, dtype="f32", slots=2, used=1, rank=4, runs=False, bare=0,
              pattern=10),
        # One decode step of 32 requests with 16 adapters, beside a Llama-3-8B gate projection.
        _lora("lora_decode32", tokens=32, n_in=4096, n_out=14336, dtype="f16", slots=24, used=16, rank=64, runs=False,
              bare=7, pattern=11),
        # Prompts of three requests, two with adapters, 2000 token rows.
        _lora("lora_prompts2000", tokens=2000, n_in=4096, n_out=4096, dtype="f16", slots=8, used=2, rank=32,
              runs=True, bare=3, pattern=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (32, 8, 128), (6, 6, 48), (32, 32, 64), (20, 20, 128), (28, 4, 128), (16, 1, 256), (24, 8, 80)]


def draw(rng):
    kind = rng.choice(["attn"] * 4 + ["lora"] * 3 + ["write", "fork", "compact"])
    pattern = rng.randrange(1, 1 << 20)
    if kind == "attn":
        heads, kv_heads, head_dim = rng.choice(HEADS)
        page, new = rng.choice([16, 32, 64, 128]), rng.choice([1, 1, 1, 2, 4, 7])
        seqs = _log_int(rng, 1, 48)
        room = 60000 * 1024 // (kv_heads * head_dim)  # positions, all sequences together
        prefix = rng.choice([0, 1]) * _log_int(rng, 64, 12000) // page * page
        hi = max(new + 1, min(4000, (room - prefix) // seqs))
        if seqs * (prefix + hi) > 800000:
            prefix = 0
        return _attn(None, seqs=seqs, new=new, prefix=prefix, own_lo=new, own_hi=_log_int(rng, new + 1, hi),
                     empty=rng.choice([0, 0, 1]) if seqs > 1 else 0, page=page, heads=heads, kv_heads=kv_heads,
                     head_dim=head_dim, pattern=pattern)
    if kind == "write":
        heads, kv_heads, head_dim = rng.choice(HEADS)
        seqs = _log_int(rng, 1, 32)
        new = _log_int(rng, 1, 2000 // seqs)
        return _write(None, seqs=seqs, new=new, lo=new, hi=new + _log_int(rng, 1, 1500), empty=rng.choice([0, 1]),
                      page=rng.choice([16, 32, 64]), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                      theta=rng.choice([10000.0, 500000.0]), pattern=pattern)
    if kind == "fork":
        fan = rng.choice([1, 2, 3, 4, 8])
        lo = _log_int(rng, 1, 300)
        return _fork(None, seqs=fan * rng.randrange(1, 9), fan=fan, keep_lo=lo, keep_hi=lo + _log_int(rng, 1, 300),
                     new=rng.choice([1, 1, 5, 40]), layers=rng.choice([1, 2, 5]), page=rng.choice([16, 32, 64]),
                     width=rng.choice([256, 288, 512, 1024]), pattern=pattern)
    if kind == "compact":
        return _compact(None, pages=_log_int(rng, 30, 1500), live=round(rng.uniform(0.2, 0.95), 3),
                        seqs=rng.randrange(1, 40), layers=rng.choice([1, 2, 4]), page=rng.choice([16, 32]),
                        width=rng.choice([256, 288, 512]), pattern=pattern)
    n_in, n_out = rng.choice([(288, 288), (288, 768), (2048, 2048), (2560, 6912), (4096, 1024), (4096, 4096),
                              (4096, 14336), (14336, 4096)])
    tokens = _log_int(rng, 1, 1500)
    slots = rng.choice([2, 8, 20])
    return _lora(None, tokens=tokens, n_in=n_in, n_out=n_out, dtype=rng.choice(["f16", "f16", "f16", "f32"]),
                 slots=slots, used=rng.randrange(1, min(slots, tokens) + 1), rank=rng.choice([4, 8, 13, 16, 32, 64]),
                 runs=tokens > 64, bare=rng.choice([0, 0, 5]), pattern=pattern)


# ---- what a case fixes besides its sizes: lengths, tables, which token has which adapter ----

def _lens(c):
    """Positions of every sequence; the empty slots are spread over the batch, the first one among them."""
    r = random.Random(c["pattern"])
    if c["kind"] == "attn":
        lens = [c["prefix"] + _log_int(r, c["own_lo"], c["own_hi"]) for _ in range(c["seqs"])]
    else:
        lens = [_log_int(r, c["lo"], c["hi"]) for _ in range(c["seqs"])]
    for e in range(min(c["empty"], c["seqs"] - 1)):
        lens[e * c["seqs"] // c["empty"]] = 0
    return lens


def _pages_of(n, page):
    return -(-n // page)


def _tables(c):
    """(table [seqs][max_pages], refs, prefix page ids, lengths): pages in scattered order, the prefix's shared."""
    r = random.Random(c["pattern"] + 1)
    lens, page = _lens(c), c["page"]
    npre = c.get("prefix", 0) // page
    per = [_pages_of(n, page) for n in lens]
    total = npre + sum(max(0, n - npre) for n in per) + 3
    ids = list(range(total))
    r.shuffle(ids)
    pre, at = ids[:npre], npre
    table = np.full((c["seqs"], max(per) + 1), NONE, np.int64)
    refs = np.zeros(total, np.int64)
    for s, n in enumerate(per):
        if n:
            table[s, :npre] = pre
            table[s, npre:n] = ids[at:at + n - npre]
            at += n - npre
            refs[table[s, :n]] += 1
    return table, refs, np.array(pre, np.int64), np.array(lens, np.int64)


def _fork_tables(c):
    r = random.Random(c["pattern"])
    S, fan, page = c["seqs"], c["fan"], c["page"]
    keep = np.repeat([_log_int(r, c["keep_lo"], c["keep_hi"]) for _ in range(S // fan)], fan).astype(np.int64)
    frm = (np.arange(S) // fan * fan).astype(np.int64)
    lens = np.where(frm == np.arange(S), keep, 0)
    per = -(-lens // page)
    M = int(_pages_of(int(keep.max()) + c["new"], page)) + 1
    total = int(per.sum()) + S * (2 + _pages_of(c["new"], page)) + 2
    ids = list(range(total))
    r.shuffle(ids)
    table, refs, at = np.full((S, M), NONE, np.int64), np.zeros(total, np.int64), 0
    for s in range(S):
        table[s, :per[s]] = ids[at:at + per[s]]
        refs[table[s, :per[s]]] = 1
        at += per[s]
    return table, refs, lens, frm, keep, np.full(S, c["new"], np.int64)


def _compact_tables(c):
    r = random.Random(c["pattern"])
    P, S, page = c["pages"], c["seqs"], c["page"]
    live = [p for p in range(P) if r.random() < c["live"]]
    r.shuffle(live)
    per = [len(live) // S + (s < len(live) % S) for s in range(S)]
    table, refs, at = np.full((S, max(per) + 2), NONE, np.int64), np.zeros(P, np.int64), 0
    for s, n in enumerate(per):
        table[s, :n] = live[at:at + n]
        at += n
    refs[live] = 1
    return table, refs, np.array(per, np.int64) * page


def _adapters(c):
    """(ids per token, rank per slot): `used` slots in turn or in runs of tokens, every bare-th token without one."""
    r = random.Random(c["pattern"])
    names = r.sample(range(c["slots"]), c["used"])
    T, n = c["tokens"], c["used"] + (1 if c["bare"] and c["runs"] else 0)
    ids = [(i * n // T) if c["runs"] else i % n for i in range(T)]
    ids = [names[i] if i < c["used"] and not (c["bare"] and not c["runs"] and t % c["bare"] == c["bare"] - 1) else NONE
           for t, i in enumerate(ids)]
    ranks = [r.choice([c["rank"], c["rank"], max(1, c["rank"] // 2)]) for _ in range(c["slots"])]
    return ids, ranks


# ---- inputs, made on the GPU from the seed ----

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _pools(g, layers, pages, page, width):
    return ((_randn(g, layers, pages, page, width) * 0.8).to(torch.float16),
            _randn(g, layers, pages, page, width).to(torch.float16))


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _inputs(c, seed):
    """The case's tensors by name; integers as int64."""
    g, kind = _gen(seed), c["kind"]
    t = {}
    if kind in ("attn", "write"):
        table, refs, pre, lens = _tables(c)
        hd, H, KV = c["head_dim"], c["heads"], c["kv_heads"]
        t["k"], t["v"] = _pools(g, 2, len(refs), c["page"], KV * hd)
        t["q"] = _randn(g, c["seqs"], c["new"], H * hd) * 1.5
        t["table"], t["refs"], t["lens"], t["prefix"] = _dev(table), _dev(refs), _dev(lens), _dev(pre)
        if kind == "write":
            t["nk"], t["nv"] = (_randn(g, c["seqs"], c["new"], KV * hd) for _ in range(2))
    elif kind == "fork":
        table, refs, lens, frm, keep, grow = _fork_tables(c)
        t["k"], t["v"] = _pools(g, c["layers"], len(refs), c["page"], c["width"])
        t.update(table=_dev(table), refs=_dev(refs), lens=_dev(lens), frm=_dev(frm), keep=_dev(keep), grow=_dev(grow))
    elif kind == "compact":
        table, refs, lens = _compact_tables(c)
        t["k"], t["v"] = _pools(g, c["layers"], c["pages"], c["page"], c["width"])
        t.update(table=_dev(table), refs=_dev(refs), lens=_dev(lens))
    else:
        ids, ranks = _adapters(c)
        R, dt = max(ranks), {"f16": torch.float16, "f32": torch.float32}[c["dtype"]]
        held = _dev((np.arange(R)[None, :] < np.array(ranks)[:, None]).astype(np.float32))  # [slots, R]
        big = 1 + 14 * (torch.rand(c["n_in"], generator=g, device="cuda") < 0.005)  # a few large channels
        t["x"] = _randn(g, c["tokens"], c["n_in"]) * big
        t["base"] = _randn(g, c["tokens"], c["n_out"])
        t["a"] = (_randn(g, c["slots"], R, c["n_in"]) * c["n_in"] ** -0.5 * held[:, :, None]).to(dt)
        t["b"] = (_randn(g, c["slots"], c["n_out"], R) * 0.05 * held[:, None, :]).to(dt)
        t["ids"] = _dev(np.array(ids, np.int64))
        t["scale"] = _dev(np.array([16.0 / r for r in ranks], np.float32))
        t["ranks"] = ranks
    return t


# ---- the package's side ----

class Outputs(dict):
    """Device buffers by name, each read to the host when looked at (the calls that fill them are queued on the
    backend's stream, and a program reads a result when it needs it)."""

    def __init__(self, be, bufs):
        super().__init__(bufs)
        self.be = be

    def __getitem__(self, name):
        buf, shape, dtype = dict.__getitem__(self, name)
        return self.be.download(buf, 0, math.prod(shape) * np.dtype(dtype).itemsize).view(dtype).reshape(shape)


_backends = []


def _backend():
    from mdma_amd.backend import Gfx950Backend
    if not _backends:
        _backends.append(Gfx950Backend(0))
    return _backends[0]


def _put(be, t):
    a = t.cpu().numpy()
    a = a.astype(np.uint32) if a.dtype == np.int64 else a
    b = be.alloc(a.nbytes)
    if a.nbytes:
        be.upload(b, 0, a)
    return b


def _own_prepare(c, t):
    from mdma_amd import backend as B
    be, kind = _backend(), c["kind"]
    s = {"be": be, "c": c}
    if kind == "lora":
        dt = {"f16": B.GGML_F16, "f32": B.GGML_F32}[c["dtype"]]
        s["lora"] = be.lora(dt, c["n_in"], c["n_out"], max(t["ranks"]), c["slots"])
        a, b, scale = t["a"].cpu().numpy(), t["b"].cpu().numpy(), t["scale"].cpu().numpy()
        for i, r in enumerate(t["ranks"]):
            s["lora"].load(i, a[i, :r], b[i, :, :r], float(scale[i]))
        s.update(ids=_put(be, t["ids"]), x=_put(be, t["x"]), base=_put(be, t["base"]),
                 y=be.alloc(c["tokens"] * c["n_out"] * 4))
        s["out"] = Outputs(be, {"y": (s["y"], (c["tokens"], c["n_out"]), np.float32)})
        return s
    b = {n: _put(be, v) for n, v in t.items()}
    L, P, page, W = t["k"].shape
    S, M = t["table"].shape
    s["b"] = b
    s["pages"] = B.KvPages(b["k"], b["v"], b["table"], b["lens"], b["refs"], n_layers=L, n_pages=P, page_len=page,
                           kv_width=W, n_seqs=S, max_pages=M)
    pool = {n: (b[n], tuple(t[n].shape), np.float16) for n in "kv"}
    books = {"table": (b["table"], (S, M), np.int32), "refs": (b["refs"], (P,), np.int32),
             "lens": (b["lens"], (S,), np.int32)}
    if kind == "attn":
        s["spec"] = B.AttnSpec(c["head_dim"], c["heads"], c["kv_heads"])
        s["o"] = be.alloc(t["q"].numel() * 4)
        s["prefix"] = b["prefix"] if c["prefix"] else None
        s["out"] = Outputs(be, {"o": (s["o"], tuple(t["q"].shape), np.float32)})
    elif kind == "write":
        s["rope"] = B.RopeSpec(c["head_dim"], c["theta"])
        s["out"] = Outputs(be, dict(pool, q=(b["q"], tuple(t["q"].shape), np.float32)))
    elif kind == "fork":
        s["status"] = be.alloc(S * 4)
        s["out"] = Outputs(be, dict(pool, **books, status=(s["status"], (S,), np.int32)))
    else:
        s["snap"] = {n: _put(be, t[n]) for n in ("table", "refs")}
        s["live"] = be.alloc(4)
        s["out"] = Outputs(be, dict(pool, **books, live=(s["live"], (1,), np.int32)))
    return s


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        return _own_prepare(case, t)
    if case["kind"] == "compact":
        t["snap"] = {n: t[n].clone() for n in ("table", "refs")}
    return {"c": case, "t": t}


def _own_run(s):
    be, kind = s["be"], s["c"]["kind"]
    if kind == "attn":
        be.attn_paged(s["b"]["q"], s["pages"], LAYER, s["prefix"], s["spec"], s["o"])
    elif kind == "write":
        be.rope_kv_write_paged(s["b"]["q"], s["b"]["nk"], s["b"]["nv"], s["pages"], LAYER, s["rope"])
    elif kind == "fork":
        be.kv_pages_fork(s["pages"], s["b"]["frm"], s["b"]["keep"])
        be.kv_pages_grow(s["pages"], s["b"]["grow"], s["status"])
    elif kind == "compact":
        for n, buf in s["snap"].items():  # back to the tables before: as the program finds them
            be.copy(buf, 0, s["b"][n], 0, buf.len)
        be.kv_pages_compact(s["pages"], s["live"])
    else:
        be.lora_add(s["lora"], s["ids"], s["x"], s["base"], s["y"])
    return s["out"]


# ---- the plain forms ----

def _gather(pool, table, kv_heads, hd):
    """[seqs * kv_heads, positions, hd] in 32 bits; entries that name no page give some page (masked later)."""
    rows = pool[table.clamp(min=0)]  # [S, M, page, W]
    S, M, page, _ = rows.shape
    return rows.float().view(S, M * page, kv_heads, hd).permute(0, 2, 1, 3).reshape(S * kv_heads, M * page, hd)


def _positions(lens, new):
    """Positions of each sequence's new tokens, [seqs, new]: the last of its lens; below 0: no such token."""
    return lens[:, None] - new + torch.arange(new, device=lens.device)


def _plain_attn(c, t):
    S, n, H, KV, hd = c["seqs"], c["new"], c["heads"], c["kv_heads"], c["head_dim"]
    G = H // KV
    q = t["q"].view(S, n, KV, G, hd).permute(0, 2, 1, 3, 4).reshape(S * KV, n * G, hd)
    sc = torch.bmm(q, _gather(t["k"][LAYER], t["table"], KV, hd).transpose(1, 2).contiguous()) * hd ** -0.5
    N = sc.shape[-1]
    seen = torch.arange(N, device=sc.device) <= _positions(t["lens"], n)[:, :, None]  # [S, n, N]
    sc = sc.view(S, KV, n, G, N).masked_fill(~seen[:, None, :, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, torch.zeros_like(m), m))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-37)
    o = torch.bmm(p.view(S * KV, n * G, N), _gather(t["v"][LAYER], t["table"], KV, hd))
    return {"o": o.view(S, KV, n, G, hd).permute(0, 2, 1, 3, 4).reshape(S, n, H * hd)}


def _angles(pos, hd, theta):
    """The framework's angles (`rope`): position times the frequency, each and the frequency's exponent rounded to 32
    bits; their cosine and sine."""
    f = (theta ** (-torch.arange(0, hd, 2, device=pos.device).float() / hd).double()).float()
    a = (pos.clamp(min=0).float()[..., None] * f).double()
    return torch.cos(a).float(), torch.sin(a).float()


def _rotate(x, cos, sin, hd):
    p = x.view(*x.shape[:-1], -1, hd // 2, 2)
    a, b, cos, sin = p[..., 0], p[..., 1], cos[:, :, None], sin[:, :, None]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).view(x.shape)


def _plain_write(c, t):
    hd, page = c["head_dim"], c["page"]
    pos = _positions(t["lens"], c["new"])
    there = pos >= 0
    cos, sin = _angles(pos, hd, c["theta"])
    t["q"].copy_(torch.where(there[..., None], _rotate(t["q"], cos, sin, hd), t["q"]))
    ids = torch.gather(t["table"], 1, (pos.clamp(min=0) // page))[there]
    rows = (pos % page)[there]
    t["k"][LAYER, ids, rows] = _rotate(t["nk"], cos, sin, hd)[there].to(torch.float16)
    t["v"][LAYER, ids, rows] = t["nv"][there].to(torch.float16)
    return {"q": t["q"], "k": t["k"], "v": t["v"]}


def _plain_fork(c, t):
    page, S, M = c["page"], *t["table"].shape
    P = t["refs"].numel()
    # fork: every row a copy of the first keep positions of the row that it comes from
    lens = torch.minimum(t["keep"], t["lens"][t["frm"]])
    table = t["table"][t["frm"]]
    table = torch.where(torch.arange(M, device=lens.device) < ((lens + page - 1) // page)[:, None], table,
                        torch.full_like(table, NONE))
    flat = table.reshape(-1)
    refs = torch.zeros(P + 1, dtype=torch.int64, device=lens.device)
    refs.index_add_(0, torch.where(flat < 0, P, flat), torch.ones_like(flat))
    refs = refs[:P]
    # grow: a last page that others hold too is copied, further pages follow; the lowest free ids, in order
    grow = t["grow"]
    before, after = (lens + page - 1) // page, (lens + grow + page - 1) // page
    grows = (grow > 0) & (after <= M)
    at = (before - 1).clamp(min=0)[:, None]
    last = torch.gather(table, 1, at)[:, 0]
    part = grows & (lens % page != 0)
    i = torch.arange(S, device=lens.device)
    earlier = ((last[:, None] == last[None, :]) & part[:, None] & part[None, :] & (i[None, :] < i[:, None])).sum(1)
    cow = part & (earlier < refs[last.clamp(min=0)] - 1)
    need = torch.where(grows, cow + after - before, torch.zeros_like(lens))
    end = need.cumsum(0)
    free = torch.nonzero(refs == 0)[:, 0]
    fits = grows & (end <= free.numel())
    status = torch.where((grow > 0) & ~fits, torch.where(after > M, 2, 1), 0)
    cow = cow & fits
    free = torch.cat([free, free.new_zeros(int(S * M) + 1)])
    start = end - need
    src, dst = last[cow], free[start[cow]]
    refs.index_add_(0, src, -torch.ones_like(src))
    table.scatter_(1, at, torch.where(cow, free[start], last)[:, None])
    e = torch.arange(M, device=lens.device) - before[:, None]
    new = (e >= 0) & (e < (after - before)[:, None]) & fits[:, None]
    table = torch.where(new, free[(start + cow)[:, None] + e.clamp(min=0)], table)
    refs.index_add_(0, torch.cat([dst, table[new]]), torch.ones(dst.numel() + int(new.sum()), dtype=torch.int64,
                                                                device=lens.device))
    held = (torch.arange(page, device=lens.device) < (lens % page)[cow][:, None])[None, :, :, None]
    for pool in (t["k"], t["v"]):
        pool[:, dst] = torch.where(held, pool[:, src], pool[:, dst])
    t["table"].copy_(table)
    t["refs"].copy_(refs)
    t["lens"].copy_(torch.where(fits, lens + grow, lens))
    return dict(_books(t), status=status.to(torch.int32))


def _books(t):
    return {"k": t["k"], "v": t["v"], **{n: t[n].to(torch.int32) for n in ("table", "refs", "lens")}}


def _plain_compact(c, t):
    for n, x in t["snap"].items():
        t[n].copy_(x)
    table, refs = t["table"], t["refs"]
    live = refs > 0
    n = live.sum()
    ids = torch.arange(refs.numel(), device=refs.device)
    src, dst = torch.nonzero(live & (ids >= n))[:, 0], torch.nonzero(~live & (ids < n))[:, 0]
    ids[src] = dst
    table.copy_(torch.where(table < 0, table, ids[table.clamp(min=0)]))
    refs[dst] = refs[src]
    refs[src] = 0
    for pool in (t["k"], t["v"]):
        pool[:, dst] = pool[:, src]
    return dict(_books(t), live=n[None].to(torch.int32))


def _plain_lora(c, t):
    slots, R, _ = t["a"].shape
    mine = torch.arange(slots, device="cuda")[None, :] == t["ids"][:, None]  # [T, slots]
    u = t["x"] @ t["a"].float().view(slots * R, -1).t()
    u = u.view(-1, slots, R) * (mine * t["scale"])[:, :, None]
    b = t["b"].float().permute(0, 2, 1).reshape(slots * R, -1)
    return {"y": t["base"] + u.view(-1, slots * R) @ b}


_PLAIN = {"attn": _plain_attn, "write": _plain_write, "fork": _plain_fork, "compact": _plain_compact,
          "lora": _plain_lora}


def run(s):
    return _own_run(s) if own else _PLAIN[s["c"]["kind"]](s["c"], s["t"])


# ---- what a pass cannot do without ----

def work(case):
    c, kind = case, case["kind"]
    if kind == "lora":
        ids, ranks = _adapters(c)
        eb, io = {"f16": 2, "f32": 4}[c["dtype"]], c["n_in"] + c["n_out"]
        with_one = [ranks[i] for i in ids if i >= 0]
        return {"bytes": eb * io * sum(ranks[i] for i in set(ids) if i >= 0) + 4.0 * len(with_one) * c["n_in"] +
                8.0 * c["tokens"] * c["n_out"], "flops": 2.0 * io * sum(with_one)}
    if kind == "fork":
        _, refs, _, _, keep, grow = _fork_tables(c)
        rows = sum(int(k) % c["page"] for i, k in enumerate(keep) if i % c["fan"])  # all of a group but one copy
        return {"bytes": 8.0 * rows * c["width"] * c["layers"] + 8.0 * len(refs) + 24.0 * c["seqs"], "flops": 0}
    if kind == "compact":
        table, refs, _ = _compact_tables(c)
        moved = int((refs[int((refs > 0).sum()):] > 0).sum())
        return {"bytes": 8.0 * moved * c["page"] * c["width"] * c["layers"] + 8.0 * table.size + 8.0 * refs.size,
                "flops": 0}
    lens, H, W, n = _lens(c), c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"], c["new"]
    rows = sum(min(n, x) for x in lens)
    if kind == "write":
        return {"bytes": 8.0 * rows * H + 12.0 * rows * W, "flops": 3.0 * rows * (H + W)}
    held = c["prefix"] + sum(max(0, x - c["prefix"]) for x in lens)
    pairs = sum(sum(x - j for j in range(min(n, x))) for x in lens)
    return {"bytes": 4.0 * held * W + 8.0 * c["seqs"] * n * H, "flops": 4.0 * pairs * H}


# ---- the same results in 64 bits ----

def _exact_attn(c, t):
    S, n, H, KV, hd, page = c["seqs"], c["new"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    out = torch.zeros(S, n, H, hd, dtype=torch.float64, device="cuda")
    for s, N in enumerate(t["lens"].tolist()):
        if not N:
            continue
        ids = t["table"][s, :_pages_of(N, page)]
        k, v = (t[x][LAYER][ids].double().reshape(-1, KV, hd)[:N] for x in "kv")
        for j in range(max(0, n - N), n):
            end = N - n + j + 1
            for h in range(KV):
                q = t["q"][s, j].double().view(KV, -1, hd)[h]
                w = torch.softmax(q @ k[:end, h].t().contiguous() / math.sqrt(hd), -1)
                out[s, j].view(KV, -1, hd)[h] = w @ v[:end, h]
    return {"o": out.view(S, n, H * hd).cpu().numpy()}


def _exact_write(c, t):
    hd, page, n = c["head_dim"], c["page"], c["new"]
    f = np.array([np.float32(c["theta"] ** float(np.float32(-2.0 * i / hd))) for i in range(hd // 2)], np.float32)
    q, nk, nv = (t[x].cpu().numpy().astype(np.float64) for x in ("q", "nk", "nv"))
    k, v = (t[x].cpu().numpy().astype(np.float64) for x in "kv")
    table = t["table"].cpu().numpy()
    for s, N in enumerate(t["lens"].tolist()):
        for j in range(max(0, n - N), n):
            p = N - n + j
            z = np.exp(1j * (np.float32(p) * f).astype(np.float64))  # a rotation of each pair
            for x in (q, nk):
                w = (x[s, j].reshape(-1, hd // 2, 2) @ np.array([1, 1j])) * z
                x[s, j] = np.stack([w.real, w.imag], -1).reshape(-1)
            k[LAYER, table[s, p // page], p % page] = nk[s, j]
            v[LAYER, table[s, p // page], p % page] = nv[s, j]
    return {"q": q, "k": k, "v": v}


def _exact_lora(c, t):
    y = t["base"].double()
    for i in set(t["ids"].tolist()) - {NONE}:
        at = torch.nonzero(t["ids"] == i)[:, 0]
        u = t["x"][at].double() @ t["a"][i].double().t().contiguous()
        y[at] += t["scale"][i].double() * (u @ t["b"][i].double().t().contiguous())
    return {"y": y.cpu().numpy()}


def exact(case, seed):
    form = {"attn": _exact_attn, "write": _exact_write, "lora": _exact_lora}.get(case["kind"])
    return form(case, _inputs(case, seed)) if form else None
