"""Accumulated attention weights and eviction by them on the GPU, against plain 64-bit forms."""
import math
import random

import pytest

from tests.paged_reference import attention, close, rope_freqs, rotated

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pg(torch_gpu):
    from mechta_amd import paged
    return paged


def given(torch, q, k, pos0, scale, window=0, sinks=None):
    """What tokens q [t, q_heads, d] at positions pos0 .. give to each of the keys k [n, kv_heads, d], [kv_heads, n], in 64
    bits, and the tolerance. A score's error is that of head_dim products and sums in f32, of its scaling and of the exponent's
    difference (2^-22 of the largest magnitudes each), and moves a weight by that factor, once by itself and once through the
    row's sum; the exponentials, the reciprocal and the product add 2^-20; sums over n keys and over the rows add a rounding
    of 2^-24 a term at most."""
    t, heads, d = q.shape
    n, kv_heads = k.shape[:2]
    group = heads // kv_heads
    p = torch.arange(pos0, pos0 + t, device=q.device)[:, None]
    j = torch.arange(n, device=q.device)[None]
    seen = (j <= p) & ((j > p - window) if window else (j >= 0))
    out = torch.zeros(kv_heads, n, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for h in range(heads):
        kk = k[:, h // group].double()
        fine = torch.nan_to_num(kk, 0.0, 0.0, 0.0)
        x = scale * (q[:, h].double() @ kk.T.contiguous())
        x = x.masked_fill(~seen, -math.inf)
        size = (scale * (q[:, h].double().abs() @ fine.abs().T.contiguous())).masked_fill(~seen, 0.0).amax(1, keepdim=True)
        top = x.amax(1, keepdim=True)
        if sinks is not None:
            top = torch.maximum(top, sinks[h].double())
        w = torch.exp(x - top)
        total = w.sum(1, keepdim=True)
        if sinks is not None:
            total = total + torch.exp(sinks[h].double() - top)
        w = (w / total).masked_fill(~seen, 0.0)
        ds = size * (d + 8) * 2.0 ** -24 + top.abs() * 2.0 ** -22
        out[h // group] += w.sum(0)
        tol[h // group] += (w * (2 * ds + n * 2.0 ** -24 + 2.0 ** -20)).sum(0)
    return out, tol + out * (t * group) * 2.0 ** -24 + 1e-30


class Model:
    """A one-layer cache that keeps weights, and beside it each sequence's rows and weights."""

    def __init__(self, torch, pg, kv_heads, group, dim, typ, page, last=0, pages=400, seqs=16, window=0, ctx=70000, **more):
        self.torch, self.last, self.window = torch, last, window
        self.fmt, self.type = {"f16": (pg.F16, torch.float16), "bf16": (pg.BF16, torch.bfloat16)}[typ]
        self.kv = pg.PagedKv(1, kv_heads * group, kv_heads, dim, pages, page=page, seqs=seqs, ctx=ctx, fmt=self.fmt,
                             windows=[window], weigh_last=last, **more)
        self.heads, self.group, self.dim = kv_heads, group, dim
        self.rows = {s: (torch.zeros(0, kv_heads, dim, dtype=self.type, device="cuda"),) * 2 for s in range(seqs)}
        self.w = {s: torch.zeros(kv_heads, 0, dtype=torch.float64, device="cuda") for s in range(seqs)}
        self.tol = {s: torch.zeros(kv_heads, 0, dtype=torch.float64, device="cuda") for s in range(seqs)}
        self.g = torch.Generator(device="cuda").manual_seed(11)
        for which in (0, 1):
            self.kv.pages(0, which).fill_(math.nan)  # what is not written must not matter
        self.kv.weights(0).fill_(math.nan)

    def rnd(self, *shape):
        return self.torch.randn(shape, generator=self.g, device="cuda").to(self.type)

    def grown(self, s, k, v):
        torch, n = self.torch, len(k)
        self.rows[s] = tuple(torch.cat((a, b)) for a, b in zip(self.rows[s], (k, v)))
        for x in (self.w, self.tol):
            x[s] = torch.cat((x[s], torch.zeros(self.heads, n, dtype=torch.float64, device="cuda")), 1)

    def begin(self, seqs, counts, shared=False, scale=1.0):
        n = self.kv.begin(seqs, counts, shared=shared)
        k, v = self.rnd(n, self.heads, self.dim) * scale, self.rnd(n, self.heads, self.dim)
        if n:
            self.kv.append(0, k, v)
        at = 0
        for s, c in zip(seqs, counts):
            self.grown(s, k[at:at + c], v[at:at + c])
            at += c
        self.batch = (seqs, counts)
        return n

    def weigh(self, sinks=None, decay=1.0, q=None, scale=None, run=True):
        seqs, counts = self.batch
        n = sum(counts)
        q = self.rnd(n, self.heads * self.group, self.dim) if q is None else q
        if run:
            self.kv.weigh(0, q, scale=scale, sinks=sinks, decay=decay)
        at = 0
        for s, c in zip(seqs, counts):
            k = self.rows[s][0]
            m = min(c, self.last or c)
            if c:
                new, tol = given(self.torch, q[at + c - m:at + c], k, len(k) - m, scale or self.dim ** -0.5, self.window, sinks)
                old = decay * self.w[s] if decay else 0 * self.tol[s]
                self.w[s] = old + new
                # the product and the sum are a rounding each
                self.tol[s] = (decay * self.tol[s] + tol + (old.abs() + self.w[s].abs()) * 2.0 ** -24)
            at += c
        return q

    def check(self, seqs=None, what=""):
        for s in seqs if seqs is not None else self.rows:
            n = self.kv.length(s)
            assert n == len(self.rows[s][0]) == self.w[s].shape[1]
            if n:
                close(self.kv.weights(0)[s, :, :n], self.w[s], self.tol[s], f"{what} sequence {s} of {n}")
                for which in (0, 1):
                    assert self.torch.equal(self.kv.read_rows(0, which, s), self.rows[s][which]), (what, s, which)

    def fork(self, src, dst, lens=None):
        self.kv.fork(src, dst, lens)
        for i, (a, b) in enumerate(zip(src, dst)):
            n = lens[i] if lens else len(self.rows[a][0])
            self.rows[b] = tuple(x[:n] for x in self.rows[a])
            self.w[b], self.tol[b] = self.w[a][:, :n], self.tol[a][:, :n]

    def evict(self, seqs, keep, first=0, recent=0):
        """The order of the weights as the device has them, so that no rounding decides."""
        torch = self.torch
        keeps = [keep] * len(seqs) if isinstance(keep, int) else keep
        dev = {s: self.kv.weights(0)[s, :, :self.kv.length(s)].double().cpu() for s in seqs}
        self.kv.evict(seqs, keep, first=first, recent=recent)
        for s, m in zip(seqs, keeps):
            n = dev[s].shape[1]
            if n <= m:
                continue
            rows, w, tol = [], [], []
            for h in range(self.heads):
                kept = picks(dev[s][h].tolist(), m, first, recent)
                at = torch.tensor(kept, device="cuda")
                rows.append([x[at, h] for x in self.rows[s]])
                w.append(self.w[s][h, at]), tol.append(self.tol[s][h, at])
            self.rows[s] = tuple(torch.stack([r[i] for r in rows], 1) for i in (0, 1))
            self.w[s], self.tol[s] = torch.stack(w), torch.stack(tol)


def picks(w, keep, first, recent):
    mid = range(first, len(w) - recent)
    heavy = sorted(mid, key=lambda i: (not math.isnan(w[i]), -w[i] if not math.isnan(w[i]) else 0, i))[:keep - first - recent]
    return sorted(list(range(first)) + heavy + list(range(len(w) - recent, len(w))))


# kv_heads, group, page, window, last, [(old positions, new tokens)]
SHAPES = {
    "one token, one position": (2, 8, 32, 0, 0, [(0, 1)]),
    "tokens side by side": (2, 4, 64, 0, 0, [(0, 1), (31, 1), (32, 1), (300, 1), (1000, 1), (77, 0)]),
    "rows of two tiles": (1, 8, 32, 0, 0, [(100, 4), (999, 3), (64, 2)]),
    "many pieces": (1, 2, 256, 0, 0, [(9000, 1)]),
    "a chunk": (2, 4, 64, 0, 0, [(700, 130)]),
    "a prompt": (1, 5, 32, 0, 0, [(0, 517)]),
    "an observing tail": (2, 8, 64, 0, 3, [(3000, 200), (50, 1), (0, 40)]),
    "an observing tail of many rows": (1, 16, 128, 0, 32, [(2000, 300)]),
    "chunks and tokens": (3, 2, 32, 0, 0, [(0, 300), (500, 1), (33, 65), (1200, 2), (5, 1)]),
    "a window": (2, 8, 32, 100, 0, [(1000, 1), (20, 1), (99, 3), (700, 150), (0, 300)]),
    "a window of one": (1, 4, 64, 1, 0, [(200, 2), (64, 100)]),
    "one query head a head": (2, 1, 64, 33, 0, [(500, 1), (100, 200)]),
    "forty query heads a head": (1, 40, 32, 0, 0, [(500, 1), (3, 7)]),
}


@pytest.mark.parametrize("typ,dim", [("f16", 64), ("bf16", 128), ("f16", 256), ("bf16", 256)])
@pytest.mark.parametrize("name", SHAPES)
def test_weigh(torch_gpu, pg, name, typ, dim):
    torch = torch_gpu
    heads, group, page, window, last, batch = SHAPES[name]
    m = Model(torch, pg, heads, group, dim, typ, page, last=last, window=window)
    seqs = list(range(len(batch)))
    for s, (old, _) in enumerate(batch):
        for at in range(0, old, 4000):
            m.begin([s], [min(4000, old - at)])
    m.check(what="new")
    sinks = torch.randn(heads * group, generator=m.g, device="cuda")
    m.begin(seqs[::-1], [c for _, c in batch][::-1])
    q = m.weigh()
    m.check(what="first")
    m.weigh(q=q, sinks=sinks, decay=0.75, scale=0.3)
    m.check(what="second")
    m.begin(seqs, [1] * len(seqs))
    m.weigh(decay=1.0)
    m.check(what="third")
    m.weigh(decay=0.0)
    m.check(what="afresh")


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("group,tokens", [(8, 1), (4, 60)])
def test_scores_far_apart(torch_gpu, pg, typ, group, tokens):
    m = Model(torch_gpu, pg, 1, group, 128, typ, 64)
    m.begin([0], [800], scale=12.0)
    m.begin([0], [tokens], scale=30.0)
    m.weigh()
    m.check()


@pytest.mark.parametrize("typ,dim", [("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("group,tokens", [(8, 1), (2, 5), (4, 50)])
@pytest.mark.parametrize("window", [0, 40])
def test_odd_values(torch_gpu, pg, typ, dim, group, tokens, window):
    """NaN and infinities of K reach the weights that the rows which see them give, and no others."""
    torch = torch_gpu
    for odd in (math.nan, math.inf, -math.inf):
        for at in (0, 131, 149):
            m = Model(torch, pg, 1, group, dim, typ, 32, window=window)
            m.begin([0, 1], [150, 70])
            m.begin([1, 0], [2, tokens])
            page = m.kv.table(0)[at // 32]
            m.kv.pages(0, pg.K)[page, 0, at % 32 // 16, 0, at % 16, 3] = odd
            q = m.rnd(2 + tokens, group, dim)
            q[:, :, 3] = q[:, :, 3].abs() + 0.01  # the score is as odd
            m.kv.weigh(0, q)
            k = m.rows[0][0].clone()
            k[at, 0, 3] = odd
            want, tol = given(torch, q[2:], k, 150, dim ** -0.5, window)
            got = m.kv.weights(0)[0, :, :150 + tokens]
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            fine = torch.isfinite(want)
            close(got[fine], want[fine], tol[fine], f"{odd} at {at}")
            want, tol = given(torch, q[:2], m.rows[1][0], 70, dim ** -0.5, window)
            close(m.kv.weights(0)[1, :, :72], want, tol)


def test_rows_that_see_minus_infinity_alone(torch_gpu, pg):
    """0 / 0 where such a row sees, nothing where it does not; a sink takes it all."""
    torch = torch_gpu
    for tokens, group in ((1, 2), (50, 2)):
        m = Model(torch, pg, 1, group, 64, "bf16", 32, window=1)
        m.begin([0], [100])
        m.begin([0], [tokens])
        at = 100
        m.kv.pages(0, pg.K)[m.kv.table(0)[at // 32], 0, at % 32 // 16, 0, at % 16, 0] = -math.inf
        q = m.rnd(tokens, group, 64).abs() + 0.1
        m.kv.weigh(0, q)
        got = m.kv.weights(0)[0, 0, :100 + tokens]
        assert torch.isnan(got[100]) and torch.isfinite(got[:100]).all() and (got[:100] == 0).all()
        assert torch.allclose(got[101:], torch.full_like(got[101:], group))
        m.kv.weigh(0, q, sinks=torch.zeros(group, device="cuda"), decay=0.0)
        assert m.kv.weights(0)[0, 0, 100] == 0


@pytest.mark.parametrize("seed", range(3))
def test_weights_follow_their_sequences(torch_gpu, pg, seed):
    """Rollbacks, forks, copies, frees and compactions: new positions weigh nothing whatever was in their place."""
    r = random.Random(seed)
    m = Model(torch_gpu, pg, 2, 4, 64, "f16", 32, seqs=6, pages=120)
    alive = []
    for step in range(60):
        op = r.choice(["step", "step", "step", "cut", "fork", "copy", "free", "compact", "reserve"])
        free = [s for s in range(6) if s not in alive]
        if op == "step" or not alive:
            seqs = r.sample(range(6), r.randint(1, 4))
            m.begin(seqs, [r.choice([1, 1, 2, 9, 40]) for _ in seqs], shared=r.random() < 0.5)
            m.weigh(decay=r.choice([1.0, 0.5, 0.0]))
            alive = [s for s in range(6) if m.kv.length(s)]
        elif op == "cut":
            s = r.choice(alive)
            n = r.randint(0, m.kv.length(s))
            m.kv.set_len(s, n)
            m.rows[s] = tuple(x[:n] for x in m.rows[s])
            m.w[s], m.tol[s] = m.w[s][:, :n], m.tol[s][:, :n]
        elif op in ("fork", "copy") and free:
            s, n = r.choice(alive), None
            if op == "fork":
                m.fork([s], [free[0]], [r.randint(0, m.kv.length(s))])
            else:
                m.kv.copy([s], [free[0]])
                m.rows[free[0]], m.w[free[0]], m.tol[free[0]] = m.rows[s], m.w[s], m.tol[s]
        elif op == "free":
            s = r.choice(alive)
            m.kv.free([s])
            m.rows[s] = tuple(x[:0] for x in m.rows[s])
            m.w[s], m.tol[s] = m.w[s][:, :0], m.tol[s][:, :0]
        elif op == "compact":
            m.kv.compact()
        elif op == "reserve":
            s = r.choice(alive)
            n = m.kv.length(s)
            m.kv.reserve([s], [5])
            assert (m.kv.weights(0)[s, :, n:n + 5] == 0).all()
            m.kv.set_len(s, n)
        alive = [s for s in range(6) if m.kv.length(s)]
        m.check(what=f"step {step}, {op}")


# ---- eviction ----

@pytest.mark.parametrize("typ,dim,page,heads", [("f16", 64, 32, 1), ("bf16", 128, 64, 3), ("f16", 256, 256, 2), ("bf16", 256, 32, 2)])
def test_evict(torch_gpu, pg, typ, dim, page, heads):
    torch = torch_gpu
    m = Model(torch, pg, heads, 2, dim, typ, page, pages=600 * 32 // page, seqs=12)
    lens = [1, 2, 31, 32, 33, 64, 257, 300, 1000, 2049, 4100, 1]
    for s, n in enumerate(lens):
        m.begin([s], [n])
    g = torch.Generator(device="cuda").manual_seed(3)
    for s, n in enumerate(lens):
        w = torch.randn(heads, n, generator=g, device="cuda").exp()
        w = torch.where(w < 1, (w * 4).round() / 4, w)  # many alike, some nothing
        m.kv.weights(0)[s, :, :n] = w
        m.w[s] = w.double()
    m.tol = {s: x.abs() * 0 for s, x in m.w.items()}
    for seqs, keep, first, recent in [([7, 3], 100, 0, 0), (list(range(12)), [1, 1, 30, 32, 32, 33, 200, 90, 513, 2048, 1500, 5], 1, 0),
                                      ([10, 9, 8], [1024, 700, 512], 4, 500), ([10], 31, 7, 24), ([9, 8], [33, 64], 0, 33),
                                      (list(range(12)), 1, 0, 1), ([], 5, 0, 0)]:
        before = {s: m.kv.position(s) for s in seqs}
        m.evict(seqs, keep, first, recent)
        m.check(what=f"{seqs} to {keep}")
        assert all(m.kv.position(s) == before[s] for s in seqs)
        owned = {p for s in range(12) for p in m.kv.table(s)}
        assert m.kv.free_pages() == 600 * 32 // page - len(owned)


def test_evict_orders_odd_weights(torch_gpu, pg):
    """NaN weighs most, whatever its sign; infinities are in order; both zeros are alike; of equal ones the first stay."""
    torch = torch_gpu
    m = Model(torch, pg, 1, 1, 64, "f16", 32)
    odd = [0.0, -0.0, 1.0, math.nan, -math.inf, math.inf, 1e-45, -1.0, -math.nan, 0.0, 3e38, -0.0, 1.0, 1e-45, math.inf] * 3
    for keep in (1, 2, 6, 7, 11, 13, 20, 30, 44):
        m.kv.free([0])
        m.rows[0] = tuple(x[:0] for x in m.rows[0])
        m.w[0] = m.w[0][:, :0]
        m.begin([0], [len(odd)])
        m.kv.weights(0)[0, 0, :len(odd)] = torch.tensor(odd, device="cuda")
        rows = [x[:, 0] for x in m.rows[0]]
        m.kv.evict([0], keep)
        kept = picks(odd, keep, 0, 0)
        for which in (0, 1):
            assert torch.equal(m.kv.read_rows(0, which, 0)[:, 0], rows[which][kept]), keep
        got, want = m.kv.weights(0)[0, 0, :keep], torch.tensor(odd, device="cuda")[kept]
        assert torch.equal(torch.nan_to_num(got, 7.0), torch.nan_to_num(want, 7.0))


def test_evict_long_and_all_alike(torch_gpu, pg):
    torch = torch_gpu
    m = Model(torch, pg, 1, 1, 64, "bf16", 256, pages=310, seqs=2)
    m.begin([0], [8000])
    for _ in range(7):
        m.begin([0], [7001])
    n = m.kv.length(0)
    for w in (0.0, 2.5):
        m.fork([0], [1])
        m.kv.weights(0)[1, :, :n] = w
        m.kv.evict([1], 3001, first=3, recent=1000)
        at = list(range(2001)) + list(range(n - 1000, n))
        for which in (0, 1):
            assert torch.equal(m.kv.read_rows(0, which, 1), m.rows[0][which][at])
        m.kv.free([1])
    w = torch.rand(n, device="cuda")
    m.fork([0], [1])
    m.kv.weights(0)[1, 0, :n] = w
    m.kv.evict([1], 20000)
    at = torch.sort(torch.sort(w, descending=True, stable=True).indices[:20000]).values
    assert torch.equal(m.kv.weights(0)[1, 0, :20000], w[at])
    assert torch.equal(m.kv.read_rows(0, 0, 1), m.rows[0][0][at]) and torch.equal(m.kv.read_rows(0, 1, 1), m.rows[0][1][at])
    m.kv.free([1])
    assert torch.equal(m.kv.read_rows(0, 0, 0), m.rows[0][0])


def test_many_layers_and_sequences(torch_gpu, pg):
    """More sequences and pages than a launch's arguments hold, layers that keep different positions."""
    torch = torch_gpu
    layers, heads, n = 3, 2, 150
    kv = pg.PagedKv(layers, heads, heads, 64, 1600, page=32, seqs=n, ctx=400, weigh_last=0, tokens=8192)
    g = torch.Generator(device="cuda").manual_seed(5)
    lens = [60 + 7 * i % 200 for i in range(n)]
    kv.reserve(range(n), lens)
    for layer in range(layers):
        for which in (0, 1):
            p = kv.pages(layer, which)
            p.copy_(torch.randn(p.shape, generator=g, device="cuda"))
        kv.weights(layer).copy_(torch.rand(n, heads, 400, generator=g, device="cuda"))
    before = {(layer, which, s): kv.read_rows(layer, which, s) for layer in range(layers) for which in (0, 1) for s in range(n)}
    w = [kv.weights(layer).clone() for layer in range(layers)]
    kv.evict(range(n), 70, first=2, recent=10)
    for layer in range(layers):
        for s in range(n):
            assert kv.length(s) == min(70, lens[s])
            for h in range(heads):
                at = picks(w[layer][s, h, :lens[s]].tolist(), 70, 2, 10) if lens[s] > 70 else list(range(lens[s]))
                for which in (0, 1):
                    assert torch.equal(kv.read_rows(layer, which, s)[:, h], before[layer, which, s][at, h]), (layer, s, h)
                assert torch.equal(kv.weights(layer)[s, h, :len(at)], w[layer][s, h, at])


# ---- all of it together ----

def test_a_run_with_eviction(torch_gpu, pg):
    """Prompts, forks, generation attended as shared and weighed, evicted, carried on: positions go on counting, attention is
    over what is left."""
    torch = torch_gpu
    th, amp = rope_freqs(32, 1e4)
    rope = pg.Rope(32, base=1e4)
    m = Model(torch, pg, 2, 4, 64, "bf16", 32, last=8, seqs=8, pages=200, rope=rope)
    pos = {s: 0 for s in range(8)}
    r = random.Random(2)

    def step(seqs, counts, shared=True):
        n = m.kv.begin(seqs, counts, shared=shared)
        q, k, v = m.rnd(n, 8, 64), m.rnd(n, 2, 64), m.rnd(n, 2, 64)
        at = torch.tensor([pos[s] + t for s, c in zip(seqs, counts) for t in range(c)], device="cuda", dtype=torch.int32)
        turned = m.kv.append(0, k, v, q)
        for x, y in ((k, None), (q, turned)):
            want, tol = rotated(x, at, 32, "half", th, amp)
            if y is not None:
                close(y, want, tol, "q")
        k = pg.rotate(k, at, rope)
        i = 0
        for s, c in zip(seqs, counts):
            m.grown(s, k[i:i + c], v[i:i + c])
            pos[s] += c
            i += c
        m.batch = (seqs, counts)
        out = m.kv.attend(0, turned)
        i = 0
        for s, c in zip(seqs, counts):
            kk, vv = m.rows[s]
            want, tol = attention(turned[i:i + c], kk, vv, len(kk) - c, 64 ** -0.5)
            close(out[i:i + c], want, tol, f"sequence {s}")
            i += c
        m.weigh(q=turned)
        m.check(seqs)
        assert all(m.kv.position(s) == pos[s] for s in seqs)

    step([0], [700])
    m.fork([0] * 3, [1, 2, 3])
    pos.update({1: 700, 2: 700, 3: 700})
    for _ in range(5):
        step([3, 0, 2, 1], [1, 2, 1, 1])
    m.evict([0, 2], [300, 128], first=4, recent=64)
    m.check()
    step([0, 1, 2, 3], [1, 1, 40, 2])
    m.fork([2, 2], [4, 5])
    pos[4] = pos[5] = pos[2]
    for _ in range(3):
        step([5, 4, 2, 0], [1, 1, 1, 1])
    m.evict([4], [60], recent=20)
    m.kv.free([1])
    step([4, 5, 3], [3, 1, 1])
    with pytest.raises(pg.MkvError) as e:
        m.kv.set_len(4, 59)
    assert e.value.code == -3
    m.kv.set_len(4, 61)
    m.rows[4] = tuple(x[:61] for x in m.rows[4])
    m.w[4], m.tol[4] = m.w[4][:, :61], m.tol[4][:, :61]
    pos[4] -= 2
    step([4], [5])
    m.check([s for s in range(8) if s != 1])


def test_captured_weighing_follows_the_batch(torch_gpu, pg):
    torch = torch_gpu
    stream = torch.cuda.Stream()
    m = Model(torch, pg, 2, 4, 128, "f16", 64, last=0, window=0, rope=pg.Rope(64))
    m2 = Model(torch, pg, 2, 4, 128, "f16", 64, last=0, window=0, rope=pg.Rope(64))
    rows = 300
    for x in (m, m2):
        x.begin([0, 1, 2], [500, 40, 3])
        x.begin([0], [1])
    q = m.rnd(rows, 8, 128)
    k, v = m.rnd(rows, 2, 128), m.rnd(rows, 2, 128)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    m.kv.set_stream(stream)
    with torch.cuda.graph(graph, stream=stream):
        turned = m.kv.append(0, k, v, q)
        m.kv.weigh(0, turned, decay=0.5)
    m.kv.set_stream(torch.cuda.current_stream())
    for seqs, counts, cut in [([0], [1], None), ([2, 0, 1], [1, 200, 4], None), ([1], [40], 0), ([0, 1], [1, 1], None), ([2], [60], 1)]:
        for x in (m, m2):
            if cut is not None:
                x.kv.evict([cut], 33, recent=5)
            x.kv.begin(seqs, counts)
        n = sum(counts)
        eager = m2.kv.append(0, k[:n], v[:n], q[:n])
        m2.kv.weigh(0, eager, decay=0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(turned[:n], eager)
        for s in range(3):
            a, b = (x.kv.weights(0)[s, :, :x.kv.length(s)] for x in (m, m2))
            assert torch.equal(a, b), (seqs, s)
            assert torch.equal(m.kv.read_rows(0, 0, s), m2.kv.read_rows(0, 0, s))
    with pytest.raises(pg.MkvError, match="capturing"):
        m.kv.set_stream(stream)
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            m.kv.evict([0], 5)
    m.kv.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("last,window", [(1, 0), (1, 40), (4, 0)])
def test_captured_weighing_of_few_rows(torch_gpu, pg, last, window):
    """A cache that counts a token or a few of each sequence, whose graphs have fewer kernels."""
    torch = torch_gpu
    stream = torch.cuda.Stream()
    m = Model(torch, pg, 2, 8, 64, "bf16", 64, last=last, window=window)
    m.begin([0, 1, 2], [700, 40, 3])
    m.weigh()
    m.begin([0], [1])
    rows = 300
    q = m.rnd(rows, 16, 64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    m.kv.set_stream(stream)
    with torch.cuda.graph(graph, stream=stream):
        m.kv.weigh(0, q, decay=0.5)
    m.kv.set_stream(torch.cuda.current_stream())
    for seqs, counts in [([0], [1]), ([2, 0, 1], [1, 200, 4]), ([1], [40]), ([0, 1], [1, 1])]:
        m.begin(seqs, counts)
        graph.replay()
        torch.cuda.synchronize()
        m.weigh(q=q[:sum(counts)], decay=0.5, run=False)
        m.check(what=f"{seqs} {counts}")


def test_fewer_rows_than_the_batch_in_a_replay(torch_gpu, pg):
    """Tokens behind the captured rows are left out, of what they give as of what they are given."""
    torch = torch_gpu
    for counts, captured in (([1, 1, 1], 2), ([40, 50], 60), ([3, 2], 4)):
        stream = torch.cuda.Stream()
        m = Model(torch, pg, 1, 4, 64, "bf16", 32)
        m.begin([0, 1, 2], [90, 70, 100])
        m.kv.weights(0)[:] = 0
        m.kv.begin([0], [1])
        q = m.rnd(captured, 4, 64)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        m.kv.set_stream(stream)
        with torch.cuda.graph(graph, stream=stream):
            m.kv.weigh(0, q, decay=0.0)
        m.kv.set_stream(torch.cuda.current_stream())
        m.kv.set_len(0, 90)
        seqs = list(range(len(counts)))
        n = m.begin(seqs, counts)
        graph.replay()
        torch.cuda.synchronize()
        at = 0
        for s, c in zip(seqs, counts):
            k = m.rows[s][0]
            have = max(0, min(c, captured - at))
            got = m.kv.weights(0)[s, :, :len(k)]
            if have:
                want, tol = given(torch, q[at:at + have], k, len(k) - c, 64 ** -0.5)
                close(got, want, tol, f"sequence {s}")
            else:
                assert (got == 0).all()
            at += c


@pytest.mark.parametrize("tokens", [1, 5])
def test_as_many_rows_as_there_are_numbers(torch_gpu, pg, tokens):
    """Rows behind the batch's last are not read, however many the call says there are."""
    import ctypes
    m = Model(torch_gpu, pg, 2, 8, 64, "f16", 64)
    m.begin([0], [600])
    m.begin([0, 1], [tokens, tokens])
    q = m.weigh(run=False)
    rc = m.kv._lib.mpg_weigh(m.kv._h, 0, 2 ** 31 - 1, ctypes.c_void_p(q.data_ptr()), q.stride(0), q.stride(1), 64 ** -0.5, None, 1.0)
    assert rc == 0
    m.check()


def test_another_current_stream(torch_gpu, pg):
    torch = torch_gpu
    m = Model(torch, pg, 1, 8, 64, "f16", 32)
    m.begin([0], [300])
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        m.begin([0], [1])
        torch.cuda.synchronize()
        m.weigh()
        m.kv.sync()
        m.check([0])


def test_two_caches_on_two_streams(torch_gpu, pg):
    """Each has its own room to work in: calls of one run beside the other's."""
    torch = torch_gpu
    streams = [torch.cuda.Stream() for _ in range(2)]
    with torch.cuda.stream(streams[0]):
        a = Model(torch, pg, 2, 4, 64, "bf16", 64)
    with torch.cuda.stream(streams[1]):
        b = Model(torch, pg, 1, 8, 128, "f16", 32, last=4)
    for step in range(6):
        for m, s in ((a, streams[0]), (b, streams[1])):
            with torch.cuda.stream(s):
                m.begin([0, 1, 2], [300, 1, 40] if step % 2 else [1, 60, 2], shared=step > 3)
                m.weigh(decay=0.9)
                if step == 3:
                    m.evict([0], [100], first=2, recent=30)
    for m, s in ((a, streams[0]), (b, streams[1])):
        with torch.cuda.stream(s):
            m.check()


def test_refusals(torch_gpu, pg):
    torch = torch_gpu

    def refused(code, call):
        with pytest.raises(pg.MkvError) as e:
            call()
        assert e.value.code == code

    plain = pg.PagedKv(1, 4, 2, 64, 8, page=32, seqs=2, ctx=200)
    x = torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda")
    plain.begin([0], [3])
    refused(-1, lambda: plain.weigh(0, x))
    refused(-1, lambda: plain.weights(0))
    refused(-1, lambda: plain.evict([0], 2))
    lib = pg.lib()
    assert lib.mpg_keep_weights(plain.handle, 0) == -1  # a batch has stood
    with pytest.raises(pg.MkvError):
        pg.PagedKv(1, 4, 2, 64, 8, page=32, seqs=2, ctx=200, weigh_last=-1)
    kv = pg.PagedKv(2, 4, 2, 64, 8, page=32, seqs=3, ctx=200, weigh_last=4, windows=[0, 20])
    assert lib.mpg_keep_weights(kv.handle, 0) == -1  # it keeps them
    refused(-1, lambda: kv.weigh(0, x))  # no batch
    kv.begin([0], [3])
    refused(-4, lambda: kv.weigh(2, x))
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(decay=-0.5), dict(decay=math.nan), dict(decay=math.inf)):
        refused(-1, lambda: kv.weigh(0, x, **bad))
    with pytest.raises(pg.MkvError):
        kv.weigh(0, x[:2])  # fewer rows than tokens
    for bad in (x.float(), x.cpu(), x[:, :3], x[..., :32]):
        with pytest.raises(ValueError):
            kv.weigh(0, bad)
    with pytest.raises(ValueError):
        kv.weigh(0, x, sinks=torch.zeros(4, dtype=torch.float64, device="cuda"))
    kv.begin([0, 1], [100, 60])
    for args in (([0], 0), ([0], -1), ([0, 0], 30), ([3], 30), ([-1], 30)):
        refused(-1, lambda: kv.evict(*args, recent=20))
    for kw in (dict(first=-1, recent=20), dict(recent=-1), dict(first=20, recent=20), dict(recent=19), dict(recent=31)):
        refused(-1, lambda: kv.evict([0], 30, **kw))
    with pytest.raises(ValueError):
        kv.evict([0, 1], [30], recent=20)
    refused(-7, lambda: kv.evict([0, 1], [99, 59], recent=20))  # 6 pages, 2 free
    assert kv.length(0) == 103 and kv.length(1) == 60 and kv.position(0) == 103
    kv.evict([0, 1], [200, 60], recent=20)  # nothing to cut
    assert kv.length(0) == 103 and kv.position(1) == 60
    kv.evict([0], 40, recent=20)
    refused(-1, lambda: kv.weigh(0, x))  # the batch has ended
    kv.close()
    for call in (lambda: kv.weights(0), lambda: kv.weigh(0, x), lambda: kv.evict([0], 3), lambda: kv.position(0)):
        refused(-1, call)

