"""The paged cache on the GPU against plain 64-bit forms (tests/paged_reference.py): rotary positions, append, attention,
page operations, captured graphs, streams, refusals, and a run of them together."""
import ctypes
import math
import random

import pytest

from tests.paged_reference import attention, close, rope_freqs, rotated

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pg(torch_gpu):
    from mechta_amd import paged
    return paged


def rnd(torch, seed, *shape, dtype=None, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda") * scale
    return x if dtype is None else x.to(dtype)


def types(torch, pg):
    return {"f16": (pg.F16, torch.float16), "bf16": (pg.BF16, torch.bfloat16)}


class Model:
    """A one-layer cache and beside it each sequence's rows, appended without rotation."""

    def __init__(self, torch, pg, kv_heads, group, dim, typ, page, pages=200, seqs=8, window=0, **more):
        self.torch, self.fmt = torch, types(torch, pg)[typ]
        self.kv = pg.PagedKv(1, kv_heads * group, kv_heads, dim, pages, page=page, seqs=seqs, ctx=100000, fmt=self.fmt[0],
                             windows=[window], **more)
        self.heads, self.group, self.dim, self.window = kv_heads, group, dim, window
        self.rows = {s: (rnd(torch, 1, 0, kv_heads, dim, dtype=self.fmt[1]),) * 2 for s in range(seqs)}
        self.seed = 1000

    def foul(self, value=math.nan):
        """NaN in every page: rows that are not written must not matter."""
        for w in (0, 1):
            self.kv.pages(0, w).fill_(value)

    def step(self, seqs, counts, write=True):
        torch = self.torch
        n = self.kv.begin(seqs, counts)
        assert n == sum(counts)
        self.seed += 2
        # k and v side by side, so their rows are strided
        both = rnd(torch, self.seed, n, 2 * self.heads, self.dim, dtype=self.fmt[1])
        k, v = both[:, :self.heads], both[:, self.heads:]
        if write:
            self.kv.append(0, k, v)
        self.batch = (seqs, counts)
        at = 0
        for s, c in zip(seqs, counts):
            self.rows[s] = tuple(torch.cat((a, b[at:at + c])) for a, b in zip(self.rows[s], (k, v)))
            at += c
        return k, v

    def check(self, sinks=None, gate=False, scale=None, out_rows=0, strided=False, what=""):
        torch = self.torch
        seqs, counts = self.batch
        n, h = sum(counts), self.heads * self.group
        q = rnd(torch, self.seed + 1, n + out_rows, h, 2 * self.dim if strided else self.dim, dtype=self.fmt[1])
        g = q[..., self.dim:] if strided else rnd(torch, self.seed + 7, n + out_rows, h, self.dim, dtype=self.fmt[1])
        q = q[..., :self.dim]
        out = torch.full((n + out_rows, h, self.dim), 7.0, dtype=self.fmt[1], device="cuda")
        self.kv.attend(0, q, scale=scale, sinks=sinks, gate=g if gate else None, out=out)
        assert (out[n:] == 7).all()
        at = 0
        for s, c in zip(seqs, counts):
            k, v = self.rows[s]
            if c:
                want, tol = attention(q[at:at + c], k, v, len(k) - c, scale or self.dim ** -0.5, self.window, sinks,
                                      g[at:at + c] if gate else None)
                close(out[at:at + c], want, tol, f"{what} sequence {s}, {c} tokens of {len(k)}")
            at += c
        return out


# ---- rotary positions ----

SCALED = [dict(scaling="none"), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
          dict(scaling="yarn", factor=32.0, original=4096), dict(scaling="bands", factor=8.0, original=8192)]


@pytest.mark.parametrize("typ", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,heads,d,dim", [(1, 1, 64, 64), (1, 16, 256, 64), (9, 3, 128, 128), (37, 5, 40, 24),
                                              (8, 2, 10, 6), (130, 4, 80, 16), (3, 1, 512, 512)])
def test_rotate(torch_gpu, pg, typ, layout, rows, heads, d, dim):
    torch = torch_gpu
    t = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[typ]
    for i, sc in enumerate(SCALED):
        rope = pg.Rope(dim, layout=layout, base=5e5, **sc)
        th, amp = rope.freqs()
        want_th, want_amp = rope_freqs(dim, 5e5, **sc)
        assert amp == pytest.approx(want_amp, rel=1e-14) and th == pytest.approx(want_th, rel=1e-12)
        x = rnd(torch, 11 + i, rows, heads, d, dtype=t)
        pos = torch.randint(0, 4194304, (rows,), device="cuda", dtype=torch.int32)
        pos[0] = 4194303
        want, tol = rotated(x, pos, dim, layout, want_th, want_amp)
        close(pg.rotate(x, pos, rope), want, tol, f"{sc}")
        y = x.clone()
        assert pg.rotate(y, pos, rope, out=y) is y  # in place
        assert torch.equal(y, pg.rotate(x, pos, rope))
        # heads before rows, odd offsets: another path, the same results
        odd = torch.empty(rows * heads * d + 1, dtype=t, device="cuda")[1:].view(heads, rows, d).transpose(0, 1)
        odd.copy_(x)
        out = torch.empty(rows, heads, d + 1, dtype=t, device="cuda")[..., 1:]
        assert torch.equal(pg.rotate(odd, pos, rope, out=out), y)


def test_rotate_keeps_lengths_and_turns_back(torch_gpu, pg):
    torch = torch_gpu
    x = rnd(torch, 3, 50, 2, 64)
    pos = torch.arange(50, device="cuda", dtype=torch.int32) * 1000
    rope = pg.Rope(64, base=1e4)
    y = pg.rotate(x, pos, rope)
    assert torch.equal(pg.rotate(x, torch.zeros_like(pos), rope), x)
    assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1), rtol=2 ** -20)
    assert torch.allclose(pg.rotate(y, -pos, rope), x, atol=2 ** -19 * float(x.abs().max()))
    assert pg.rotate(x[:0], pos[:0], rope).shape == (0, 2, 64)


# ---- append ----

@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim,rot,layout", [(64, 64, "half"), (128, 32, "interleaved"), (256, 64, "half"), (128, 128, "half"),
                                            (64, 22, "half"), (64, 22, "interleaved"), (256, 256, "interleaved")])
@pytest.mark.parametrize("page", [32, 256])
def test_append(torch_gpu, pg, typ, dim, rot, layout, page):
    torch = torch_gpu
    fmt, t = types(torch, pg)[typ]
    heads, group, layers = 3, 5, 2
    th, amp = rope_freqs(rot, 1e4, "yarn", 4.0, 2048)
    rope = pg.Rope(rot, layout=layout, base=1e4, scaling="yarn", factor=4.0, original=2048)
    with pg.PagedKv(layers, heads * group, heads, dim, 40, page=page, seqs=4, ctx=5000, fmt=fmt, rope=rope) as kv:
        kv.pages(0, 0).fill_(5.0), kv.pages(0, 1).fill_(5.0), kv.pages(1, 0).fill_(5.0), kv.pages(1, 1).fill_(5.0)
        rows = {(layer, s): ([], []) for layer in range(layers) for s in range(4)}
        tols = {k: [] for k in rows}
        lens = [0] * 4
        for i, (seqs, counts) in enumerate([([0, 2], [33, 1]), ([2, 1, 0], [1, 0, 31]), ([3, 0, 2], [100, 1, 63]),
                                            ([1], [32]), ([2, 3, 0, 1], [1, 1, 1, 1])]):
            n = kv.begin(seqs, counts)
            for layer in range(layers):
                x = rnd(torch, 10 * i + layer, n + 2, heads * (group + 2), dim, dtype=t)
                q, k, v = x[:, :heads * group], x[:, heads * group:heads * (group + 1)], x[:, heads * (group + 1):]
                pos = torch.cat([torch.arange(lens[s], lens[s] + c) for s, c in zip(seqs, counts)]).cuda()
                q_out = torch.full((n + 2, heads * group, dim), 9.0, dtype=t, device="cuda")
                assert kv.append(layer, k, v, q, q_out=q_out) is q_out
                assert (q_out[n:] == 9).all()
                close(q_out[:n], *rotated(q[:n], pos, rot, layout, th, amp), "q")
                want, tol = rotated(k[:n], pos, rot, layout, th, amp)
                at = 0
                for s, c in zip(seqs, counts):
                    rows[layer, s][0].append(want[at:at + c])
                    rows[layer, s][1].append(v[at:at + c])
                    tols[layer, s].append(tol[at:at + c])
                    at += c
            for s, c in zip(seqs, counts):
                lens[s] += c
            for (layer, s), (k, v) in rows.items():
                if k and lens[s]:
                    close(kv.read_rows(layer, 0, s), torch.cat(k), torch.cat(tols[layer, s]), f"layer {layer} sequence {s}")
                    assert torch.equal(kv.read_rows(layer, 1, s), torch.cat(v))
                    assert torch.equal(kv.read_rows(layer, 1, s, lens[s] // 2, lens[s]), torch.cat(v)[lens[s] // 2:])
        # rows that no token was written to are as they were
        total = sum(lens) * heads * dim
        for layer in range(layers):
            for which in (0, 1):
                assert int((kv.pages(layer, which) != 5).sum()) <= total
                assert int((kv.pages(layer, which) == 5).sum()) >= kv.pages(layer, which).numel() - total


# ---- attention ----

BATCHES = [([0], [1]), ([0, 1, 2], [1, 17, 4]), ([2, 0], [1, 1]), ([3, 1, 0, 2], [40, 1, 0, 3]), ([1], [3]),
           ([0, 1, 2, 3, 4], [1, 1, 130, 1, 64]), ([4, 0], [1, 33]), ([2], [2])]


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv_heads,group,page,window", [(2, 8, 64, 0), (1, 1, 32, 0), (3, 5, 128, 33), (1, 16, 256, 0),
                                                       (2, 4, 32, 64), (1, 40, 64, 1)])
def test_attend(torch_gpu, pg, typ, dim, kv_heads, group, page, window):
    torch = torch_gpu
    m = Model(torch, pg, kv_heads, group, dim, typ, page, window=window)
    m.foul()
    sinks = rnd(torch, 5, kv_heads * group, scale=2.0)
    for i, (seqs, counts) in enumerate(BATCHES):
        m.step(seqs, counts)
        m.check(sinks=sinks if i % 3 == 1 else None, gate=i % 2 == 1, out_rows=i % 3, strided=i % 2 == 1, what=f"batch {i}")
    m.kv.close()


@pytest.mark.parametrize("typ,dim,kv_heads,group,page,window", [
    ("f16", 256, 2, 8, 64, 0), ("bf16", 128, 4, 8, 32, 513), ("f16", 128, 1, 3, 128, 0), ("bf16", 64, 2, 1, 256, 700)])
def test_attend_long(torch_gpu, pg, typ, dim, kv_heads, group, page, window):
    """Thousands of positions (the keys split over work-groups), decodes beside a chunk."""
    m = Model(torch_gpu, pg, kv_heads, group, dim, typ, page, pages=40000 // page + 9, window=window,
              tokens=16384)
    for i, (seqs, counts) in enumerate([([0, 1, 2], [9000, 3001, 57]), ([0, 1, 2], [1, 1, 1]), ([1, 0], [4, 300]),
                                        ([2, 0, 1], [512, 1, 2]), ([0], [4]), ([3], [1])]):
        m.step(seqs, counts)
        if i:
            m.check(gate=i % 2 == 0, what=f"batch {i}")
    m.kv.close()


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [1e-3, 1.0])
def test_scores_far_apart(torch_gpu, pg, typ, scale):
    """Scores that hardly differ, and scores that rise over the keys by hundreds, so that the reference moves again and
    again; a row whose weight is all on its first key."""
    torch = torch_gpu
    m = Model(torch, pg, 1, 4, 64, typ, 32)
    m.step([0], [600])
    k = m.rows[0][0]
    ramp = torch.linspace(-3, 3, 600, device="cuda").view(-1, 1, 1)
    k = (k * 0.1 + ramp).to(k.dtype)
    m.kv.append(0, k, m.rows[0][1])
    m.rows[0] = (k, m.rows[0][1])
    m.check(scale=scale, what="ramp")
    m.kv.close()


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim,group,tokens", [(64, 4, 3), (128, 8, 4), (256, 8, 9), (128, 3, 100), (64, 1, 300)])
@pytest.mark.parametrize("window", [0, 40])
def test_odd_values(torch_gpu, pg, typ, dim, group, tokens, window):
    """NaN and infinities in K and V of a position reach the rows that see it, and no others: those are as with other
    values there, bit for bit."""
    torch = torch_gpu
    m = Model(torch, pg, 2, group, dim, typ, 32, window=window)
    m.foul()
    m.step([0, 1], [70, 33])
    m.step([1, 0], [1, tokens])
    n = 70 + tokens
    q = rnd(torch, 77, 1 + tokens, 2 * group, dim, dtype=m.fmt[1])
    clean = m.kv.attend(0, q)
    k, v = (x.clone() for x in m.rows[0])
    odd = {n - 1: (0, math.nan), n - 2: (1, math.inf), 60: (1, -math.inf), 45: (1, math.nan), 3: (0, math.inf)}
    if tokens > 50:
        odd[n - 40] = (1, math.nan)
    for at, (which, value) in odd.items():
        kk, vv = k.clone(), v.clone()
        (kk, vv)[which][at, 1, 5] = value
        m.kv.set_len(0, 0)
        m.kv.begin([0], [70])
        m.kv.append(0, kk[:70], vv[:70])
        m.kv.set_len(1, 33)
        m.kv.begin([1, 0], [1, tokens])
        pad = torch.cat((m.rows[1][0][33:], kk[70:])), torch.cat((m.rows[1][1][33:], vv[70:]))
        m.kv.append(0, *pad)
        out = m.kv.attend(0, q)
        pos = torch.arange(70, n, device="cuda")
        sees = (pos >= at) & ((pos - window < at) if window else (pos >= 0))
        hit = torch.zeros(1 + tokens, 2 * group, dim, dtype=torch.bool, device="cuda")
        if which:
            hit[1:, group:, 5] = sees[:, None]
        else:
            hit[1:, group:] = sees[:, None, None]
        assert torch.equal(out[~hit], clean[~hit]), (at, which, value)
        # V: the value itself (its weight is not zero); K: NaN, or (an infinite score) NaN or a weight of one or zero
        if which and math.isnan(value):
            assert torch.isnan(out[hit]).all()
        elif which:
            assert (out[hit] == value).all(), (at, value, out[hit])
        elif math.isnan(value):
            assert torch.isnan(out[hit]).all()
    m.kv.close()


def test_large_offsets(torch_gpu, pg):
    """Pages whose element offsets pass 2^31 (a plane of more than 4 GiB)."""
    torch = torch_gpu
    heads, dim, page = 8, 128, 64
    pages = (1 << 31) // (heads * dim * page) + 80
    with pg.PagedKv(1, 16, heads, dim, pages, page=page, seqs=2, ctx=4194304) as kv:
        kv.reserve([0], [(pages - 70) * page])
        m = Model.__new__(Model)
        m.torch, m.fmt, m.kv, m.heads, m.group, m.dim, m.window, m.seed = torch, (0, torch.float16), kv, heads, 2, dim, 0, 5
        m.rows = {1: (torch.empty(0, heads, dim, dtype=torch.float16, device="cuda"),) * 2}
        m.step([1], [3000])
        assert min(kv.table(1)) * heads * dim * page > 1 << 31 or kv.table(1)[-1] * heads * dim * page > 1 << 31
        assert torch.equal(kv.read_rows(0, 0, 1), m.rows[1][0]) and torch.equal(kv.read_rows(0, 1, 1), m.rows[1][1])
        m.check(what="far pages")
        m.step([1], [1])
        m.check(what="far pages, one token")
        kv.free([0])
        assert kv.compact() > 0 and max(kv.table(1)) < 70
        m.step([1], [2])
        m.check(what="moved down")


# ---- pages ----

@pytest.mark.parametrize("typ,page,layers,heads,dim", [("f16", 32, 1, 1, 64), ("bf16", 64, 3, 2, 128), ("f16", 256, 2, 3, 256)])
def test_page_histories(torch_gpu, pg, typ, page, layers, heads, dim):
    """Random reserves, appends, forks, copies, truncations, frees and compactions: every sequence reads what was written
    to it, in every layer."""
    torch = torch_gpu
    fmt, t = types(torch, pg)[typ]
    r = random.Random(page)
    with pg.PagedKv(layers, heads, heads, dim, 60, page=page, seqs=6, ctx=100000, fmt=fmt) as kv:
        rows = [[[torch.empty(0, heads, dim, dtype=t, device="cuda")] * 2 for _ in range(layers)] for _ in range(6)]
        for step in range(120):
            op = r.choice(["append", "append", "append", "fork", "copy", "free", "set_len", "compact"])
            s = r.randrange(6)
            n = len(rows[s][0][0])
            try:
                if op == "append":
                    seqs = r.sample(range(6), r.randint(1, 3))
                    counts = [r.choice([0, 1, 31, page, page + 1, 3 * page // 2]) for _ in seqs]
                    tokens = kv.begin(seqs, counts)
                    for layer in range(layers):
                        k, v = (rnd(torch, step * 100 + layer * 2 + w, tokens, heads, dim, dtype=t) for w in (0, 1))
                        kv.append(layer, k, v)
                        at = 0
                        for x, c in zip(seqs, counts):
                            rows[x][layer] = [torch.cat((a, b[at:at + c])) for a, b in zip(rows[x][layer], (k, v))]
                            at += c
                elif op in ("fork", "copy"):
                    empty = [x for x in range(6) if not len(rows[x][0][0]) and x != s]
                    dst = r.sample(empty, min(2, len(empty)))
                    lens = [r.randint(0, n) for _ in dst]
                    if op == "fork":
                        kv.fork([s] * len(dst), dst, lens)
                    else:
                        kv.copy([s] * len(dst), dst)
                        lens = [n] * len(dst)
                    for d, m in zip(dst, lens):
                        rows[d] = [[x[:m] for x in layer] for layer in rows[s]]
                elif op == "free":
                    kv.free([s])
                    rows[s] = [[x[:0] for x in layer] for layer in rows[s]]
                elif op == "set_len":
                    m = r.randint(0, n)
                    kv.set_len(s, m)
                    rows[s] = [[x[:m] for x in layer] for layer in rows[s]]
                else:
                    kv.compact()
                    assert set(sum((kv.table(x) for x in range(6)), [])) == set(range(60 - kv.free_pages()))
            except pg.MkvError as e:
                assert e.code == -7, e
                kv.free([s])
                rows[s] = [[x[:0] for x in layer] for layer in rows[s]]
            if step % 5 == 4:
                for x in range(6):
                    assert kv.length(x) == len(rows[x][0][0])
                    for layer in range(layers):
                        for w in (0, 1):
                            assert torch.equal(kv.read_rows(layer, w, x), rows[x][layer][w]), (step, op, x, layer, w)


def test_many_copies(torch_gpu, pg):
    """More pairs than one launch takes."""
    torch = torch_gpu
    with pg.PagedKv(2, 1, 1, 64, 1400, page=32, seqs=4, ctx=100000) as kv:
        kv.reserve([0], [600 * 32 + 5])
        for layer in (0, 1):
            for w in (0, 1):
                kv.pages(layer, w).copy_(rnd(torch, 4 * layer + w, *kv.pages(layer, w).shape, dtype=torch.float16))
        want = [kv.read_rows(layer, w, 0) for layer in (0, 1) for w in (0, 1)]
        kv.copy([0], [1])
        kv.free([0])
        assert kv.compact() == 601
        assert [torch.equal(kv.read_rows(layer, w, 1), want[2 * layer + w]) for layer in (0, 1) for w in (0, 1)] == [True] * 4


# ---- together ----

def test_a_serving_run(torch_gpu, pg):
    """Prompts of two users, samples forked off one, verify steps with rejected drafts, one user leaving, a compaction, a
    late prompt in chunks: rotated keys, a sliding layer with sinks and a full one, gated."""
    torch = torch_gpu
    heads, group, dim, rot = 2, 4, 128, 64
    rope = pg.Rope(rot, base=1e6)
    th, amp = rope_freqs(rot, 1e6)
    t = torch.bfloat16
    kv = pg.PagedKv(2, heads * group, heads, dim, 40, page=32, seqs=6, ctx=4096, fmt=pg.BF16, windows=[100, 0], rope=rope)
    sinks = rnd(torch, 9, heads * group)
    none = torch.empty(0, heads, dim, dtype=t, device="cuda")
    rows = [[(none, none)] * 2 for _ in range(6)]
    seed = [100]

    def step(seqs, counts):
        n = kv.begin(seqs, counts)
        for layer in (0, 1):
            seed[0] += 10
            x = rnd(torch, seed[0], n, heads * (group + 2), dim, dtype=t)
            q, k, v = x[:, :heads * group], x[:, heads * group:heads * (group + 1)], x[:, heads * (group + 1):]
            gate = rnd(torch, seed[0] + 1, n, heads * group, dim, dtype=t)
            qr = kv.append(layer, k, v, q)
            out = kv.attend(layer, qr, sinks=sinks if layer == 0 else None, gate=gate if layer else None)
            at = 0
            for s, c in zip(seqs, counts):
                n0 = len(rows[s][layer][0])
                pos = torch.arange(n0, n0 + c, device="cuda", dtype=torch.int32)
                close(qr[at:at + c], *rotated(q[at:at + c], pos, rot, "half", th, amp), "q")
                close(kv.read_rows(layer, 0, s, n0, n0 + c), *rotated(k[at:at + c], pos, rot, "half", th, amp), "k")
                kr = kv.read_rows(layer, 0, s, n0, n0 + c)
                rows[s][layer] = tuple(torch.cat((a, b)) for a, b in zip(rows[s][layer], (kr, v[at:at + c])))
                want, tol = attention(qr[at:at + c], *rows[s][layer], n0, dim ** -0.5, 100 if layer == 0 else 0,
                                      sinks if layer == 0 else None, gate[at:at + c] if layer else None)
                close(out[at:at + c], want, tol, f"layer {layer} sequence {s}")
                at += c

    def cut(s, n):
        kv.set_len(s, n)
        rows[s] = [(k[:n], v[:n]) for k, v in rows[s]]

    step([0, 1], [77, 200])
    kv.fork([1, 1], [2, 3], [200, 130])
    rows[2], rows[3] = list(rows[1]), [(k[:130], v[:130]) for k, v in rows[1]]
    for i in range(6):  # drafts of 3 verified with the token before them; some are taken back
        seqs = [0, 1, 2, 3]
        step(seqs, [4] * 4)
        for s in seqs:
            cut(s, kv.length(s) - (i + s) % 4)
    cut(2, 150)  # inside a page that is shared: it is copied
    step([2, 3, 1], [1, 1, 1])
    kv.free([0])
    rows[0] = [(none, none)] * 2
    assert kv.compact() > 0
    step([1, 2, 3], [1, 2, 1])
    step([0, 1, 4], [300, 1, 33])
    step([0, 4], [45, 1])
    kv.copy([0], [5])
    rows[5] = list(rows[0])
    step([5, 0], [1, 1])
    kv.close()


# ---- graphs and streams ----

@pytest.mark.parametrize("typ,dim", [("f16", 128), ("bf16", 256)])
def test_captured_layers_follow_the_batch(torch_gpu, pg, typ, dim):
    """append and attend of two layers captured once; replays after other mpg_begins do those batches, bit for bit as eager
    calls do, with eager work between them; tokens behind the captured rows are left out; with no batch standing a replay
    writes nothing."""
    torch = torch_gpu
    fmt, t = types(torch, pg)[typ]
    heads, group, rows = 2, 8, 600
    kv = pg.PagedKv(2, heads * group, heads, dim, 300, page=32, seqs=6, ctx=8192, fmt=fmt, windows=[0, 130],
                    rope=pg.Rope(64))
    x = torch.zeros(rows, heads * (group + 2), dim, dtype=t, device="cuda")
    q, k, v = x[:, :heads * group], x[:, heads * group:heads * (group + 1)], x[:, heads * (group + 1):]
    qr = [torch.empty(rows, heads * group, dim, dtype=t, device="cuda") for _ in (0, 1)]
    out = [torch.full((rows, heads * group, dim), 3.0, dtype=t, device="cuda") for _ in (0, 1)]

    def layers(outs):
        for layer in (0, 1):
            kv.append(layer, k, v, q, q_out=qr[layer])
            kv.attend(layer, qr[layer], out=outs[layer])

    kv.begin([0, 1], [1500, 3])
    kv.begin([0], [1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    base = torch.cuda.current_stream()
    with torch.cuda.graph(g):
        kv.set_stream(torch.cuda.current_stream())
        layers(out)
    kv.set_stream(base)
    other = [torch.empty_like(o) for o in out]
    for i, (seqs, counts) in enumerate([([0], [1]), ([1, 0], [4, 1]), ([2, 0, 3], [400, 1, 33]), ([0, 1, 2, 3], [1, 1, 1, 1]),
                                        ([4], [600]), ([3, 4], [2, 1])]):
        kv.begin(seqs, counts)
        x.copy_(rnd(torch, 50 + i, *x.shape, dtype=t))
        layers(other)  # eager
        n = sum(counts)
        want = [o[:n].clone() for o in other] + [kv.read_rows(layer, w, s) for layer in (0, 1) for w in (0, 1) for s in seqs]
        for _ in range(3):
            for o in out:
                o.fill_(3.0)
            g.replay()
            torch.cuda.synchronize()
            got = [o[:n] for o in out] + [kv.read_rows(layer, w, s) for layer in (0, 1) for w in (0, 1) for s in seqs]
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i
            assert all((o[n:] == 3).all() for o in out)
            (torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")).sum().item()
    kv.begin([5], [rows + 7])  # more tokens than the captured rows
    g.replay()
    torch.cuda.synchronize()
    kv.free([5])
    for o in out:
        o.fill_(3.0)
    before = [kv.pages(layer, w).clone() for layer in (0, 1) for w in (0, 1)]
    g.replay()
    torch.cuda.synchronize()
    assert all((o == 3).all() for o in out)
    assert all(torch.equal(a, kv.pages(layer, w)) for a, (layer, w) in zip(before, [(0, 0), (0, 1), (1, 0), (1, 1)]))
    kv.close()


def test_page_calls_are_refused_while_capturing(torch_gpu, pg):
    torch = torch_gpu
    kv = pg.PagedKv(1, 2, 1, 64, 20, page=32, seqs=4, ctx=1024)
    kv.begin([0], [5])
    k = rnd(torch, 1, 5, 1, 64, dtype=torch.float16)
    kv.append(0, k, k)
    kv.read_rows(0, 0, 0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    base = torch.cuda.current_stream()
    with torch.cuda.graph(g):
        kv.set_stream(torch.cuda.current_stream())
        for call in (lambda: kv.begin([0], [1]), lambda: kv.reserve([0], [1]), lambda: kv.set_len(0, 1), lambda: kv.free([0]),
                     lambda: kv.fork([0], [1]), lambda: kv.copy([0], [1]), kv.compact):
            with pytest.raises(pg.MkvError) as e:
                call()
            assert e.value.code == -1 and "capturing" in str(e.value)
        y = kv.read_rows(0, 0, 0)
    kv.set_stream(base)
    assert kv.length(0) == 5
    for _ in range(3):
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, k)
    kv.close()


def test_two_caches_on_two_streams(torch_gpu, pg):
    """Each cache has workspaces of its own: split attention of two at once."""
    torch = torch_gpu
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    models = []
    for s in (a, b):
        with torch.cuda.stream(s):
            m = Model(torch, pg, 2, 8, 128, "bf16", 64, pages=400, tokens=16384)
            m.step([0, 1], [6000, 5000])
            m.step([0, 1], [1, 3])
            m.q = rnd(torch, 3, 4, 16, 128, dtype=torch.bfloat16)
            m.want = m.kv.attend(0, m.q)
            models.append(m)
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for s, m in zip((a, b), models):
            with torch.cuda.stream(s):
                outs.append((m, m.kv.attend(0, m.q)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, m.want) for m, o in outs)
    for m in models:
        m.kv.close()


def test_results_do_not_depend_on_the_pages(torch_gpu, pg):
    """The same sequence on other pages, beside other sequences: bit for bit, where the split is the same."""
    torch = torch_gpu
    m = Model(torch, pg, 2, 8, 128, "f16", 32)
    m.step([0], [700])
    m.kv.reserve([5], [100])
    m.kv.copy([0], [1])
    m.kv.free([5])
    m.kv.fork([1], [2], [650])
    q = rnd(torch, 3, 1, 16, 128, dtype=torch.float16)
    k = rnd(torch, 4, 1, 2, 128, dtype=torch.float16)
    outs = []
    for s in (0, 1):
        m.kv.begin([s], [1])
        m.kv.append(0, k, k)
        outs.append(m.kv.attend(0, q))
        outs.append(m.kv.attend(0, q))
    assert all(torch.equal(o, outs[0]) for o in outs)
    m.kv.close()


# ---- refusals ----

def test_refusals(torch_gpu, pg):
    torch = torch_gpu
    E = pg.MkvError
    good = dict(layers=2, q_heads=4, kv_heads=2, head_dim=64, pages=8, page=32, seqs=3, ctx=200)
    for bad, code in [(dict(layers=0), -1), (dict(q_heads=3), -1), (dict(kv_heads=0), -1), (dict(head_dim=96), -1),
                      (dict(pages=0), -1), (dict(page=16), -1), (dict(page=48), -1), (dict(seqs=0), -1), (dict(ctx=0), -2),
                      (dict(ctx=4194305), -2), (dict(tokens=0), -1), (dict(fmt=1), -1), (dict(fmt=7), -1),
                      (dict(windows=[0, -1]), -1), (dict(rope=pg.Rope(128)), -1)]:
        with pytest.raises(E) as e:
            pg.PagedKv(**{**good, **bad})
        assert e.value.code == code, bad
    with pytest.raises(E) as e:
        pg.PagedKv(**{**good, "layers": 5}, windows=[1, 2, 3, 4, 5])
    assert e.value.code == -1
    with pytest.raises(ValueError):
        pg.PagedKv(**good, windows=[1])
    kv = pg.PagedKv(**good, tokens=40)
    h = torch.float16
    k = torch.zeros(5, 2, 64, dtype=h, device="cuda")
    q = torch.zeros(5, 4, 64, dtype=h, device="cuda")
    with pytest.raises(E, match="no batch"):
        kv.append(0, k, k)
    with pytest.raises(E, match="no batch"):
        kv.attend(0, q)
    with pytest.raises(E, match="at most 40"):
        kv.begin([0], [41])
    assert kv.length(0) == 0
    kv.begin([0], [5])
    for call, code in [(lambda: kv.append(2, k, k), -4), (lambda: kv.append(-1, k, k), -4), (lambda: kv.attend(2, q), -4),
                       (lambda: kv.append(0, k[:4], k[:4]), -5), (lambda: kv.attend(0, q[:4]), -5),
                       (lambda: kv.append(0, k, k, rotate=True), -1), (lambda: kv.append(0, k, k, q), -1),
                       (lambda: kv.attend(0, q, scale=0.0), -1), (lambda: kv.attend(0, q, scale=-1.0), -1),
                       (lambda: kv.attend(0, q, scale=math.inf), -1), (lambda: kv.attend(0, q, scale=math.nan), -1),
                       (lambda: kv.read_rows(0, 0, 0, 0, 6), -3), (lambda: kv.read_rows(0, 0, 3), -1),
                       (lambda: kv.read_rows(0, 2, 0), -1), (lambda: kv.length(3), -1), (lambda: kv.table(-1), -1),
                       (lambda: kv.begin([0, 0], [1, 1]), -1), (lambda: kv.begin([0], [196]), -1),
                       (lambda: kv.reserve([0], [196]), -3), (lambda: kv.reserve([1, 2], [200, 100]), -7)]:
        with pytest.raises(E) as e:
            call()
        assert e.value.code == code
    for call in (lambda: kv.append(0, k.float(), k), lambda: kv.append(0, k, k[:, :1]), lambda: kv.append(0, k.cpu(), k),
                 lambda: kv.attend(0, q.to(torch.bfloat16)), lambda: kv.attend(0, q[:, :, ::2]),
                 lambda: kv.attend(0, q, sinks=torch.zeros(4)), lambda: kv.attend(0, q, out=q[:3]),
                 lambda: kv.begin([0], [1, 2]), lambda: kv.attend(0, q, gate=q[:3]), lambda: kv.fork([0], [1, 2])):
        with pytest.raises(ValueError):
            call()
    odd = torch.zeros(5 * 4 * 64 + 4, dtype=h, device="cuda")[4:].view(5, 4, 64)
    with pytest.raises(E, match="aligned"):
        kv.attend(0, odd)
    with pytest.raises(E, match="aligned"):
        kv.attend(0, torch.zeros(5, 4, 68, dtype=h, device="cuda")[..., :64])
    assert kv.attend(0, q).shape == q.shape  # the batch still stands
    kv.reserve([1], [1])
    with pytest.raises(E, match="no batch"):
        kv.attend(0, q)
    assert kv.begin([], []) == 0 and kv.attend(0, q[:0]).shape == (0, 4, 64)
    kv.append(0, k[:0], k[:0])
    assert kv.begin([0, 1], [0, 0]) == 0
    kv.close()
    x = torch.zeros(3, 2, 64, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    rope = pg.Rope(64)
    for call in (lambda: pg.rotate(x, pos.long(), rope), lambda: pg.rotate(x, pos[:2], rope), lambda: pg.rotate(x.double(), pos, rope),
                 lambda: pg.rotate(x, pos.cpu(), rope), lambda: pg.rotate(x, pos, rope, out=x[:2]), lambda: pg.rotate(x[0], pos, rope)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(E):
        pg.rotate(x[..., :32], pos, rope)
    # at the C entry: in place with other strides
    lib, P = pg.lib(), ctypes.c_void_p
    assert lib.mpg_rotate(rope._ptr, 1, 3, 2, 64, P(x.data_ptr()), 128, 64, P(pos.data_ptr()), P(x.data_ptr()), 64,
                          192, None) == -1
