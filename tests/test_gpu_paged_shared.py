"""Batches begun as shared on the GPU: forks of a prompt, and of each other, against the plain 64-bit form over each
sequence's own rows (tests/paged_reference.py)."""
import math
import random

import pytest

from tests.paged_forests import FORESTS
from tests.paged_reference import attention, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pg(torch_gpu):
    from mechta_amd import paged
    return paged


class Forest:
    """A one-layer cache of sequences that are forked, and beside it each sequence's rows."""

    def __init__(self, torch, pg, kv_heads, group, dim, typ, page, pages=400, seqs=64, window=0, ctx=100000, **more):
        self.torch = torch
        self.fmt, self.type = {"f16": (pg.F16, torch.float16), "bf16": (pg.BF16, torch.bfloat16)}[typ]
        self.kv = pg.PagedKv(1, kv_heads * group, kv_heads, dim, pages, page=page, seqs=seqs, ctx=ctx, fmt=self.fmt,
                             windows=[window], **more)
        self.heads, self.group, self.dim, self.window = kv_heads, group, dim, window
        self.rows = {s: (torch.zeros(0, kv_heads, dim, dtype=self.type, device="cuda"),) * 2 for s in range(seqs)}
        self.g = torch.Generator(device="cuda").manual_seed(7)
        for w in (0, 1):
            self.kv.pages(0, w).fill_(math.nan)  # what is not written must not matter

    def rnd(self, *shape):
        return self.torch.randn(shape, generator=self.g, device="cuda").to(self.type)

    def begin(self, seqs, counts, shared):
        n = self.kv.begin(seqs, counts, shared=shared)
        k, v = self.rnd(n, self.heads, self.dim), self.rnd(n, self.heads, self.dim)
        if n:
            self.kv.append(0, k, v)
        at = 0
        for s, c in zip(seqs, counts):
            self.rows[s] = tuple(self.torch.cat((a, b[at:at + c])) for a, b in zip(self.rows[s], (k, v)))
            at += c
        self.batch = (seqs, counts)
        return n

    def grow(self, seqs, counts):
        for i in range(0, len(seqs), 4):
            self.begin(seqs[i:i + 4], counts[i:i + 4], False)

    def fork(self, src, dst, lens=None):
        self.kv.fork(src, dst, lens)
        for i, (a, b) in enumerate(zip(src, dst)):
            self.rows[b] = tuple(x[:lens[i]] if lens else x for x in self.rows[a])

    def check(self, sinks=None, gate=False, q=None, out=None, what=""):
        seqs, counts = self.batch
        n, h = sum(counts), self.heads * self.group
        q = self.rnd(n, h, self.dim) if q is None else q
        g = self.rnd(n, h, self.dim) if gate else None
        out = self.kv.attend(0, q, sinks=sinks, gate=g) if out is None else out
        at = 0
        for s, c in zip(seqs, counts):
            k, v = self.rows[s]
            if c:
                want, tol = attention(q[at:at + c], k, v, len(k) - c, self.dim ** -0.5, self.window, sinks,
                                      g[at:at + c] if gate else None)
                # a shared batch puts a few more partial sums together: each a rounding of 2^-24 of the values' size
                close(out[at:at + c], want, tol, f"{what} sequence {s}, {c} tokens of {len(k)}")
            at += c
        return out


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("name", FORESTS)
def test_forks_of_a_prompt(torch_gpu, pg, name, typ):
    torch = torch_gpu
    heads, group, dim, page, prompt, forks, own, tokens, window, _ = FORESTS[name]
    f = Forest(torch, pg, heads, group, dim, typ, page, pages=(prompt + forks * (own + 600)) // page + 100, window=window)
    for at in range(0, prompt, 8000):
        f.grow([0], [min(8000, prompt - at)])
    f.fork([0] * (forks - 1), list(range(1, forks)))
    r = random.Random(3)
    f.grow(list(range(forks)), [r.randint(1, own) for _ in range(forks)])
    seqs = r.sample(range(forks), forks)
    f.begin(seqs, [tokens[i % len(tokens)] for i in range(forks)], True)
    sinks = torch.randn(heads * group, generator=f.g, device="cuda")
    f.check(what=name)
    f.check(sinks=sinks, gate=True, what=name)


@pytest.mark.parametrize("typ,dim,page,window", [("f16", 128, 32, 0), ("bf16", 64, 64, 3900), ("f16", 256, 32, 0)])
def test_a_tree_of_forks(torch_gpu, pg, typ, dim, page, window):
    f = Forest(torch_gpu, pg, 2, 8, dim, typ, page, pages=1800, window=window)
    f.grow([0], [7100])
    f.fork([0] * 3, [1, 2, 3])
    f.grow([0, 1, 2, 3], [2500, 2700, 33, 1640])
    f.fork([s % 4 for s in range(4, 16)], list(range(4, 16)))
    f.grow(list(range(16)), [300 + s for s in range(16)])
    f.fork([s % 16 for s in range(16, 40)], list(range(16, 40)), [7200 + 5 * s for s in range(16, 40)])
    r = random.Random(1)
    for step in range(3):
        seqs = r.sample(range(40), 30)
        f.begin(seqs, [r.choice([1, 1, 2, 5]) for _ in seqs], True)
        f.check(gate=step == 1, what=f"step {step}")


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("forks", [24, 60])  # in tiles of 32 rows, of 128
def test_odd_values_behind_a_shared_window(torch_gpu, pg, typ, forks):
    """Infinities and NaN of the prompt in front of a row's window do not reach it; those inside reach the rows that see them."""
    torch = torch_gpu
    f = Forest(torch, pg, 4, 8, 64, typ, 32, pages=1500, window=5000)
    f.grow([0], [6400])
    f.fork([0] * (forks - 1), list(range(1, forks)))
    f.grow(list(range(forks)), [10 + 20 * (i % 7) for i in range(forks)])
    seqs = list(range(forks))
    random.Random(2).shuffle(seqs)
    f.begin(seqs, [1] * forks, True)
    assert f.kv.table(0)[:200] == f.kv.table(4)[:200]
    at = 1472  # seen by rows at positions up to 6,471
    page = f.kv.table(0)[at // 32]
    v = f.kv.pages(0, pg.V).view(-1, 4, 1, 4, 64, 2, 4)
    for value in (math.nan, math.inf):
        v[page, 1, 0, 0, :, 0, 0] = value
        q = f.rnd(forks, 32, 64)
        out = f.kv.attend(0, q)
        sees = [f.kv.length(s) - 1 - 5000 < at for s in seqs]
        assert set(sees) == {True, False}
        for i in range(forks):
            assert torch.isfinite(out[i, :8]).all() and torch.isfinite(out[i, 16:]).all()
            assert not torch.isfinite(out[i, 8:16]).any() if sees[i] else torch.isfinite(out[i, 8:16]).all(), i


def test_captured_attention_follows_shared_batches(torch_gpu, pg):
    """A graph captured under either kind of batch does whatever batch stands when it is replayed."""
    torch = torch_gpu
    for first_shared in (False, True):
        stream = torch.cuda.Stream()
        f = Forest(torch, pg, 2, 8, 128, "bf16", 64, stream=torch.cuda.current_stream(), tokens=8192)
        f.grow([0], [8000] if first_shared else [7900])
        f.grow([0], [512])
        f.fork([0] * 39, list(range(1, 40)))
        rows = 64
        q, out = f.rnd(rows, 16, 128), torch.zeros(rows, 16, 128, dtype=f.type, device="cuda")
        f.begin(list(range(8)), [1] * 8, first_shared)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        f.kv.set_stream(stream)
        with torch.cuda.graph(graph, stream=stream):
            f.kv.attend(0, q, out=out)
        f.kv.set_stream(torch.cuda.current_stream())
        for seqs, counts, shared in [(list(range(20)), [1] * 20, True), ([3, 1], [4, 1], False), (list(range(39, -1, -1)), [1] * 40, True),
                                     (list(range(16)), [2] * 16, False), ([5], [1], True), (list(range(16)), [4] * 16, True)]:
            n = f.begin(seqs, counts, shared)
            eager = f.kv.attend(0, q[:n].contiguous())
            out.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[:n], eager) and (out[n:] == 7).all()
            f.check(q=q[:n], out=eager, what=f"{shared}")


def test_shared_batches_are_repeatable_and_near_the_plain_ones(torch_gpu, pg):
    torch = torch_gpu
    f = Forest(torch, pg, 2, 8, 128, "f16", 64)
    f.grow([0], [8100])
    f.fork([0] * 29, list(range(1, 30)))
    f.begin(list(range(30)), [1] * 30, True)
    q = f.rnd(30, 16, 128)
    a, b = f.kv.attend(0, q), f.kv.attend(0, q)
    assert torch.equal(a, b)
    f.kv.begin(list(range(30)), [0] * 30, shared=True)  # nothing new: nothing to attend
    assert f.kv.attend(0, q[:0]).shape == (0, 16, 128)


def test_refusals(torch_gpu, pg):
    f = Forest(torch_gpu, pg, 1, 1, 64, "f16", 32, pages=8, seqs=4, tokens=10)
    for seqs, counts, code in [([0, 0], [1, 1], -1), ([4], [1], -1), ([0], [-1], -1), ([0], [11], -1), ([0, 1], [6, 6], -1)]:
        with pytest.raises(pg.MkvError) as e:
            f.kv.begin(seqs, counts, shared=True)
        assert e.value.code == code
    with pytest.raises(ValueError, match="2 needed"):
        f.kv.begin([0, 1], [1], shared=True)
    assert [f.kv.length(s) for s in range(4)] == [0] * 4 and f.kv.free_pages() == 8
