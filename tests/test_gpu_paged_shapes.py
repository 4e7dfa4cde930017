"""The paged cache's kernels over batches that reach each of them (tests/paged_shapes.py): attention against the 64-bit
form, values that no row may see, captured calls, large rotations, another current stream."""
import math

import pytest

from tests.paged_reference import attention, close, rope_freqs, rotated
from tests.paged_shapes import SHAPES
from tests.test_gpu_paged import Model, pg, rnd  # noqa: F401

pytestmark = pytest.mark.gpu


def model(torch, pg, name, typ, page):
    """The batch of a shape, begun, its earlier positions written."""
    dim, kv, group, window, batch, _, _ = SHAPES[name]
    m = Model(torch, pg, kv, group, dim, typ, page, pages=sum(n // page + 1 for _, n in batch) + 5, seqs=len(batch),
              window=window, tokens=sum(n for _, n in batch))
    m.foul()
    seqs = list(range(len(batch)))
    if any(n > c for c, n in batch):
        m.step(seqs, [n - c for c, n in batch])
    m.step(seqs, [c for c, _ in batch])
    return m


@pytest.mark.parametrize("typ,page", [("f16", 32), ("bf16", 128)])
@pytest.mark.parametrize("name", SHAPES)
def test_attend_shapes(torch_gpu, pg, name, typ, page):
    m = model(torch_gpu, pg, name, typ, page)
    m.check(out_rows=3, what=name)
    m.check(sinks=rnd(torch_gpu, 5, m.heads * m.group, scale=2.0), gate=True, strided=True, what=f"{name}, sinks and gate")
    m.kv.close()


def element(kv, which, seq, pos, head, d):
    """The place in the pages of an element of a sequence's K or V, as a tensor of no dimensions."""
    p, x = kv.table(seq)[pos // kv.page], pos % kv.page
    pages = kv.pages(0, which)
    if which == 0:
        return pages[p, head, x // 16, d // 8, x % 16, d % 8]
    y = x % 32
    return pages[p, head, x // 32, y % 16 // 4, d, y // 16 * 4 + y % 4]


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("name,seq", [("large tiles split, 128", 1), ("prompts of large tiles, 64", 1),
                                      ("prompts of large tiles, 256", 0), ("chunk of 40, many splits", 0),
                                      ("prompt of small tiles", 0), ("four tokens, many splits", 0), ("uneven tokens", 3),
                                      ("large tiles split, 256", 1)])
def test_odd_values_in_shapes(torch_gpu, pg, name, seq, typ):
    """NaN and infinities at a position reach the rows that see it and change no other row, bit for bit."""
    torch = torch_gpu
    dim, kv, group, window, batch, _, _ = SHAPES[name]
    m = model(torch, pg, name, typ, 64)
    tokens = sum(c for c, _ in batch)
    q = rnd(torch, 77, tokens, kv * group, dim, dtype=m.fmt[1])
    clean = m.kv.attend(0, q)
    count, n = batch[seq]
    first, head = sum(c for c, _ in batch[:seq]), kv - 1
    pos = torch.arange(n - count, n, device="cuda")
    at = sorted({n - 1, n - 2, n - 1 - count // 3, n - count, max(0, n - count - 40), max(0, n - 1 - count - window // 2), n // 2})
    for i, x in enumerate(at):
        for which, value in ((1, math.nan), (1, -math.inf if i % 2 else math.inf), (0, math.nan)):
            e = element(m.kv, which, seq, x, head, 7)
            assert torch.equal(e, m.rows[seq][which][x, head, 7])  # the place is the one meant
            e.fill_(value)
            out = m.kv.attend(0, q)
            e.copy_(m.rows[seq][which][x, head, 7])
            sees = (pos >= x) & ((pos - window < x) if window else (pos >= 0))
            hit = torch.zeros_like(out, dtype=torch.bool)
            rows = slice(first, first + count), slice(head * group, (head + 1) * group)
            if which:
                hit[rows[0], rows[1], 7] = sees[:, None]
            else:
                hit[rows[0], rows[1]] = sees[:, None, None]
            assert torch.equal(out[~hit], clean[~hit]), (x, which, value)
            if math.isnan(value):
                assert torch.isnan(out[hit]).all(), (x, which)
            else:
                assert (out[hit] == value).all(), (x, value)
    assert torch.equal(m.kv.attend(0, q), clean)
    m.kv.close()


def test_captured_attention_of_every_kernel(torch_gpu, pg):
    """One captured call, replayed over batches of every kernel of its head size: each replay equals the eager call."""
    torch = torch_gpu
    rows, kv_heads, group, dim = 1400, 2, 8, 128
    m = Model(torch, pg, kv_heads, group, dim, "bf16", 64, pages=1200, seqs=8, tokens=40000)
    q = torch.zeros(rows, kv_heads * group, dim, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros_like(q)
    m.step(list(range(6)), [20000, 9000, 2101, 666, 50, 3000])
    m.step([4], [1])
    torch.cuda.synchronize()
    base, g = torch.cuda.current_stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.kv.set_stream(torch.cuda.current_stream())
        m.kv.attend(0, q, out=out)
    m.kv.set_stream(base)
    for seqs, counts in [([0], [1]), ([4, 2, 3, 6], [42, 831, 399, 41]), ([1], [40]), ([0], [4]), ([5, 7], [1, 1300]),
                         ([0, 1, 5], [1, 1, 1]), ([0], [16])]:
        m.step(seqs, counts)
        n = sum(counts)
        q[:n].copy_(rnd(torch, n, n, *q.shape[1:], dtype=torch.bfloat16))
        eager = torch.zeros_like(out)
        m.kv.attend(0, q, out=eager)
        for _ in range(3):
            out.fill_(2.0)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[:n], eager[:n]) and (out[n:] == 2).all(), (seqs, counts)
            rnd(torch, 1, 1 << 20).sum().item()  # eager work between replays
    m.kv.close()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim", [128, 96])
def test_large_rotation(torch_gpu, pg, layout, dim):
    """More than the L2s hold."""
    torch = torch_gpu
    x = rnd(torch, 3, 8203, 16, 128, dtype=torch.bfloat16)
    pos = torch.randint(0, 4194304, (8203,), device="cuda", dtype=torch.int32)
    rope = pg.Rope(dim, layout=layout, base=1e6)
    y = pg.rotate(x, pos, rope)
    for at in range(0, 8203, 1024):
        want, tol = rotated(x[at:at + 1024], pos[at:at + 1024], dim, layout, *rope_freqs(dim, 1e6))
        close(y[at:at + 1024], want, tol, f"rows from {at}")
    assert pg.rotate(x, pos, rope, out=x) is x and torch.equal(x, y)


def test_more_rows_than_a_launch_takes(torch_gpu, pg):
    torch = torch_gpu
    n = (1 << 25) + 5
    x = rnd(torch, 3, n, 1, 2, dtype=torch.float16)
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    rope = pg.Rope(2)
    y = pg.rotate(x, pos, rope)
    for at in (0, (1 << 25) - 1000, n - 1000):
        close(y[at:at + 1000], *rotated(x[at:at + 1000], pos[at:at + 1000], 2, "half", *rope_freqs(2, 1e4)), f"rows from {at}")


def test_another_current_stream(torch_gpu, pg):
    """A cache on a stream of its own, its outputs made and used on torch's current one, ordered by the caller."""
    torch = torch_gpu
    own, cur = torch.cuda.Stream(), torch.cuda.current_stream()
    heads, group, dim = 2, 4, 128
    rope = pg.Rope(64)
    kvs = [pg.PagedKv(1, heads * group, heads, dim, 100, seqs=2, rope=rope, **k) for k in (dict(stream=own), {})]
    for i in range(12):
        n = [700, 1, 33][i % 3]
        q, k, v = (rnd(torch, 10 * i + j, n, h, dim, dtype=torch.float16) for j, h in enumerate((heads * group, heads, heads)))
        got = []
        for kv in kvs:
            own.wait_stream(cur)
            kv.begin([i % 2], [n])
            qr = kv.append(0, k, v, q)
            out = kv.attend(0, qr)
            rows = kv.read_rows(0, 0, i % 2)
            cur.wait_stream(own)
            got.append((qr, out, rows))
        assert all(torch.equal(a, b) for a, b in zip(*got))
    for kv in kvs:
        kv.close()


def test_more_refusals(torch_gpu, pg):
    torch = torch_gpu
    with pg.PagedKv(1, 4, 2, 64, 8, seqs=2) as kv:
        kv.begin([0], [3])
        x = rnd(torch, 1, 3, 4, 64, dtype=torch.float16)
        with pytest.raises(pg.MkvError, match="place of an input"):
            kv.attend(0, x, out=x)
        gate = x.clone()
        with pytest.raises(pg.MkvError, match="place of an input"):
            kv.attend(0, x, gate=gate, out=gate)
    g = torch.cuda.CUDAGraph()
    y = torch.zeros(4, device="cuda")
    with torch.cuda.graph(g):
        y += 1
        with pytest.raises(pg.MkvError, match="capturing"):
            pg.PagedKv(1, 4, 2, 64, 8)
    g.replay(), g.replay()
    assert (y == 2).all()
