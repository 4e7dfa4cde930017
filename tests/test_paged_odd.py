"""NaN and infinities that a row sees only in a part of its keys with no weight of its own: a piece whose only key for the row
has a NaN score, pieces and waves whose weights are all too small for 32 bits. They reach the row all the same."""
import math

import pytest

from tests.paged_reference import attention, close
from tests.test_gpu_paged import pg, rnd, types  # noqa: F401
from tests.test_gpu_paged_shapes import element
from tests.test_paged_book import TILE, make_plan, shim  # noqa: F401

# dim, kv_heads, window, new tokens, length; one query head per K/V head
ALONE = [(64, 1, 0, 128, 1128), (64, 1, 0, 128, 4128), (64, 1, 0, 128, 8128), (256, 8, 0, 512, 512), (64, 1, 1000, 128, 4128),
         (64, 1, 513, 256, 4128), (128, 2, 300, 256, 4000)]


def test_some_rows_see_one_key_of_a_piece(shim):
    """The batches below are cut so that a row has a single key in a piece, at a multiple of 32 or right before one."""
    for dim, kv, window, count, n in ALONE:
        items, joins = make_plan(shim, kv, kv, dim, [(0, count, n)], window)
        alone = set()
        for kind in range(4):
            for _, _, _, row0, rows, pos0, k0, k1, part in items[kind]:
                for p in range(pos0 + row0, pos0 + min(rows, row0 + TILE[kind])):
                    lo, hi = max(k0, p - window + 1 if window else 0), min(k1 - 1, p)
                    if part >= 0 and lo == hi:
                        alone.add(lo)
        assert joins and alone and all(x % 32 in (0, 31) for x in alone), (dim, kv, window)


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim,kv_heads,window,count,n", ALONE)
def test_a_nan_score_alone_in_a_piece(torch_gpu, pg, typ, dim, kv_heads, window, count, n):
    torch = torch_gpu
    fmt, t = types(torch, pg)[typ]
    with pg.PagedKv(1, kv_heads, kv_heads, dim, n // 64 + 1, page=64, seqs=1, ctx=n, fmt=fmt, tokens=n,
                    windows=[window]) as kv:
        k, v = (rnd(torch, i, n, kv_heads, dim, dtype=t) for i in (1, 2))
        for at, c in ((0, n - count), (n - count, count)):
            if c:
                kv.begin([0], [c])
                kv.append(0, k[at:at + c], v[at:at + c])
        q = rnd(torch, 3, count, kv_heads, dim, dtype=t)
        clean = kv.attend(0, q)
        close(clean, *attention(q, k, v, n - count, dim ** -0.5, window))
        pos = torch.arange(n - count, n, device="cuda")
        first = max(0, n - count - window + 1) if window else n - count
        for x in range(first // 32 * 32, n):
            if x < first or x % 32 not in (0, 31):
                continue
            e = element(kv, 0, 0, x, kv_heads - 1, 7)
            e.fill_(math.nan)
            out = kv.attend(0, q)
            e.copy_(k[x, kv_heads - 1, 7])
            hit = torch.zeros_like(out, dtype=torch.bool)
            hit[:, -1] = ((pos >= x) & ((pos - window < x) if window else (pos >= 0)))[:, None]
            assert torch.isnan(out[hit]).all(), x
            assert torch.equal(out[~hit], clean[~hit]), x


# dim, kv_heads, group, new tokens, length, kind of tile, split over the keys
FAINT = [(64, 1, 4, 1, 300, 0, False), (128, 2, 8, 1, 3000, 0, True), (128, 1, 8, 1, 40000, 0, True), (256, 2, 8, 4, 200, 1, False),
         (256, 2, 8, 4, 9000, 1, True), (64, 8, 16, 400, 600, 3, False), (64, 8, 4, 300, 4000, 3, True), (128, 2, 8, 40, 9001, 2, True), (256, 2, 8, 300, 400, 2, False),
         (64, 1, 16, 200, 9001, 2, True), (256, 2, 8, 512, 9512, 2, True)]


def test_faint_batches_go_to_their_kernels(shim):
    for dim, kv, group, count, n, kind, split in FAINT:
        items, joins = make_plan(shim, kv * group, kv, dim, [(0, count, n)], 0)
        assert items[kind] and bool(joins) == split, (dim, count, n, [len(i) for i in items], len(joins))


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim,kv_heads,group,count,n,kind,split", FAINT)
def test_odd_values_of_weights_too_small(torch_gpu, pg, typ, dim, kv_heads, group, count, n, kind, split):
    """Every earlier position has a score 4 dim below the new ones' 0: e^-256 at most, zero in 32 bits, and zero times NaN or
    an infinity is NaN. A weight of exactly e^-256 would make an infinity infinite: one or the other, and never a finite row."""
    torch = torch_gpu
    fmt, t = types(torch, pg)[typ]
    with pg.PagedKv(1, kv_heads * group, kv_heads, dim, n // 64 + 1, page=64, seqs=1, ctx=n, fmt=fmt, tokens=n) as kv:
        k = torch.zeros(n, kv_heads, dim, dtype=t, device="cuda")
        k[:n - count] = -4
        v = rnd(torch, 2, n, kv_heads, dim, dtype=t)
        for at, c in ((0, n - count), (n - count, count)):
            kv.begin([0], [c])
            kv.append(0, k[at:at + c], v[at:at + c])
        q = torch.ones(count, kv_heads * group, dim, dtype=t, device="cuda")
        clean = kv.attend(0, q, scale=1.0)
        close(clean, *attention(q, k, v, n - count, 1.0))
        old = n - count
        for x in sorted({0, 31, old // 3, old // 2, old - 70, old - 33, old - 1} & set(range(old))):
            for value in (math.nan, math.inf):
                e = element(kv, 1, 0, x, kv_heads - 1, 7)
                e.fill_(value)
                out = kv.attend(0, q, scale=1.0)
                e.copy_(v[x, kv_heads - 1, 7])
                hit = torch.zeros_like(out, dtype=torch.bool)
                hit[:, (kv_heads - 1) * group:, 7] = True
                assert not torch.isfinite(out[hit]).any(), (x, value)
                if math.isnan(value):
                    assert torch.isnan(out[hit]).all(), x
                assert torch.equal(out[~hit], clean[~hit]), (x, value)
