"""NaN that a row sees only in a part of its keys with no weight of its own, a piece whose only key for the row has a NaN
score, reaches the row all the same."""
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
