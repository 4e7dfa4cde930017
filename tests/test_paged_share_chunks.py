"""Batches of forks beside chunks (no GPU): few rows may go among a chunk's tiles, and what forks share with them; each tile begins
where its kind's tiles do, so that no score is taken twice."""
import random

import pytest

from tests.test_paged_share import TILE, Forest, check, planned, shim  # noqa: F401

# name: kv_heads, group, dim, page, prompt, forks, own part, tokens each, [(tokens, positions before them) of the others], window
BESIDE_CHUNKS = {
    "37 forks, two tokens each": (8, 1, 64, 128, 1152, 37, 8, 2, [(100, 200)], 0),
    "20 forks, heads of 64 in fours": (8, 4, 64, 64, 2000, 20, 100, 1, [(40, 1500), (300, 1500), (100, 1500)], 0),
    "32 forks, heads of 128, a window": (8, 2, 128, 64, 1152, 32, 100, 1, [(100, 200), (300, 1500), (100, 1500)], 1300),
    "23 forks, heads of 256, a window": (8, 2, 256, 32, 8000, 23, 8, 1, [(300, 1500), (40, 200), (100, 1500)], 1300),
    "32 rows of 10 forks": (8, 3, 64, 64, 2000, 10, 30, 1, [(100, 1500)], 0),
}


def forks_and_chunks(L, name):
    """The forks of a prompt, each with a part of its own, and behind them sequences of their own; counts of new tokens."""
    kv, group, dim, page, prompt, forks, own, tokens, chunks, window = BESIDE_CHUNKS[name]
    f = Forest(L, page, seqs=forks + len(chunks))
    f.grow([0], [prompt])
    if forks > 1:
        f.fork([0] * (forks - 1), list(range(1, forks)))
    f.grow(list(range(forks)), [own] * forks)
    others = list(range(forks, forks + len(chunks)))
    f.grow(others, [c[1] for c in chunks])
    return f, (kv, group, dim, list(range(forks)) + others, [tokens] * forks + [c[0] for c in chunks], window)


def aligned(items):
    return all(row0 % TILE[kind] == 0 for kind, list_ in enumerate(items) for _, _, _, row0, *_ in list_)


@pytest.mark.parametrize("name", BESIDE_CHUNKS)
def test_what_forks_share_among_a_chunks_tiles(shim, name):  # noqa: F811
    f, batch = forks_and_chunks(shim, name)
    ranges, shared, kinds = check(f, *batch)
    assert ranges == 1 and shared and kinds == (2,)
    f.close()
    f, batch = forks_and_chunks(shim, name)
    _, items, *_ = planned(f, *batch)
    assert aligned(items) and not items[0] and not items[1]  # few rows are there too
    f.close()


@pytest.mark.parametrize("seed", range(12))
def test_forks_and_chunks(shim, seed):  # noqa: F811
    """Of few heads and short prompts, where the ways to cut a batch cost about the same: 50 batches each."""
    r = random.Random(40 + seed)
    for _ in range(50):
        kv, group, dim = r.choice([1, 2, 4, 8, 16]), r.choice([1, 2, 4, 8]), r.choice([64, 128, 256])
        forks, others = r.randint(2, 48), r.randint(0, 3)
        f = Forest(shim, r.choice([32, 64, 128]), seqs=64, pages=4000)
        f.grow([0], [r.choice([300, 1152, 2000, 4000])])
        f.fork([0] * (forks - 1), list(range(1, forks)))
        f.grow(list(range(forks)), [r.choice([1, 8, 100])] * forks)
        if others:
            f.grow(list(range(forks, forks + others)), [r.choice([1, 200, 1500])] * others)
        counts = [r.choice([1, 2, 3])] * forks + [r.choice([1, 40, 100, 300]) for _ in range(others)]
        _, items, *_ = planned(f, kv, group, dim, list(range(forks + others)), counts, r.choice([0, 0, 0, 400, 1300]))
        assert aligned(items)
        assert sum(map(len, items)) <= shim.shim_most_items(kv * group, kv, dim, sum(counts), forks + others)
        f.close()
