"""The first reading of the scores (no GPU): the statistics of every counted row, of every piece and kind of tile, take each position
that the row sees once."""
import random

import pytest

from tests.test_paged_weights import covers, shim, weigh  # noqa: F401


def check(L, kv, group, batch, window, last, stats, work):
    scores, *_ = weigh(L, kv, group, batch, window, last, stats, work)
    spans = {}
    for kind, items in enumerate(scores):
        for seq, head, _, rows, row0, _, k0, k1, *_ in items:
            for r in range(row0, min(row0 + (16, 32, 128)[kind], rows)):
                spans.setdefault((seq, head, r), []).append((k0, k1))
    pieces, want = 0, set()
    for seq, count, n in batch:
        m = min(last or count, count)
        for head in range(kv):
            for r in range(m * group):
                pos = n - m + r // group
                want.add((seq, head, r))
                assert covers(spans[seq, head, r], max(0, pos - window + 1) if window else 0, pos + 1), "scores left out, or taken twice"
                pieces = max(pieces, len(spans[seq, head, r]))
    assert set(spans) == want  # and no row that is not counted
    return [bool(x) for x in scores], pieces


@pytest.mark.parametrize("seed", range(60))
def test_statistics_take_every_score_once(shim, seed):  # noqa: F811
    r = random.Random(1900 + seed)
    kv, group = r.choice([1, 2, 3, 8]), r.choice([1, 2, 5, 8, 16])
    window, last = r.choice([0, 0, 1, 31, 33, 513]), r.choice([0, 0, 1, 3, 32])
    batch = []
    for s in range(r.choice([1, 2, 5, 20])):
        c = r.choice([0, 1, 1, 1, 2, 4, 7, 33, 200, 513])
        batch.append((s, c, c + r.choice([0, 0, 1, 30, 31, 32, 1000, 20000])))
    tokens = sum(c for _, c, _ in batch)
    check(shim, kv, group, batch, window, last, max(tokens, 1) * kv * group + r.choice([0, 5, 300, 1 << 18]),
          r.choice([0, 1000, 100000, 1 << 26]))


@pytest.mark.parametrize("kv,group,batch,last,kind", [
    (4, 8, [(s, 1, 500 + 110 * s) for s in range(64)], 0, 0),  # a token each, in pieces
    (2, 8, [(0, 4, 65536)], 0, 1),
    (8, 16, [(0, 1, 131072)], 0, 0),
    (2, 8, [(0, 32, 16000)], 0, 2),  # many rows, in pieces
    (4, 8, [(0, 700, 700)], 0, 2),
    (1, 5, [(0, 300, 40000)], 32, 2)])
def test_statistics_of_long_sequences(shim, kv, group, batch, last, kind):  # noqa: F811
    tokens = sum(c for _, c, _ in batch)
    kinds, pieces = check(shim, kv, group, batch, 0, last, tokens * kv * group + (1 << 18), 1 << 26)
    assert kinds[kind] and pieces > 1
