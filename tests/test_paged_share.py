"""Batches of sequences with pages in common (no GPU): a shared batch's work covers every score once, on the pages that each
of its sequences has, every row's partials are joined, and nothing leaves the buffers it was given."""
import ctypes
import os
import random
import subprocess

import pytest

from tests.paged_forests import FORESTS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TILE = {0: 16, 1: 32, 2: 128, 3: 256}


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("share") / "share.so")
    src = [os.path.join(ROOT, "tests", "paged_share_shim.cpp"), os.path.join(ROOT, "mechta_amd", "csrc", "paged_book.cpp")]
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-shared", "-fPIC", "-Wall", "-Werror", "-D_GLIBCXX_ASSERTIONS",
                    "-fsanitize=undefined", "-fno-sanitize-recover=all", "-static-libubsan", *src, "-o", so], check=True)
    L = ctypes.CDLL(so)
    L.shim_new.restype = ctypes.c_void_p
    L.shim_message.restype = ctypes.c_char_p
    L.shim_most_items.restype = L.shim_most_joins.restype = ctypes.c_size_t
    return L


def ints(xs):
    return (ctypes.c_int * max(len(xs), 1))(*xs)


class Forest:
    def __init__(self, L, page, seqs=64, pages=40000):
        self.L, self.page, self.pages = L, page, pages
        self.h = ctypes.c_void_p(L.shim_new(pages, page, seqs, 1 << 20))

    def grow(self, seqs, counts):
        assert self.L.shim_reserve(self.h, len(seqs), ints(seqs), ints(counts)) == 0, self.L.shim_message()

    def fork(self, src, dst, lens=None):
        assert self.L.shim_fork(self.h, len(dst), ints(src), ints(dst), ints(lens) if lens else None) == 0

    def table(self, s):
        t = ints([0] * (self.pages + 1))
        return t[:self.L.shim_table(self.h, s, t)]

    def length(self, s):
        return self.L.shim_len(self.h, s)

    def close(self):
        self.L.shim_delete(self.h)


def planned(f, kv, group, dim, seqs, counts, window):
    L = f.L
    f.grow(seqs, counts)
    ranges = L.shim_share(f.h, kv * group, kv, dim, len(seqs), ints(seqs), ints(counts))
    sizes = ints([0] * 7)
    L.shim_plan(kv * group, kv, dim, window, sizes)
    items = []
    for kind in range(4):
        buf = ints([0] * (12 * sizes[kind]))
        L.shim_items(kind, buf)
        items.append([list(buf[12 * i:12 * i + 12]) for i in range(sizes[kind])])
    joins, segs, order = ints([0] * (8 * sizes[4])), ints([0] * (4 * sizes[5])), ints([0] * (2 * sizes[6]))
    L.shim_joins(joins), L.shim_segs(segs), L.shim_order(order)
    return (ranges, items, [list(joins[8 * i:8 * i + 8]) for i in range(sizes[4])],
            [list(segs[4 * i:4 * i + 4]) for i in range(sizes[5])], [tuple(order[2 * i:2 * i + 2]) for i in range(sizes[6])])


def check(f, kv, group, dim, seqs, counts, window):
    """Returns the ranges, how many scores the shared tiles have, and of which kinds they are."""
    L = f.L
    ranges, items, joins, segs, order = planned(f, kv, group, dim, seqs, counts, window)
    tokens = sum(counts)
    most, most_joins = (fn(kv * group, kv, dim, max(tokens, 1), len(seqs)) for fn in (L.shim_most_items, L.shim_most_joins))
    assert sum(map(len, items)) <= most and len(joins) <= most_joins and len(order) <= tokens
    assert len(segs) in (0, L.shim_levels() * len(joins))
    tables = {s: f.table(s) for s in seqs}
    owner, place = {}, {}
    at = 0
    for s, c in zip(seqs, counts):
        for t in range(c):
            owner[at], place[at] = s, f.length(s) - c + t
            at += 1
    pages_of = {}
    done, partial, shared = {}, {}, 0  # (token, query head): intervals; partial row: whose, and its interval
    for kind, list_ in enumerate(items):
        for seq, head, tok0, row0, rows, pos0, k0, k1, part, split, top, _ in list_:
            assert k0 % 32 == 0 and k0 < k1 and 0 <= row0 < rows
            last = min(row0 + TILE[kind], rows) - 1
            far = 0
            for row in range(row0, last + 1):
                if top:
                    tok, pos = order[tok0 + row // group]
                    assert pos >= pos0 >= k1 and k1 % 32 == 0 and part >= 0
                    far = max(far, pos)
                    key = (owner[tok], seq, k0 // f.page, (k1 - 1) // f.page)
                    if key not in pages_of:
                        pages_of[key] = tables[owner[tok]][key[2]:key[3] + 1] == tables[seq][key[2]:key[3] + 1]
                    assert pages_of[key], "pages that a row's sequence does not have"
                else:
                    tok, pos = tok0 + row // group, pos0 + row // group
                    assert owner[tok] == seq
                assert place[tok] == pos
                who = (tok, head * group + row % group)
                lo, hi = max(k0, pos - window + 1 if window else 0), min(k1, pos + 1)
                shared += max(0, hi - lo) if top else 0
                if part < 0:
                    assert who not in done
                    done[who] = [(lo, hi)]
                else:
                    p = part + row - row0
                    assert 0 <= p < L.shim_part_rows() and p not in partial
                    partial[p] = (who, lo, hi)
            assert not top or far == top - 1
    used = set()
    for n, (head, tok0, row0, count, part, splits, wide, nsegs) in enumerate(joins):
        assert splits >= 1 and 0 <= nsegs <= L.shim_levels() and (splits > 1 or nsegs)
        parts = [(part, count, splits)] + [tuple(s[:3]) for s in segs[n * L.shim_levels():n * L.shim_levels() + nsegs]]
        assert sum(p[2] for p in parts) <= L.shim_splits_most()
        for r in range(count):
            row = row0 + r
            who = (tok0 + row // group, head * group + row % group)
            assert who not in done
            done[who] = []
            for base, stride, m in parts:
                for s in range(m):
                    p = base + s * stride + r
                    assert partial[p][0] == who, "another row's partial"
                    used.add(p)
                    done[who].append(partial[p][1:])
    assert used == set(partial), "a partial that nothing joins"
    assert len(done) == tokens * kv * group
    for (tok, _), spans in done.items():
        pos = place[tok]
        spans = sorted(s for s in spans if s[0] < s[1])
        assert spans[0][0] == (max(0, pos - window + 1) if window else 0) and spans[-1][1] == pos + 1
        assert all(a[1] == b[0] for a, b in zip(spans, spans[1:])), "keys that are left out, or taken twice"
    return ranges, shared, tuple(k for k, list_ in enumerate(items) if any(i[10] for i in list_))


@pytest.mark.parametrize("seed", range(60))
def test_a_shared_plan_covers_every_score_once(shim, seed):
    r = random.Random(500 + seed)
    f = Forest(shim, r.choice([32, 64, 256]), seqs=40)
    kv, group, dim = r.choice([1, 2, 3]), r.choice([1, 2, 5, 8]), r.choice([64, 128, 256])
    alive = [0]
    f.grow([0], [r.choice([1, 100, 700, 3000, 9000])])
    for s in range(1, r.choice([2, 5, 12, 30])):
        src = r.choice(alive)
        n = f.length(src)
        f.fork([src], [s], [r.choice([n, n, r.randint(0, n)])])
        alive.append(s)
        if r.random() < 0.5:
            a = r.choice(alive)
            f.grow([a], [r.choice([1, 31, 32, 200, 1000])])
    seqs = r.sample(alive, r.randint(1, len(alive)))
    counts = [r.choice([0, 1, 1, 1, 2, 3, 4, 7, 40, 300]) for _ in seqs]
    check(f, kv, group, dim, seqs, counts, r.choice([0, 0, 0, 1, 33, 513, 4000]))
    f.close()


@pytest.mark.parametrize("name", FORESTS)
def test_forks_of_a_prompt(shim, name):
    kv, group, dim, page, prompt, forks, own, tokens, window, kinds = FORESTS[name]
    f = Forest(shim, page)
    f.grow([0], [prompt])
    f.fork([0] * (forks - 1), list(range(1, forks)))
    r = random.Random(3)
    f.grow(list(range(forks)), [r.randint(1, own) for _ in range(forks)])
    seqs = r.sample(range(forks), forks)
    counts = [tokens[i % len(tokens)] for i in range(forks)]
    ranges, shared, got = check(f, kv, group, dim, seqs, counts, window)
    assert ranges == 1 and got == kinds
    if kinds and not window:  # all whole pages of the prompt, for all that are not chunks
        assert shared == prompt // page * page * kv * group * sum(c for c in counts if c * group <= 256)
    f.close()


def test_a_tree_of_forks(shim):
    """Three levels and no more; a level that is not worth a tile of its own goes to the ones below it."""
    f = Forest(shim, 32)
    f.grow([0], [8192])
    f.fork([0] * 3, [1, 2, 3])
    f.grow([0, 1, 2, 3], [4096] * 4)
    f.fork([s % 4 for s in range(4, 16)], list(range(4, 16)))
    f.grow(list(range(16)), [2048] * 16)
    f.fork([s % 16 for s in range(16, 48)], list(range(16, 48)))
    f.grow(list(range(48)), [33] * 48)
    ranges, shared, kinds = check(f, 2, 8, 128, list(range(48)), [1] * 48, 0)
    assert ranges == 1 + 4 + 16 and shared == 48 * 16 * (8192 + 4096 + 2048) and kinds
    f.close()
    f = Forest(shim, 32)
    f.grow([0], [64])  # too short to be worth it: the two prompts behind it take it with them
    f.fork([0], [1])
    f.grow([0, 1], [20000, 30000])
    f.fork([0] * 7 + [1] * 7, list(range(2, 16)))
    ranges, shared, kinds = check(f, 4, 8, 128, list(range(15, -1, -1)), [1] * 16, 0)
    assert ranges == 2 and shared == 32 * 8 * (20064 // 32 * 32 + 30064 // 32 * 32)
    f.close()


def test_deep_chains_of_forks(shim):
    f = Forest(shim, 32, seqs=300, pages=4000)
    f.grow([0], [320])
    for s in range(1, 300):
        f.fork([s - 1], [s])
        f.grow([s], [32])
    check(f, 1, 1, 64, list(range(300)), [1] * 300, 0)
    f.close()


def test_without_anything_in_common_the_plan_is_the_plain_one(shim):
    f = Forest(shim, 64)
    f.grow([0, 1, 2], [5000, 100, 3000])
    f.fork([1], [3])  # 100 positions: one page
    ranges, shared, _ = check(f, 2, 8, 128, [2, 3, 1, 0], [1, 2, 1, 300], 0)
    assert ranges == 0 and shared == 0 and shim.shim_plain(16, 2, 128, 0) == 1
    f.close()


def test_a_window_past_the_prompt_leaves_it_out(shim):
    f = Forest(shim, 64)
    f.grow([0], [4000])
    f.fork([0] * 7, list(range(1, 8)))
    f.grow(list(range(8)), [600] * 8)
    ranges, shared, _ = check(f, 2, 8, 128, list(range(8)), [1] * 8, 513)
    assert ranges == 1 and shared == 0 and shim.shim_plain(16, 2, 128, 513) == 1
    f.close()


def test_more_rows_than_partials_fit_are_attended_apart(shim):
    f = Forest(shim, 32, seqs=600, pages=2000)
    f.grow([0], [2000])
    f.fork([0] * 599, list(range(1, 600)))
    ranges, shared, _ = check(f, 8, 16, 64, list(range(600)), [1] * 600, 0)  # 76,800 rows
    assert ranges == 1 and shared == 0 and shim.shim_plain(128, 8, 64, 0) == 1
    f.close()
