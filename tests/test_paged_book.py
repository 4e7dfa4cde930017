"""The paged cache's host side (no GPU): whose pages are whose, against a plain model that keeps what every page holds,
and that a plan's work covers every score once and stays inside the buffers it was given."""
import ctypes
import os
import random
import subprocess

import pytest

from tests.paged_shapes import SHAPES, UNEVEN

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARG, POS, NOMEM = -1, -3, -7


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("book") / "book.so")
    src = [os.path.join(ROOT, "tests", "paged_book_shim.cpp"), os.path.join(ROOT, "mechta_amd", "csrc", "paged_book.cpp")]
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-shared", "-fPIC", "-Wall", "-Werror", "-D_GLIBCXX_ASSERTIONS",
                    "-fsanitize=undefined", "-fno-sanitize-recover=all", "-static-libubsan", *src, "-o", so], check=True)
    L = ctypes.CDLL(so)
    L.shim_new.restype = ctypes.c_void_p
    L.shim_message.restype = ctypes.c_char_p
    L.shim_most_items.restype = L.shim_most_joins.restype = ctypes.c_size_t
    return L


def ints(xs):
    return (ctypes.c_int * max(len(xs), 1))(*xs)


class Book:
    """The book, and beside it what each page would hold on the device: sequence content is a list of marks."""

    def __init__(self, L, pages, page, seqs, ctx):
        self.L, self.page, self.seqs, self.pages = L, page, seqs, pages
        self.h = ctypes.c_void_p(L.shim_new(pages, page, seqs, ctx))
        self.memory = [[None] * page for _ in range(pages)]
        self.content = [[] for _ in range(seqs)]
        self.mark = 0

    def close(self):
        self.L.shim_delete(self.h)

    def table(self, s):
        t = ints([0] * (self.pages + 1))
        return list(t)[:0] + list(t[:self.L.shim_table(self.h, s, t)])

    def state(self):
        return ([self.table(s) for s in range(self.seqs)], [self.L.shim_len(self.h, s) for s in range(self.seqs)],
                self.L.shim_free_pages(self.h), [self.L.shim_owners(self.h, p) for p in range(self.pages)])

    def copied(self):
        buf = ints([0] * (2 * self.pages + 2))
        n = self.L.shim_copies(buf)
        pairs = [(buf[2 * i], buf[2 * i + 1]) for i in range(n)]
        dsts = [d for _, d in pairs]
        assert len(set(dsts)) == n and not set(dsts) & {s for s, _ in pairs}, "a launch's pages overlap"
        for s, d in pairs:
            self.memory[d] = list(self.memory[s])
        return pairs

    def reserve(self, seqs, counts):
        rc = self.L.shim_reserve(self.h, len(seqs), ints(seqs), ints(counts))
        if rc == 0:  # and the rows are written
            for s, c in zip(seqs, counts):
                t = self.table(s)
                for _ in range(c):
                    p = len(self.content[s])
                    self.mark += 1
                    self.content[s].append(self.mark)
                    self.memory[t[p // self.page]][p % self.page] = self.mark
        return rc

    def fork(self, src, dst, lens=None, own=False):
        rc = self.L.shim_fork(self.h, len(dst), ints(src), ints(dst), None if lens is None else ints(lens), int(own))
        if rc == 0:
            self.copied()
            for i, (s, d) in enumerate(zip(src, dst)):
                self.content[d] = self.content[s][:len(self.content[s]) if lens is None else lens[i]]
        return rc

    def free(self, seqs):
        rc = self.L.shim_free(self.h, len(seqs), ints(seqs))
        if rc == 0:
            for s in seqs:
                self.content[s] = []
        return rc

    def set_len(self, s, n):
        rc = self.L.shim_set_len(self.h, s, n)
        if rc == 0:
            self.copied()
            self.content[s] = self.content[s][:n]
        return rc

    def compact(self):
        n = self.L.shim_compact(self.h)
        assert len(self.copied()) == n
        return n

    def check(self):
        """Every sequence reads what was written, owners are counted, a partly filled page has one owner."""
        tables, lens, free, owners = self.state()
        want = [0] * self.pages
        for s in range(self.seqs):
            assert lens[s] == len(self.content[s])
            assert len(tables[s]) == -(-lens[s] // self.page)
            for p in tables[s]:
                want[p] += 1
            for i, m in enumerate(self.content[s]):
                assert self.memory[tables[s][i // self.page]][i % self.page] == m, (s, i)
            if lens[s] % self.page:
                assert owners[tables[s][-1]] == 1
        assert owners == want and free == want.count(0)


@pytest.mark.parametrize("seed", range(8))
def test_random_histories(shim, seed):
    r = random.Random(seed)
    b = Book(shim, r.choice([3, 17, 64, 130]), r.choice([1, 4, 32]), 7, 400)
    sent = [[] for _ in range(7)]  # what the device has
    done = 0
    for _ in range(400):
        op = r.choice(["reserve", "reserve", "reserve", "fork", "copy", "free", "set_len", "compact"])
        before = b.state()
        seqs = r.sample(range(7), r.randint(0, 3))
        if op == "reserve":
            rc = b.reserve(seqs, [r.choice([0, 1, 2, 31, 32, 33, 90]) for _ in seqs])
        elif op in ("fork", "copy"):
            empty = [s for s in range(7) if not b.content[s]]
            dst = r.sample(empty, min(len(empty), r.randint(0, 2)))
            src = [r.choice([s for s in range(7) if s not in dst]) for _ in dst]
            lens = [r.randint(0, len(b.content[s])) for s in src] if op == "fork" and r.random() < 0.5 else None
            rc = b.fork(src, dst, lens, own=op == "copy")
        elif op == "free":
            rc = b.free(seqs[:1])
        elif op == "set_len":
            s = r.randrange(7)
            rc = b.set_len(s, r.randint(0, len(b.content[s])))
        else:
            b.compact()
            rc = 0
            used = b.pages - b.state()[2]
            assert all(o > 0 for o in b.state()[3][:used]) and not any(b.state()[3][used:])
        assert rc in (0, NOMEM, POS)
        if rc:
            assert b.state() == before
        else:
            done += 1
        b.check()
        # the entries not yet sent are all that changed since the tables were
        for s in range(7):
            t, fresh = b.table(s), shim.shim_fresh(b.h, s)
            assert t[:fresh] == sent[s][:fresh] and fresh <= len(t)
        if r.random() < 0.5:
            sent = [b.table(s) for s in range(7)]
            shim.shim_sent(b.h)
    assert done > 200
    b.close()


def test_pages_are_taken_lowest_first_and_shared(shim):
    b = Book(shim, 10, 4, 4, 100)
    assert b.reserve([0, 1], [6, 9]) == 0
    assert b.table(0) == [0, 1] and b.table(1) == [2, 3, 4]
    assert b.fork([1, 1], [2, 3], [8, 9]) == 0
    assert b.table(2) == [2, 3] and b.table(3) == [2, 3, 5]  # full pages shared, the last one copied
    assert b.free([0]) == 0 and b.free([1]) == 0
    assert b.state()[2] == 7 and b.compact() == 2
    assert b.table(2) == [0, 1] and b.table(3) == [0, 1, 2] or b.table(3) == [2, 0, 1]
    b.check()
    # a shared page that becomes partly filled is copied
    assert b.set_len(2, 5) == 0
    assert len(set(b.table(2)) & set(b.table(3))) == 1
    b.check()
    b.close()


def test_refusals_change_nothing(shim):
    b = Book(shim, 4, 4, 3, 12)
    assert b.reserve([0], [7]) == 0
    before = b.state()
    for rc, want in [(b.reserve([0, 0], [1, 1]), ARG), (b.reserve([3], [1]), ARG), (b.reserve([-1], [1]), ARG),
                     (b.reserve([1], [-1]), ARG), (b.reserve([0], [6]), POS), (b.reserve([0], [2**31 - 1]), POS),
                     (b.reserve([1, 2], [5, 4]), NOMEM), (b.fork([0], [0]), ARG), (b.fork([0, 1], [1, 2]), ARG),
                     (b.fork([0], [1], [8]), POS), (b.fork([0], [1], [-1]), POS), (b.fork([0, 0], [1, 1]), ARG),
                     (b.fork([5], [1]), ARG), (b.free([0, 0]), ARG), (b.free([9]), ARG), (b.set_len(0, 8), POS),
                     (b.set_len(0, -1), POS), (b.set_len(7, 0), ARG), (shim.shim_reserve(b.h, -1, None, None), ARG),
                     (shim.shim_reserve(b.h, 1, None, None), ARG), (shim.shim_fork(b.h, 1, None, ints([1]), None, 0), ARG)]:
        assert rc == want, shim.shim_message()
        assert b.state() == before
    assert b.fork([0], [1]) == 0  # not empty any more
    assert b.fork([0], [1]) == ARG
    # no page is free, and none that is given back can serve as the copy of a shared one
    c = Book(shim, 2, 4, 3, 12)
    assert c.reserve([0], [8]) == 0 and c.fork([0], [1]) == 0
    assert c.set_len(1, 6) == NOMEM
    c.check()
    assert c.free([0]) == 0 and c.set_len(1, 6) == 0
    c.check()
    b.close()
    c.close()


# ---- plans ----

def make_plan(L, q_heads, kv_heads, dim, batch, window):
    sizes = ints([0] * 5)
    L.shim_plan(q_heads, kv_heads, dim, len(batch), ints([x for m in batch for x in m]), window, sizes)
    items = []
    for kind in range(4):
        buf = ints([0] * (12 * sizes[kind] + 1))
        L.shim_items(kind, buf)
        items.append([list(buf[12 * i:12 * i + 9]) for i in range(sizes[kind])])
    buf = ints([0] * (8 * sizes[4] + 1))
    L.shim_joins(buf)
    return items, [list(buf[8 * i:8 * i + 6]) for i in range(sizes[4])]


TILE = {0: 16, 1: 32, 2: 128, 3: 256}


@pytest.mark.parametrize("seed", range(40))
def test_a_plan_covers_every_score_once(shim, seed):
    r = random.Random(100 + seed)
    kv, group = r.choice([1, 2, 3, 8]), r.choice([1, 2, 5, 8, 16, 40])
    dim, window = r.choice([64, 128, 256]), r.choice([0, 0, 1, 31, 32, 33, 513])
    batch = []
    for s in range(r.choice([1, 2, 5, 20])):
        c = r.choice([0, 1, 1, 1, 2, 4, 7, 33, 200, 513])
        batch.append((s, c, c + r.choice([0, 0, 1, 30, 31, 32, 1000, 20000])))
    tokens = sum(c for _, c, _ in batch)
    items, joins = make_plan(shim, kv * group, kv, dim, batch, window)
    assert sum(map(len, items)) <= shim.shim_most_items(kv * group, kv, dim, max(tokens, 1), len(batch))
    assert len(joins) <= shim.shim_most_joins(kv * group, kv, dim, max(tokens, 1), len(batch))
    first = {}
    at = 0
    for s, c, _ in batch:
        first[s] = at
        at += c
    tiles = {}
    for kind in range(4):
        for seq, head, tok0, row0, rows, pos0, k0, k1, part in items[kind]:
            _, c, n = batch[seq]
            assert tok0 == first[seq] and rows == c * group and pos0 == n - c and 0 <= head < kv
            assert 0 <= row0 < rows and k0 % 32 == 0 and 0 <= k0 < k1 <= n
            count = min(TILE[kind], rows - row0)
            tiles.setdefault((seq, head, row0, count), []).append((k0, k1, part))
    # the tiles of a head are its rows, each once
    for s, c, _ in batch:
        for head in range(kv):
            own = sorted((row0, n) for (seq, h, row0, n) in tiles if seq == s and h == head)
            assert [a for a, _ in own] == [sum(n for _, n in own[:i]) for i in range(len(own))]
            assert sum(n for _, n in own) == c * group
    joined = {(h, tok0, row0): (count, part, splits) for h, tok0, row0, count, part, splits in joins}
    assert len(joined) == len(joins)
    used = []
    for (seq, head, row0, count), ranges in tiles.items():
        _, c, n = batch[seq]
        lo, hi = n - c + row0 // group, n - c + (row0 + count - 1) // group  # positions of its first and last row
        ranges.sort()
        assert ranges[0][0] <= (max(0, lo - window + 1) if window else 0) and ranges[-1][1] == hi + 1
        assert all(a[1] == b[0] for a, b in zip(ranges, ranges[1:]))
        key = (head, first[seq], row0)
        if len(ranges) == 1:
            assert ranges[0][2] == -1 and key not in joined
        else:
            assert joined[key] == (count, ranges[0][2], len(ranges))
            for i, (_, _, part) in enumerate(ranges):
                assert part == ranges[0][2] + i * count
                used.append((part, part + count))
    used.sort()
    assert all(a[1] <= b[0] for a, b in zip(used, used[1:]))
    assert not used or (used[0][0] >= 0 and used[-1][1] <= shim.shim_part_rows())


@pytest.mark.parametrize("name", SHAPES)
def test_shapes_go_to_their_kernels(shim, name):
    dim, kv, group, window, batch, kind, split = SHAPES[name]
    items, joins = make_plan(shim, kv * group, kv, dim, [(s, *m) for s, m in enumerate(batch)], window)
    assert items[kind] and any(i[8] >= 0 for i in items[kind]) == split
    assert "among" not in name or not items[0] + items[1] + items[3]


def test_long_decodes_stay_apart_from_a_chunk(shim):
    """Among the chunk's tiles they would stream slower than on their own."""
    batch = [(0, 64, 1000)] + [(s, 1, 100 * s) for s in range(10, 70)]
    items, _ = make_plan(shim, 32, 4, 128, batch, 0)
    assert items[0] and items[2] + items[3]


def test_uneven_sequences_are_shared_out(shim):
    """A piece is never much longer than a CU's share of all keys."""
    for kv, batch in [(4, UNEVEN), (2, UNEVEN + UNEVEN[:40]), (8, UNEVEN[:20])]:
        items, _ = make_plan(shim, kv * 4, kv, 128, [(s, *m) for s, m in enumerate(batch)], 0)
        share = sum(n for _, n in batch) * kv / 256
        assert max(i[7] - i[6] for i in items[0]) <= 1.4 * share + 512 + 32


def test_splits_stay_inside_their_room(shim):
    """Batches whose splits ask for the most: many long keys behind few rows of many heads."""
    for kv, group, batch in [(8, 16, [(1, 4000000)] * 3), (64, 1, [(33, 1000000)] * 40), (1, 33, [(1, 4194304)] * 64),
                             (1, 1, [(33, 100000), (17, 3000000), (1, 2000000)] * 30), (255, 1, [(1, 100 * i) for i in range(1, 9)])]:
        batch = [(s, *m) for s, m in enumerate(batch)]
        items, joins = make_plan(shim, kv * group, kv, 64, batch, 0)
        tokens = sum(c for _, c, _ in batch)
        assert sum(map(len, items)) <= shim.shim_most_items(kv * group, kv, 64, tokens, len(batch))
        assert len(joins) <= shim.shim_most_joins(kv * group, kv, 64, tokens, len(batch))
        assert all(j[4] + j[3] * j[5] <= shim.shim_part_rows() for j in joins)


def test_short_rows_are_not_split(shim):
    for dim, most in [(64, 512), (128, 512), (256, 256)]:
        for n, split in [(1, False), (most, False), (most + 32, True)]:
            items, joins = make_plan(shim, 8, 2, dim, [(0, 1, n), (1, 1, 7)], 0)
            assert bool(joins) == split


def test_the_last_round_of_chunks_is_cut(shim):
    """A few tiles more than the CUs: those are cut into pieces for all CUs, the others stay whole."""
    for kv, group, dim, batch in [(4, 8, 128, [(0, 1050, 8000)]), (4, 8, 128, [(0, 1100, 8000)]), (2, 8, 256, [(0, 2100, 16000)])]:
        items, joins = make_plan(shim, kv * group, kv, dim, batch, 0)
        for kind in (2, 3):
            whole = [i for i in items[kind] if i[8] < 0]
            pieces = [i for i in items[kind] if i[8] >= 0]
            if items[kind]:
                assert len(whole) == 256 and 128 <= len(pieces) <= 256 and max(i[7] - i[6] for i in pieces) <= batch[0][2] / 3 + 32
