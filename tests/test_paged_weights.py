"""What positions are looked at (no GPU): the work of weighing a batch takes every score once in each reading and every weight
once, inside the buffers it was given; eviction in the host's book."""
import ctypes
import os
import random
import subprocess

import pytest

from mechta_amd import paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARG, POS, NOMEM = -1, -3, -7


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("weights") / "weights.so")
    src = [os.path.join(ROOT, "tests", "paged_weights_shim.cpp"), os.path.join(ROOT, "mechta_amd", "csrc", "paged_book.cpp")]
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-shared", "-fPIC", "-Wall", "-Werror", "-D_GLIBCXX_ASSERTIONS",
                    "-fsanitize=undefined", "-fno-sanitize-recover=all", "-static-libubsan", *src, "-o", so], check=True)
    L = ctypes.CDLL(so)
    L.shim_new.restype = ctypes.c_void_p
    L.shim_message.restype = ctypes.c_char_p
    L.shim_entries.restype = ctypes.c_size_t
    return L


def ints(xs):
    return (ctypes.c_int * max(len(xs), 1))(*xs)


def weigh(L, kv, group, batch, window, last, stats, work):
    sizes = ints([0] * 7)
    L.shim_weigh(kv * group, kv, 64, len(batch), ints([x for m in batch for x in m]), window, last, ctypes.c_longlong(stats),
                 ctypes.c_longlong(work), sizes)
    scores, sums, fades, merges = [], [], ints([0] * (8 * sizes[6])), ints([0] * (8 * sizes[3]))
    for k in range(3):
        buf = ints([0] * (12 * sizes[k]))
        L.shim_scores(k, buf)
        scores.append([buf[12 * i:12 * i + 11] for i in range(sizes[k])])
    for k in range(2):
        buf = ints([0] * (16 * sizes[4 + k]))
        L.shim_sums(k, buf)
        sums.append([buf[16 * i:16 * i + 14] for i in range(sizes[4 + k])])
    L.shim_fades(fades), L.shim_merges(merges)
    return (scores, sums, [fades[8 * i:8 * i + 7] for i in range(sizes[6])],
            [merges[8 * i:8 * i + 7] for i in range(sizes[3])])


def covers(spans, lo, hi):
    """Whether the spans take each of [lo, hi) once and, of it, nothing else."""
    spans = sorted((max(a, lo), min(b, hi)) for a, b in spans if max(a, lo) < min(b, hi))
    return bool(spans) and spans[0][0] == lo and spans[-1][1] == hi and all(x[1] == y[0] for x, y in zip(spans, spans[1:]))


def check(L, kv, group, batch, window, last, stats, work):
    scores, sums, fades, merges = weigh(L, kv, group, batch, window, last, stats, work)
    tokens = sum(c for _, c, _ in batch)
    most = L.shim_entries(kv * group, kv, max(tokens, 1), len(batch))
    assert all(len(x) <= most for x in scores + sums + [fades, merges])
    seqs, at = {}, 0
    for s, c, n in batch:
        m = min(last or c, c)
        at += c
        if m:
            seqs[s] = (at - m, m * group, n - m, n)  # first counted token, rows, its position, length
    stat, spans, kept, whole, weights, parts, pairs = {}, {}, {}, {}, {}, {}, {}
    for kind, items in enumerate(scores):
        for seq, head, tok0, rows, row0, pos0, k0, k1, st, keep, final in items:
            assert (tok0, rows, pos0) == seqs[seq][:3] and k0 % 32 == 0 and 0 <= k0 <= k1 <= seqs[seq][3]
            assert (row0 == 0 and rows <= (16, 32)[kind] and keep >= 0 and k0 < k1) if kind < 2 else keep == -1
            for r in range(row0, min(row0 + 128, rows)):
                i = st + r - row0
                assert 0 <= i < stats and i not in stat
                stat[i] = (seq, head, r)
                if final:
                    assert (seq, head, r) not in whole
                    whole[seq, head, r] = i
            if final and kind < 2:  # it takes its sums itself
                weights.setdefault((seq, head), []).append((k0, k1))
                pairs.setdefault((seq, head), []).append((k0, k1, 0, rows))
                spans.setdefault((seq, head, r), []).append((k0, k1))
            if keep >= 0:
                kept.setdefault((seq, head), []).append((keep, keep + (k1 - k0 + 31) // 32 * 32 * rows, k0))
    by_tok0 = {v[0]: s for s, v in seqs.items()}
    for head, tok0, rows, r0, r1, st, n in merges:
        seq = by_tok0[tok0]
        assert n > 1 and rows == seqs[seq][1] and 0 <= r0 < r1 <= rows
        for r in range(r0, r1):
            assert all(stat[st + p * rows + r] == (seq, head, r) for p in range(n)) and (seq, head, r) not in whole
            whole[seq, head, r] = st + r
    for (seq, _, r), s in spans.items():
        pos = seqs[seq][2] + r // group
        assert covers(s, max(0, pos - window + 1) if window else 0, pos + 1)
    used = sorted((a, b) for v in kept.values() for a, b, _ in v)
    assert all(x[1] <= y[0] for x, y in zip(used, used[1:])) and (not used or (used[0][0] >= 0 and used[-1][1] <= work))
    for kind, items in enumerate(sums):
        for seq, head, tok0, rows, pos0, k0, k1, r0, r1, st, n, sc, s0, part in items:
            assert (tok0, rows, pos0) == seqs[seq][:3] and 0 <= k0 < k1 <= seqs[seq][3] and k0 % 32 == 0
            assert (r0, r1) == (0, rows) if kind == 0 else r0 % 32 == 0 and 0 <= r0 <= rows and r1 <= rows
            for r in range(rows):
                if kind == 0:
                    assert all(stat[st + p * rows + r] == (seq, head, r) for p in range(n))
                else:  # the final ones
                    assert whole[seq, head, r] == st + r
            if kind == 0:
                for a, b, first in kept[seq, head]:  # the scores lie where they are read: block by block from s0
                    assert a == sc + (first - s0) * rows
                assert part == -1
            if part < 0:
                weights.setdefault((seq, head), []).append((k0, k1))
            else:
                assert k1 - k0 <= 256 and 0 <= part and part + 256 <= work
                parts[part] = (seq, head, k0, k1)
            pairs.setdefault((seq, head), []).append((k0, k1, r0, r1))
    for seq, head, k0, k1, part, n, stride in fades:
        weights.setdefault((seq, head), []).append((k0, k1))
        for x in range(n):
            assert parts.pop(part + x * stride) == (seq, head, k0, k1)
    assert not parts
    blocks = sorted(list(kept.values()) and used or [])
    for s, (_, rows, pos0, n) in seqs.items():
        for head in range(kv):
            assert covers(weights[s, head], 0, n), "a weight that is left out, or written twice"
            items = pairs[s, head]
            r = random.Random(s)
            for row in {0, rows - 1, *(r.randrange(rows) for _ in range(5))}:
                pos = pos0 + row // group
                assert covers([(a, b) for a, b, r0, r1 in items if r0 <= row < r1], max(0, pos - window + 1) if window else 0, pos + 1)
    return scores, sums, fades, blocks


@pytest.mark.parametrize("seed", range(60))
def test_weighing_takes_every_score_and_weight_once(shim, seed):
    r = random.Random(900 + seed)
    kv, group = r.choice([1, 2, 3, 8]), r.choice([1, 2, 5, 8, 16])
    window, last = r.choice([0, 0, 1, 31, 33, 513]), r.choice([0, 0, 1, 3, 32])
    batch = []
    for s in range(r.choice([1, 2, 5, 20])):
        c = r.choice([0, 1, 1, 1, 2, 4, 7, 33, 200, 513])
        batch.append((s, c, c + r.choice([0, 0, 1, 30, 31, 32, 1000, 20000])))
    tokens = sum(c for _, c, _ in batch)
    stats = max(tokens, 1) * kv * group + r.choice([0, 5, 300, 1 << 18])
    check(shim, kv, group, batch, window, last, stats, r.choice([0, 1000, 100000, 1 << 26]))


def test_large_batches_stay_inside_their_lists(shim):
    for kv, group, batch, last in [(4, 8, [(s, 1, 500 + 110 * s) for s in range(64)], 0), (1, 1, [(0, 1, 4194304)], 0),
                                   (8, 16, [(0, 1, 4194304)], 0), (4, 8, [(0, 4096, 4096)], 0), (2, 8, [(0, 512, 300000)], 32),
                                   (2, 40, [(s, 1, 100 + s) for s in range(300)], 0), (16, 1, [(s, 1, 3) for s in range(1000)], 0)]:
        tokens = sum(c for _, c, _ in batch)
        check(shim, kv, group, batch, 0, last, tokens * kv * group + (1 << 18), 1 << 26)


@pytest.mark.parametrize("more", [0, 5000, 200000, 3000000])
def test_parts_of_sums_find_room_behind_the_scores(shim, more):
    for kv, group, prompt in [(4, 8, 4096), (2, 4, 700), (1, 1, 3000)]:
        batch = [(s, 1 + s % 3, 900 + 410 * s) for s in range(20)] + [(30, prompt, prompt + 100)]
        tokens = sum(c for _, c, _ in batch)
        scores, sums, fades, kept = check(shim, kv, group, batch, 0, 0, tokens * kv * group + 1000, shim.shim_parts() + more)
        assert all(end <= more for _, end in kept)  # scores stay in the room that is theirs
        assert any(f[5] > 1 for f in fades)  # and sums are split


@pytest.mark.parametrize("seed", range(40))
def test_lists_that_no_batch_fills_are_known_before(shim, seed):
    r = random.Random(70 + seed)
    kv, group, last, window = r.choice([1, 2]), r.choice([1, 4, 8, 16, 17]), r.choice([0, 1, 2, 4]), r.choice([0, 33])
    seqs, ctx, tokens = r.choice([1, 3, 8]), r.choice([31, 700, 5000]), r.choice([1, 4, 40])
    work = shim.shim_parts() + r.choice([0, 20000, 1 << 26])
    may = [shim.shim_may(kv * group, kv, tokens, seqs, ctx, window, last, ctypes.c_longlong(work), k) for k in range(7)]
    seen = [0] * 7
    for _ in range(30):
        left, batch = tokens, []
        for s in range(seqs):
            c = min(r.choice([0, 1, 1, 2, 4, 40]), left, ctx)
            left -= c
            batch.append((s, c, min(ctx, c + r.choice([0, 40, 600, 5000]))))
        scores, sums, fades, merges = weigh(shim, kv, group, batch, window, last, 1 << 20, work)
        seen = [a or bool(x) for a, x in zip(seen, scores + [merges] + sums + [fades])]
    assert all(b or not a for a, b in zip(seen, may))
    if work > 1 << 26:  # and no more than that: few rows find room
        rows = min(last or tokens, tokens) * group
        assert may == [1, rows > 16, rows > 32, rows > 32, 1, rows > 32, rows > 32 or window > 0]


# ---- eviction in the book ----

class Book:
    def __init__(self, L, pages, page, seqs, ctx=100000):
        self.L, self.seqs, self.pages = L, seqs, pages
        self.h = ctypes.c_void_p(L.shim_new(pages, page, seqs, ctx))

    def table(self, s):
        t = ints([0] * (self.pages + 1))
        return t[:self.L.shim_table(self.h, s, t)]

    def all(self):
        out = ints([0] * 5)
        state = []
        for s in range(self.seqs):
            self.L.shim_state(self.h, s, out)
            state.append(tuple(out[:3]))
        return (state, [self.table(s) for s in range(self.seqs)], self.L.shim_free_pages(self.h),
                [self.L.shim_owners(self.h, p) for p in range(self.pages)])

    def state(self, s):
        out = ints([0] * 5)
        self.L.shim_state(self.h, s, out)
        return tuple(out)

    def evict(self, seqs, keep):
        return self.L.shim_evict(self.h, len(seqs), ints(seqs), ints(keep))

    def whole(self):
        owned = sum((self.table(s) for s in range(self.seqs)), [])
        assert self.all()[3] == [owned.count(p) for p in range(self.pages)]
        assert self.L.shim_free_pages(self.h) == self.pages - len(set(owned))
        for s in range(self.seqs):
            n = self.state(s)[0]
            assert len(self.table(s)) == -(-n // 32)

    def close(self):
        self.L.shim_delete(self.h)


def test_eviction_takes_new_pages_and_gives_back_the_old(shim):
    b = Book(shim, 12, 32, 4)
    assert shim.shim_reserve(b.h, 2, ints([0, 1]), ints([200, 40])) == 0  # 7 and 2 pages
    assert shim.shim_fork(b.h, 1, ints([0]), ints([2]), ints([96]), 0) == 0  # shares 3
    shim.shim_sent(b.h)
    before = b.all()
    assert b.evict([0], [100]) == NOMEM and b.all() == before  # 4 pages, 3 free
    assert b.evict([0, 1], [70, 64]) == 0
    assert b.state(0) == (70, 130, 70, 1, 0) and b.state(1) == (40, 0, 0, 0, 2)
    assert b.table(0) == [9, 10, 11] and b.table(2) == [0, 1, 2]
    b.whole()
    shim.shim_undo_evict(b.h)
    assert b.all() == before and b.state(0)[3:] == (1, 0)
    b.whole()
    b.close()


def test_an_evicted_sequence_is_cut_back_to_what_is_left_of_it(shim):
    b = Book(shim, 40, 32, 6)
    assert shim.shim_reserve(b.h, 1, ints([0]), ints([300])) == 0 and b.evict([0], [100]) == 0
    assert shim.shim_reserve(b.h, 1, ints([0]), ints([20])) == 0
    assert shim.shim_set_len(b.h, 0, 99) == POS and b"eviction" in shim.shim_message()
    assert shim.shim_fork(b.h, 1, ints([0]), ints([1]), ints([99]), 0) == POS
    assert shim.shim_set_len(b.h, 0, 100) == 0 and b.state(0)[:3] == (100, 200, 100)
    assert shim.shim_fork(b.h, 3, ints([0, 0, 0]), ints([1, 2, 3]), ints([100, 0, 100]), 0) == 0
    assert b.state(1)[:3] == (100, 200, 100) and b.state(2)[:3] == (0, 0, 0)
    assert b.evict([1], [50]) == 0 and b.state(1)[:3] == (50, 250, 50) and b.state(0)[:3] == (100, 200, 100)
    assert shim.shim_set_len(b.h, 0, 0) == 0 and b.state(0)[:3] == (0, 0, 0)
    shim.shim_undo_set_len(b.h, 0)
    assert b.state(0)[:3] == (100, 200, 100)
    assert shim.shim_free(b.h, 1, ints([3])) == 0 and b.state(3)[:3] == (0, 0, 0)
    b.whole()
    b.close()


def test_positions_stay_within_32_bits(shim):
    """A sequence that is cut again and again counts on: at most to the largest position that an int holds."""
    b = Book(shim, 1100, 4096, 1, ctx=4194304)
    assert shim.shim_reserve(b.h, 1, ints([0]), ints([1])) == 0
    for i in range(512):
        assert shim.shim_reserve(b.h, 1, ints([0]), ints([4194303])) == 0 and b.evict([0], [1]) == 0
        assert b.state(0)[:3] == (1, 4194303 * (i + 1), 1)
    left = 2 ** 31 - 1 - sum(b.state(0)[:2])
    before = b.all()
    assert shim.shim_reserve(b.h, 1, ints([0]), ints([left + 1])) == POS and b.all() == before
    assert shim.shim_reserve(b.h, 1, ints([0]), ints([left])) == 0 and sum(b.state(0)[:2]) == 2 ** 31 - 1
    b.close()


@pytest.mark.parametrize("seqs,keep,code", [([0, 0], [5, 5], ARG), ([4], [5], ARG), ([-1], [5], ARG), ([0], [0], ARG), ([0], [-3], ARG)])
def test_book_refusals(shim, seqs, keep, code):
    b = Book(shim, 12, 32, 4)
    assert shim.shim_reserve(b.h, 1, ints([0]), ints([100])) == 0
    before = b.all()
    assert b.evict(seqs, keep) == code and b.all() == before
    b.close()


@pytest.mark.parametrize("seed", range(10))
def test_histories_with_eviction(shim, seed):
    r = random.Random(seed)
    b = Book(shim, 30, 32, 5)
    done = 0
    for _ in range(400):
        a, empty = r.randrange(5), [s for s in range(5) if not b.state(s)[0]]
        n = b.state(a)[0]
        op = r.choice(["grow", "grow", "evict", "evict", "undone", "set_len", "fork", "free", "compact"])
        before = b.all()
        if op == "grow":
            rc = shim.shim_reserve(b.h, 1, ints([a]), ints([r.choice([1, 31, 70, 200])]))
        elif op in ("evict", "undone"):
            keep = [r.randint(1, 200), r.randint(1, 200)]
            rc = b.evict([a, (a + 1) % 5], keep)
            if rc == 0 and op == "undone":
                shim.shim_undo_evict(b.h)
                assert b.all() == before
            elif rc == 0:
                for s, k in zip([a, (a + 1) % 5], keep):
                    was, now = before[0][s], b.state(s)
                    assert now[0] == min(was[0], k) and now[0] + now[1] == was[0] + was[1]
        elif op == "set_len":
            rc = shim.shim_set_len(b.h, a, r.randint(0, n))
        elif op == "fork" and empty and a not in empty:
            rc = shim.shim_fork(b.h, 1, ints([a]), ints(empty), ints([r.randint(0, n)]), r.randrange(2))
        elif op == "free":
            rc = shim.shim_free(b.h, 1, ints([a]))
        else:
            rc = min(0, shim.shim_compact(b.h))
        if rc:
            assert b.all() == before, op
        else:
            done += 1
        b.whole()
    assert done > 200
    b.close()


# ---- what is refused before a device is touched ----

def test_null_handles():
    L = paged.lib()
    one = (ctypes.c_int * 1)(0)
    assert L.mpg_keep_weights(None, 0) == ARG and L.mpg_weights(None, 0, None, None, None) == ARG
    assert L.mpg_weigh(None, 0, 1, None, 0, 0, 1.0, None, 1.0) == ARG and L.mpg_evict(None, 1, one, one, 0, 0) == ARG
    assert L.mpg_position(None, 0, None) == ARG and L.mpg_begin_shared(None, 1, one, one, None) == ARG
    assert L.mpg_weights_bytes(None, 0) == 0


def test_weights_bytes():
    """Four bytes a position and head of every sequence, and room to work in."""
    L = paged.lib()
    config = lambda seqs: paged._Config(2, 8, 4, 128, 0, 8, 32, seqs, 1000, 64)  # noqa: E731
    a, b = (L.mpg_weights_bytes(ctypes.byref(config(n)), 0) for n in (10, 20))
    assert 10 * 2 * 4 * 1024 * 4 <= b - a and L.mpg_weights_bytes(ctypes.byref(config(10)), -1) == 0
    assert L.mpg_weights_bytes(ctypes.byref(paged._Config(2, 8, 3, 128, 0, 8, 32, 4, 1000, 64)), 0) == 0
