"""The paged cache's handle on a device made of host memory (tests/paged_store_shim.cpp): each step on the way to the device
that can fail, allocations of the host among them, fails once."""
import ctypes
import os
import random
import subprocess

import pytest

from mechta_amd import paged
from mechta_amd.build import HIPCC

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("store") / "store.so")
    src = [os.path.join(ROOT, "tests", "paged_store_shim.cpp"), os.path.join(ROOT, "mechta_amd", "csrc", "paged_book.cpp")]
    subprocess.run([HIPCC, "-x", "hip", "--offload-host-only", "-nogpulib", "-no-hip-rt", "-std=c++17", "-O1", "-fPIC", "-shared",
                    "-Wall", "-Werror", "-Wno-unused-result", "-D_GLIBCXX_ASSERTIONS", "-Wl,-Bsymbolic", *src, "-o", so],
                   check=True)
    L = ctypes.CDLL(so)
    L.shim_message.restype = ctypes.c_char_p
    L.shim_steps.restype = ctypes.c_long
    L.shim_fail_after.argtypes = [ctypes.c_long]
    L.mpg_append.argtypes = [P, ctypes.c_int, ctypes.c_int] + [P, ctypes.c_int64, ctypes.c_int64] * 3 + [P, ctypes.c_int]
    L.mpg_attend.argtypes = [P, ctypes.c_int, ctypes.c_int, P, ctypes.c_int64, ctypes.c_int64, ctypes.c_float, P, P,
                             ctypes.c_int64, ctypes.c_int64, P]
    return L


def ints(xs):
    return (ctypes.c_int * max(len(xs), 1))(*xs)


def rope(dim):
    return ctypes.byref(paged.Rope(dim).c)


class Store:
    """A handle of two layers with different windows, 32 positions a page; sequence content is a mark a position."""

    SEQS, PAGES, PAGE, TOKENS = 5, 12, 32, 100

    def __init__(self, L):
        self.L, self.h = L, P()
        config = ints([2, 4, 2, 64, 0, self.PAGES, self.PAGE, self.SEQS, 320, self.TOKENS])
        assert L.mpg_create(ctypes.byref(self.h), config, ints([0, 40]), None, None) == 0
        self.content = [[] for _ in range(self.SEQS)]
        self.marks = 0

    def close(self):
        self.L.shim_fail_after(-1)
        assert self.L.mpg_destroy(self.h) == 0

    def length(self, s):
        n = ctypes.c_int()
        assert self.L.mpg_len(self.h, s, ctypes.byref(n)) == 0
        return n.value

    def table(self, s):
        t = ints([0] * self.PAGES)
        return list(t[:self.L.mpg_table(self.h, s, t, self.PAGES)])

    def state(self):
        n = ctypes.c_int()
        assert self.L.mpg_free_pages(self.h, ctypes.byref(n)) == 0
        return ([self.length(s) for s in range(self.SEQS)], [self.table(s) for s in range(self.SEQS)], n.value,
                [self.L.shim_owners(self.h, p) for p in range(self.PAGES)])

    def write(self):
        """A mark for each position that has none yet."""
        for s in range(self.SEQS):
            t = self.table(s)
            for at in range(len(self.content[s]), self.length(s)):
                self.marks += 2 * 2
                self.content[s].append(self.marks)
                self.L.shim_mark(self.h, t[at // self.PAGE], at % self.PAGE, self.marks)

    def holds(self, s, content):
        t = self.table(s)
        return len(content) == self.length(s) and all(
            self.L.shim_marked(self.h, t[at // self.PAGE], at % self.PAGE, m) for at, m in enumerate(content))

    def begin(self, seqs, counts):
        return self.L.mpg_begin(self.h, len(seqs), ints(seqs), ints(counts), None)

    def runs(self):
        """What a replayed append would write: (sequence, position, page, tokens) of each run."""
        buf = ints([0] * (4 * self.TOKENS))
        n = self.L.shim_runs(self.h, buf)
        runs = [buf[4 * i:4 * i + 4] for i in range(n)]
        return [(s, pos, self.L.shim_device_table(self.h, s, pos // self.PAGE), c) for s, _, pos, c in runs]

    def check_device(self):
        """Replays do the batch that stands, or nothing."""
        stands = self.L.shim_tokens(self.h)
        runs = self.runs()
        assert sum(c for *_, c in runs) == max(stands, 0)
        assert (stands > 0) == (self.L.shim_work(self.h, 0) > 0) == (self.L.shim_work(self.h, 1) > 0)
        for s, pos, page, count in runs:
            assert pos + count <= self.length(s) and self.table(s)[pos // self.PAGE] == page

    def eager(self):
        n = self.L.shim_tokens(self.h)
        x = P(64)
        return (self.L.mpg_append(self.h, 0, max(n, 1), x, 128, 64, x, 128, 64, None, 0, 0, None, 0),
                self.L.mpg_attend(self.h, 0, max(n, 1), x, 256, 64, 1.0, None, None, 0, 0, P(128)))


def filled(L):
    """Sequences 0 and 1 share two full pages of a prompt of 70, 2 has 40 of its own; a batch of all three stands."""
    s = Store(L)
    assert s.begin([0], [70]) == 0
    s.write()
    assert L.mpg_fork(s.h, 1, ints([0]), ints([1]), None) == 0
    s.content[1] = list(s.content[0])
    assert L.mpg_reserve(s.h, 2, ints([4, 3]), ints([64, 33])) == 0 and s.begin([2], [33]) == 0
    assert L.mpg_free(s.h, 1, ints([4])) == 0  # two holes
    s.write()
    assert s.begin([0, 1, 2], [1, 2, 7]) == 0
    s.write()
    assert all(s.holds(x, s.content[x]) for x in range(s.SEQS))
    s.check_device()
    return s


CALLS = {
    "reserve": lambda s: s.L.mpg_reserve(s.h, 2, ints([4, 2]), ints([33, 40])),
    "set_len": lambda s: s.L.mpg_set_len(s.h, 2, 31),
    "set_len in a shared page": lambda s: s.L.mpg_set_len(s.h, 1, 40),
    "fork": lambda s: s.L.mpg_fork(s.h, 1, ints([0]), ints([4]), ints([50])),
    "copy": lambda s: s.L.mpg_copy(s.h, 1, ints([2]), ints([4])),
    "free": lambda s: s.L.mpg_free(s.h, 2, ints([0, 3])),
    "compact": lambda s: s.L.mpg_compact(s.h, None),
}


def each_failure(L, call):
    """(handle, whether the call succeeded) for each step of the call that can fail, the handle's batch standing before."""
    s = filled(L)
    L.shim_fail_after(-1)
    assert call(s) == 0, L.shim_message()
    steps = L.shim_steps()
    assert steps > 5
    s.close()
    for k in range(steps):
        s = filled(L)
        s.before = s.state()
        L.shim_fail_after(k)
        rc = call(s)
        L.shim_fail_after(-1)
        assert rc in (0, -6, -7), rc
        yield s, rc == 0
        s.close()


# what each call leaves of the sequences' content, {sequence: (source, positions)}
LEAVES = {"reserve": {}, "set_len": {2: (2, 31)}, "set_len in a shared page": {1: (1, 40)}, "fork": {4: (0, 50)}, "copy": {4: (2, 40)},
          "free": {0: (0, 0), 3: (3, 0)}, "compact": {}}


@pytest.mark.parametrize("name", CALLS)
def test_a_failed_page_call_changes_no_sequence(shim, name):
    """Lengths, page lists, owners and what the pages hold are as before; the call can be made again."""
    failed = 0
    for s, ok in each_failure(shim, CALLS[name]):
        if not ok:
            failed += 1
            assert s.state() == s.before, name
            assert all(s.holds(x, s.content[x]) for x in range(s.SEQS))
            assert CALLS[name](s) == 0, shim.shim_message()
        was = [list(c) for c in s.content]
        for x, (src, n) in LEAVES[name].items():
            s.content[x] = was[src][:n]
        s.write()  # what was reserved
        assert all(s.holds(x, s.content[x]) for x in range(s.SEQS))
        owned = sum((s.table(x) for x in range(s.SEQS)), [])
        assert s.state()[3] == [owned.count(p) for p in range(s.PAGES)] and s.state()[2] == s.PAGES - len(set(owned))
        # the device learns of every page that changed
        assert s.begin([2], [1]) == 0
        assert all(shim.shim_device_table(s.h, x, k) == p for x in range(s.SEQS) for k, p in enumerate(s.table(x)))
    assert failed > 4


def test_a_failed_begin_lengthens_no_sequence(shim):
    def call(s):
        return s.begin([2, 4, 0], [60, 3, 20])

    failed = 0
    for s, ok in each_failure(shim, call):
        if not ok:
            failed += 1
            assert s.state() == s.before
            assert call(s) == 0
        s.write()
        assert [s.length(x) for x in range(s.SEQS)] == [91, 72, 100, 33, 3]
        assert all(s.holds(x, s.content[x]) for x in range(s.SEQS))
        s.check_device()
    assert failed > 4


@pytest.mark.parametrize("seed", range(6))
def test_random_histories_with_failures(shim, seed):
    """Every other call fails somewhere: no sequence changes by it, and later calls find the book whole."""
    r = random.Random(seed)
    s, failed, done = Store(shim), 0, 0
    for _ in range(300):
        a, empty = r.randrange(s.SEQS), [x for x in range(s.SEQS) if not s.length(x)]
        n, leaves = s.length(a), {}
        op = r.choice(["begin", "begin", "reserve", "set_len", "fork", "copy", "free", "compact"])
        before = s.state()
        shim.shim_fail_after(r.choice([-1, r.randrange(40)]))
        if op in ("begin", "reserve"):
            seqs, counts = ints([a, (a + 1) % s.SEQS]), ints([r.choice([0, 1, 31, 40]), r.choice([1, 32])])
            rc = shim.mpg_begin(s.h, 2, seqs, counts, None) if op == "begin" else shim.mpg_reserve(s.h, 2, seqs, counts)
        elif op == "set_len":
            m = r.randint(0, n)
            rc, leaves = shim.mpg_set_len(s.h, a, m), {a: (a, m)}
        elif op in ("fork", "copy"):
            if not empty or a in empty:
                continue
            m = r.randint(0, n) if op == "fork" else n
            rc = shim.mpg_fork(s.h, 1, ints([a]), ints(empty), ints([m])) if op == "fork" else shim.mpg_copy(s.h, 1, ints([a]), ints(empty))
            leaves = {empty[0]: (a, m)}
        elif op == "free":
            rc, leaves = shim.mpg_free(s.h, 1, ints([a])), {a: (a, 0)}
        else:
            rc = shim.mpg_compact(s.h, None)
        shim.shim_fail_after(-1)
        if rc:
            failed += rc != -3
            assert s.state() == before, (op, rc)
        else:
            done += 1
            for x, (src, m) in leaves.items():
                s.content[x] = s.content[src][:m]
            s.write()
        assert all(s.holds(x, s.content[x]) for x in range(s.SEQS)), op
        s.check_device()
        owned = sum((s.table(x) for x in range(s.SEQS)), [])
        assert s.state()[3] == [owned.count(p) for p in range(s.PAGES)] and s.state()[2] == s.PAGES - len(set(owned))
        for x in range(s.SEQS):  # what the device has of the tables, but for what it will be sent
            sent = min(shim.shim_fresh(s.h, x), len(s.table(x)))
            assert [shim.shim_device_table(s.h, x, k) for k in range(sent)] == s.table(x)[:sent]
    assert failed > 30 and done > 100
    s.close()


@pytest.mark.parametrize("name", CALLS)
def test_a_failed_page_call_leaves_no_stale_batch(shim, name):
    """Whatever fails: replays do the batch that stands, or nothing; a page call that succeeds then ends it."""
    failed = 0
    for s, ok in each_failure(shim, CALLS[name]):
        s.check_device()
        stands = shim.shim_tokens(s.h) >= 0
        assert s.eager() == ((0, 0) if stands else (-1, -1)) and not (ok and stands)
        assert shim.mpg_free(s.h, 1, ints([3])) == 0
        assert shim.shim_tokens(s.h) == -1 and not s.runs() and not shim.shim_work(s.h, 0) and not shim.shim_work(s.h, 1)
        failed += not ok
    assert failed > 4


def test_a_failed_begin_leaves_the_batch_before(shim):
    failed = 0
    for s, ok in each_failure(shim, lambda s: s.begin([2, 4, 0], [60, 3, 20])):
        s.check_device()
        assert shim.shim_tokens(s.h) == (83 if ok else 10) and s.eager() == (0, 0)
        assert shim.mpg_free(s.h, 1, ints([3])) == 0 and not s.runs()
        assert s.begin([2, 4], [1, 1]) == 0
        s.check_device()
        failed += not ok
    assert failed > 4


def test_uploads_go_on_behind_an_event_that_was_not_recorded(shim):
    """The lists went out: the call has succeeded."""
    s = filled(shim)
    for i in range(12):
        shim.shim_fail_records(i % 3 != 0)
        assert s.begin([2], [1]) == 0, shim.shim_message()
        shim.shim_fail_records(0)
        s.check_device()
    s.close()


def test_splits_fit_the_join(shim):
    """The join holds the factors of SPLITS_MOST splits of a row; what all splits add to a plan stays below that too."""
    most = shim.shim_splits_most()
    for kv in (1, 2, 3, 8, 64, 1023, 1024):
        for rows in (1, 16, 33, 256):
            for part in (0, 65536 - rows * kv, 65536):
                for more in (0, most // 2, most - 1, most):
                    n = shim.shim_splits_room(rows, kv, max(part, 0), more)
                    assert n <= most and (n < 2 or (n - 1) * kv + more <= most and max(part, 0) + n * rows * kv <= 65536)
    assert shim.shim_splits_room(1, 1, 0, 0) == most


def test_strides_of_one_entry_do_not_matter(shim):
    """torch gives an axis of one entry whatever stride it was cut with. A second entry's has to fit."""
    h = P()
    assert shim.mpg_create(ctypes.byref(h), ints([1, 1, 1, 64, 0, 8, 32, 2, 200, 10]), None, rope(64), None) == 0
    x, y = P(64), P(128)
    for n, tok, head, want in [(1, 131, 67, 0), (1, 128, 1, 0), (2, 128, 67, 0), (2, 131, 64, -1)]:
        assert shim.mpg_begin(h, 1, ints([0]), ints([n]), None) == 0
        assert shim.mpg_append(h, 0, n, x, tok, head, x, tok, head, x, tok, head, y, 1) == want, (n, tok, head)
        assert shim.mpg_attend(h, 0, n, x, tok, head, 1.0, None, x, tok, head, y) == want
        # in place: q in one piece, as far as it has more than one piece
        assert shim.mpg_append(h, 0, n, x, 64, 64, x, 64, 64, x, tok, head, x, 1) == (0 if n == 1 else -1)
    assert shim.mpg_append(h, 0, 2, x, 64, 64, x, 64, 64, x, 64, 7, x, 1) == 0
    assert shim.mpg_destroy(h) == 0
    s = Store(shim)  # several heads, one token
    assert s.begin([0], [1]) == 0
    for head, want in [(64, 0), (65, -1)]:
        assert shim.mpg_append(s.h, 0, 1, x, 3, head, x, 5, head, None, 0, 0, None, 0) == want
        assert shim.mpg_attend(s.h, 0, 1, x, 3, head, 1.0, None, None, 0, 0, y) == want
    s.close()
