"""Weights and eviction on a device made of host memory (tests/paged_evict_shim.cpp): each step on the way to the device that can
fail, allocations of the host among them, fails once, and no sequence changes by a call that fails."""
import ctypes
import os
import random
import subprocess

import pytest

from mechta_amd.build import HIPCC
from tests.test_paged_store import Store, ints

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("evict") / "evict.so")
    src = [os.path.join(ROOT, "tests", "paged_evict_shim.cpp"), os.path.join(ROOT, "mechta_amd", "csrc", "paged_book.cpp")]
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
    L.mpg_weigh.argtypes = [P, ctypes.c_int, ctypes.c_int, P, ctypes.c_int64, ctypes.c_int64, ctypes.c_float, P, ctypes.c_float]
    return L


class Weighted(Store):
    """A handle that keeps weights, and beside it what each position weighs (the same in every layer and head but for a constant)."""

    def __init__(self, L):
        super().__init__(L)
        assert L.mpg_keep_weights(self.h, 0) == 0, L.shim_message()
        self.weights = [[] for _ in range(self.SEQS)]
        self.evicted = [0] * self.SEQS

    def at(self, layer):
        base, seq, head = P(), ctypes.c_int64(), ctypes.c_int64()
        assert self.L.mpg_weights(self.h, layer, ctypes.byref(base), ctypes.byref(seq), ctypes.byref(head)) == 0
        return ctypes.cast(base, ctypes.POINTER(ctypes.c_float)), seq.value, head.value

    def write(self):
        """Marks, and a weight, for each position that has none yet; it weighed nothing."""
        for layer in range(2):
            w, seq, head = self.at(layer)
            for s in range(self.SEQS):
                for p in range(len(self.weights[s]), self.length(s)):
                    for h in range(2):
                        i = s * seq + h * head + p
                        assert w[i] == 0, "a new position weighs something"
                        w[i] = self.marks + p + 1000 * layer + 100 * h
        for s in range(self.SEQS):
            self.weights[s] += [self.marks + p for p in range(len(self.weights[s]), self.length(s))]
        super().write()

    def whole(self):
        for layer in range(2):
            w, seq, head = self.at(layer)
            for s in range(self.SEQS):
                assert len(self.weights[s]) == self.length(s)
                for h in range(2):
                    assert w[s * seq + h * head:s * seq + h * head + self.length(s)] == [x + 1000 * layer + 100 * h for x in self.weights[s]]
        n = ctypes.c_int()
        for s in range(self.SEQS):
            assert self.holds(s, self.content[s])
            assert self.L.mpg_position(self.h, s, ctypes.byref(n)) == 0
            assert n.value == self.length(s) + self.evicted[s]
            if not self.L.shim_moved(self.h, s):
                assert self.L.shim_shift(self.h, s) == self.evicted[s]
        owned = sum((self.table(s) for s in range(self.SEQS)), [])
        assert self.state()[3] == [owned.count(p) for p in range(self.PAGES)] and self.state()[2] == self.PAGES - len(set(owned))

    def check_device(self):
        super().check_device()
        stands = self.L.shim_tokens(self.h)
        assert (stands > 0) == (self.L.shim_weigh_work(self.h, 0) > 0) == (self.L.shim_weigh_work(self.h, 1) > 0)

    def evict(self, seqs, keep, first, recent):
        return self.L.mpg_evict(self.h, len(seqs), ints(seqs), ints(keep), first, recent)

    def cut(self, s, keep, first, recent):
        n = self.length(s) if len(self.content[s]) == self.length(s) else len(self.content[s])
        if n <= keep:
            return
        mid, free = keep - first - recent, n - keep
        kept = list(range(first)) + [first + min(free, k + 1) + k for k in range(mid)] + list(range(n - recent, n))
        self.content[s] = [self.content[s][i] for i in kept]
        self.weights[s] = [self.weights[s][i] for i in kept]
        self.evicted[s] += n - keep


def filled(L):
    """Sequences 0 and 1 share two full pages of a prompt of 70, 2 has 40 of its own; a batch of all three stands."""
    s = Weighted(L)
    assert s.begin([0], [70]) == 0
    s.write()
    assert L.mpg_fork(s.h, 1, ints([0]), ints([1]), None) == 0
    s.content[1], s.weights[1] = list(s.content[0]), list(s.weights[0])
    assert s.begin([2], [33]) == 0
    s.write()
    assert s.begin([0, 1, 2], [1, 2, 7]) == 0
    s.write()
    s.whole()
    s.check_device()
    return s


def each_failure(L, call):
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


def test_a_failed_eviction_changes_no_sequence(shim):
    def call(s):
        return s.evict([1, 2, 0], [35, 40, 32], 2, 20 + 20)

    with_window = lambda s: s.evict([1, 2, 0], [45, 40, 42], 0, 40)  # noqa: E731
    failed = 0
    for s, ok in each_failure(shim, with_window):
        if not ok:
            failed += 1
            assert s.state() == s.before
            s.whole()
            assert with_window(s) == 0, shim.shim_message()
        for x, keep in ((1, 45), (2, 40), (0, 42)):
            s.cut(x, keep, 0, 40)
        s.whole()
        assert shim.shim_tokens(s.h) == -1 and not s.runs() and not shim.shim_weigh_work(s.h, 0)
        assert s.begin([0, 1], [1, 3]) == 0  # the device learns of the pages and of where the sequences stand
        s.write()
        s.whole()
        s.check_device()
        assert all(shim.shim_device_table(s.h, x, k) == p for x in range(s.SEQS) for k, p in enumerate(s.table(x)))
        assert [shim.shim_shift(s.h, x) for x in range(3)] == s.evicted[:3]
    assert failed > 8
    s = filled(shim)
    assert call(s) == -1 and s.state() is not None  # a window that reaches further than what is kept
    s.close()


@pytest.mark.parametrize("shared", [False, True])
def test_a_failed_begin_lengthens_no_sequence(shim, shared):
    def call(s):
        f = shim.mpg_begin_shared if shared else shim.mpg_begin
        return f(s.h, 3, ints([2, 4, 0]), ints([30, 3, 20]), None)

    failed = 0
    for s, ok in each_failure(shim, call):
        s.check_device()
        if not ok:
            failed += 1
            assert s.state() == s.before and shim.shim_tokens(s.h) == 10
            s.whole()
            assert call(s) == 0
        s.write()
        s.whole()
        s.check_device()
    assert failed > 8


def test_random_histories_with_failures(shim):
    r = random.Random(4)
    done = failed = cuts = 0
    for _ in range(9):
        s = Weighted(shim)
        for _ in range(150):
            a, empty = r.randrange(s.SEQS), [x for x in range(s.SEQS) if not s.length(x)]
            n, floor = s.length(a), 0
            op = r.choice(["begin", "begin", "reserve", "evict", "evict", "set_len", "fork", "copy", "free", "compact"])
            before = s.state()
            shim.shim_fail_after(r.choice([-1, r.randrange(50)]))
            after = lambda: None  # noqa: E731
            if op in ("begin", "reserve"):
                f = {"begin": lambda *x: shim.mpg_begin_shared(*x, None), "reserve": shim.mpg_reserve}[op]
                rc = f(s.h, 2, ints([a, (a + 1) % s.SEQS]), ints([r.choice([0, 1, 31, 40]), r.choice([1, 32])]))
            elif op == "evict":
                keep = r.randint(40, 70)
                rc = s.evict([a], [keep], 0, 40)
                after = lambda: s.cut(a, keep, 0, 40)  # noqa: E731
                cuts += rc == 0 and n > keep
            elif op == "set_len":
                m = r.randint(0, n)
                rc = shim.mpg_set_len(s.h, a, m)

                def after():
                    s.content[a], s.weights[a] = s.content[a][:m], s.weights[a][:m]
                    s.evicted[a] = s.evicted[a] if m else 0
            elif op in ("fork", "copy"):
                if not empty or a in empty:
                    continue
                m = r.randint(0, n) if op == "fork" else n
                rc = shim.mpg_fork(s.h, 1, ints([a]), ints(empty), ints([m])) if op == "fork" else shim.mpg_copy(s.h, 1, ints([a]), ints(empty))

                def after():
                    b = empty[0]
                    s.content[b], s.weights[b] = s.content[a][:m], s.weights[a][:m]
                    s.evicted[b] = s.evicted[a] if m else 0
            elif op == "free":
                rc = shim.mpg_free(s.h, 1, ints([a]))

                def after():
                    s.content[a], s.weights[a], s.evicted[a] = [], [], 0
            else:
                rc = shim.mpg_compact(s.h, None)
            shim.shim_fail_after(-1)
            if rc:
                failed += rc != -3
                assert s.state() == before, (op, rc)
            else:
                done += 1
                after()
                s.write()
            s.whole()
            s.check_device()
        s.close()
    assert done > 300 and failed > 100 and cuts > 20


def test_weights_are_kept_from_the_start_on_or_not_at_all(shim):
    for use in (lambda s: shim.mpg_reserve(s.h, 1, ints([0]), ints([3])), lambda s: s.begin([0], [3])):
        s = Store(shim)
        assert use(s) == 0 and shim.mpg_free(s.h, 1, ints([0])) == 0
        assert shim.mpg_keep_weights(s.h, 0) == -1 and b"already" in shim.shim_message()
        x = P(64)
        assert shim.mpg_weigh(s.h, 0, 1, x, 256, 64, 1.0, None, 1.0) == -1 and shim.mpg_evict(s.h, 0, None, None, 0, 40) == -1
        s.close()
    s = Weighted(shim)
    assert shim.mpg_keep_weights(s.h, 0) == -1
    assert s.begin([0, 2], [1, 3]) == 0
    x, was = P(64), shim.shim_weighed()
    assert shim.mpg_weigh(s.h, 0, 4, x, 256, 64, 1.0, None, 1.0) == 0 and shim.mpg_weigh(s.h, 1, 5, x, 256, 64, 1.0, None, 0.0) == 0
    assert shim.mpg_weigh(s.h, 0, 3, x, 256, 64, 1.0, None, 1.0) == -5  # fewer rows than tokens
    assert shim.mpg_weigh(s.h, 0, 4, P(72), 256, 64, 1.0, None, 1.0) == -1 and shim.mpg_weigh(s.h, 0, 4, x, 255, 64, 1.0, None, 1.0) == -1
    assert shim.shim_weighed() == was + 2
    s.close()
