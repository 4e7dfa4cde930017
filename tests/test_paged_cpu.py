"""The paged cache's C ABI without a GPU: exports, the header as C, what is refused before a device is touched, rotary
frequencies."""
import ctypes
import math
import os
import re
import subprocess

import pytest

from mechta_amd import paged
from tests.paged_reference import rope_freqs

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mechta_paged.h")


def test_library_exports_every_declared_symbol():
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(mpg_[a-z0-9_]+)\s*\(", src)))
    assert sorted(paged.SYMBOLS) == names
    for name in names:
        assert hasattr(paged.lib(), name)


def test_header_compiles_as_c():
    r = subprocess.run(["gcc", "-fsyntax-only", "-Wall", "-Werror", "-x", "c", HEADER], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.parametrize("sc", [dict(), dict(scaling="linear", factor=3.0), dict(scaling="ntk", factor=4.0),
                                dict(scaling="yarn", factor=16.0, original=4096), dict(scaling="yarn", factor=0.5, original=100),
                                dict(scaling="bands", factor=8.0, original=8192)])
@pytest.mark.parametrize("dim,base", [(64, 1e7), (128, 1e4), (4, 10.0), (512, 5e5)])
def test_rope_frequencies(sc, dim, base):
    th, amp = paged.Rope(dim, base=base, **sc).freqs()
    want, want_amp = rope_freqs(dim, base, **sc)
    assert th == pytest.approx(want, rel=1e-12) and amp == pytest.approx(want_amp, rel=1e-14)
    assert th[0] <= 1.0 and all(a >= b > 0 for a, b in zip(th, th[1:]))


def test_rope_known_values():
    assert paged.Rope(4, base=100.0).freqs() == ([1.0, 0.1], 1.0)
    assert paged.Rope(4, base=100.0, scaling="linear", factor=2.0).freqs()[0] == [0.5, 0.05]
    # the slowest pair of NTK scaling is slowed by the factor, the fastest not at all
    th = paged.Rope(64, base=1e4, scaling="ntk", factor=8.0).freqs()[0]
    assert th[0] == 1.0 and th[-1] == pytest.approx(1e4 ** (-62 / 64) / 8)
    # bands: fast pairs as they are, slow ones by the factor
    th, plain = paged.Rope(128, base=5e5, scaling="bands", factor=8.0, original=8192).freqs()[0], paged.Rope(128, base=5e5).freqs()[0]
    assert th[0] == plain[0] and th[-1] == pytest.approx(plain[-1] / 8)
    assert paged.Rope(64, scaling="yarn", factor=math.e, original=4096).freqs()[1] == pytest.approx(1.1)
    assert paged.Rope(64, amplitude=0.7).freqs()[1] == 0.7


@pytest.mark.parametrize("bad", [dict(dim=0), dict(dim=-2), dict(dim=63), dict(dim=514), dict(base=1.0), dict(base=math.nan),
                                 dict(base=math.inf), dict(scaling="linear", factor=0.0),
                                 dict(scaling="linear", factor=math.nan), dict(scaling="yarn", factor=2.0),
                                 dict(scaling="bands", factor=2.0), dict(scaling="yarn", factor=2.0, original=9, beta_fast=0.0),
                                 dict(scaling="bands", factor=2.0, original=9, low=4.0), dict(dim=2, scaling="ntk", factor=2.0),
                                 dict(amplitude=-1.0), dict(amplitude=math.nan)])
def test_rope_refusals(bad):
    with pytest.raises(paged.MkvError) as e:
        paged.Rope(**{"dim": 64, **bad})
    assert e.value.code == -1


def test_rope_names():
    for bad in (dict(layout="neox"), dict(scaling="cubic")):
        with pytest.raises(ValueError):
            paged.Rope(64, **bad)


def config(**k):
    return paged._Config(*{**dict(layers=1, q_heads=4, kv_heads=2, head_dim=64, fmt=0, pages=8, page=32, seqs=3, ctx=200,
                                  tokens=64), **k}.values())


@pytest.mark.parametrize("bad,code", [(dict(layers=0), -1), (dict(q_heads=3), -1), (dict(kv_heads=0), -1), (dict(head_dim=96), -1),
                                      (dict(fmt=1), -1), (dict(fmt=3), -1), (dict(pages=0), -1), (dict(pages=(1 << 27) + 1), -1),
                                      (dict(page=16), -1), (dict(seqs=0), -1), (dict(seqs=65537), -1), (dict(ctx=0), -2),
                                      (dict(ctx=4194305), -2), (dict(tokens=0), -1), (dict(tokens=262145), -1),
                                      (dict(seqs=65536, ctx=4194304), -1)])
def test_configurations_refused_without_a_device(bad, code):
    L, h = paged.lib(), ctypes.c_void_p()
    c = config(**bad)
    assert L.mpg_bytes(ctypes.byref(c)) == 0
    assert L.mpg_create(ctypes.byref(h), ctypes.byref(c), None, None, None) == code and not h.value
    assert L.mkv_last_error()


def test_bytes():
    """The pool's bytes exactly, and some for tables and split partials."""
    L = paged.lib()
    a, b = (L.mpg_bytes(ctypes.byref(config(pages=n, layers=10, head_dim=128, kv_heads=4, page=64))) for n in (100, 200))
    assert b - a == 100 * 10 * 2 * 4 * 64 * 128 * 2


def test_null_arguments():
    L, h = paged.lib(), ctypes.c_void_p()
    one = (ctypes.c_int * 1)(0)
    assert L.mpg_create(None, ctypes.byref(config()), None, None, None) == -1
    assert L.mpg_create(ctypes.byref(h), None, None, None, None) == -1
    assert L.mpg_bytes(None) == 0 and L.mpg_destroy(None) == 0
    for rc in (L.mpg_set_stream(None, None), L.mpg_sync(None), L.mpg_len(None, 0, None), L.mpg_table(None, 0, None, 0),
               L.mpg_free_pages(None, None), L.mpg_pages(None, 0, 0, None), L.mpg_reserve(None, 1, one, one),
               L.mpg_begin(None, 1, one, one, None), L.mpg_set_len(None, 0, 0), L.mpg_fork(None, 1, one, one, None),
               L.mpg_copy(None, 1, one, one), L.mpg_free(None, 1, one), L.mpg_compact(None, None),
               L.mpg_append(None, 0, 1, None, 0, 0, None, 0, 0, None, 0, 0, None, 0),
               L.mpg_attend(None, 0, 1, None, 0, 0, 1.0, None, None, 0, 0, None), L.mpg_read_rows(None, 0, 0, 0, 0, 1, None),
               L.mpg_rope_freqs(None, None, None), L.mpg_rope_turns(None, None), L.mpg_rotate(None, 0, 1, 1, 64, None, 0, 0, None, None, 0, 0, None)):
        assert rc == -1
    r = paged.Rope(64)._turns
    for args, want in [((0, 1, 1, 32), -1), ((5, 1, 1, 64), -1), ((0, -1, 1, 64), -1), ((0, 1, 70000, 64), -1),
                       ((0, 1, 1, 5000), -1), ((0, 1, 1, 64), -1), ((0, 0, 1, 64), 0)]:
        assert L.mpg_rotate(ctypes.byref(r), *args, None, 64, 64, None, None, 64, 64, None) == want


def test_a_pool_past_any_memory_is_refused():
    L = paged.lib()
    c = config(layers=4096, q_heads=1024, kv_heads=1024, head_dim=256, page=256, pages=1 << 27)
    h = ctypes.c_void_p()
    assert L.mpg_bytes(ctypes.byref(c)) == 0
    assert L.mpg_create(ctypes.byref(h), ctypes.byref(c), None, None, None) == -7 and not h


def test_rotate_refuses_turns_that_are_none():
    L = paged.lib()
    for dim, layout in [(0, 0), (3, 0), (514, 0), (-2, 0), (64, 2), (64, -1)]:
        t = paged._Turns()
        t.dim, t.layout = dim, layout
        assert L.mpg_rotate(ctypes.byref(t), 0, 1, 1, 512, 16, 512, 512, 16, 16, 512, 512, None) == -1
    t = paged._Turns()
    t.dim = 64
    for fmt, rows, heads, dim in [(3, 1, 1, 64), (0, -1, 1, 64), (0, 1, -1, 64), (0, 1, 65537, 64), (0, 1, 1, 62), (0, 1, 1, 4098)]:
        assert L.mpg_rotate(ctypes.byref(t), fmt, rows, heads, dim, 16, 512, 512, 16, 16, 512, 512, None) == -1
    assert L.mpg_rotate(ctypes.byref(t), 0, 1, 1, 64, 17, 64, 64, 16, 16, 64, 64, None) == -1  # misaligned
    assert L.mpg_rotate(ctypes.byref(t), 0, 1, 1, 64, 16, 64, 64, 16, 16, 128, 64, None) == -1  # in place, other strides
    assert L.mpg_rotate(ctypes.byref(t), 0, 0, 1, 64, None, 64, 64, None, None, 64, 64, None) == 0


def test_lists_of_ints():
    a, p = paged._ints([3, 1, 2], 3)
    assert list(a) == [3, 1, 2] and p
    assert paged._ints([])[1] == 0
    with pytest.raises(ValueError, match="4 needed"):
        paged._ints([1, 2, 3], 4, "counts")
    for bad in (1 << 32, 1 << 31, -(1 << 31) - 1):
        with pytest.raises(ValueError, match="32 bits"):
            paged._ints([0, bad], 2, "seqs")
