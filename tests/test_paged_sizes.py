"""The sizes that the paged cache's sizing calls give, and what they give none for (no GPU)."""
import ctypes

import pytest

from mechta_amd import paged


def config(layers=1, q_heads=1, kv_heads=1, head_dim=64, fmt=0, pages=1, page=32, seqs=1, ctx=32, tokens=1):
    return ctypes.byref(paged._Config(layers, q_heads, kv_heads, head_dim, fmt, pages, page, seqs, ctx, tokens))


# lists of a sequence's rows and heads that are more than 2^32 words with a handle's own, and fewer without
@pytest.mark.parametrize("more", [dict(q_heads=80, kv_heads=80, seqs=65536, tokens=65536), dict(q_heads=512, kv_heads=128, seqs=40000, tokens=40000)])
def test_weights_bytes_of_what_is_refused(more):
    L = paged.lib()
    assert L.mpg_bytes(config(**more)) > 0
    assert L.mpg_weights_bytes(config(**more), 1) == 0
    assert b"mpg_weights_bytes: lists of" in L.mkv_last_error()
    more["seqs"] = more["tokens"] = 1000
    assert L.mpg_weights_bytes(config(**more), 1) > 0


# lists past 2^32 words
@pytest.mark.parametrize("more", [dict(q_heads=1024, kv_heads=1024, tokens=262144), dict(q_heads=512, kv_heads=256, seqs=65536, tokens=65536, ctx=8192)])
def test_bytes_of_what_is_refused(more):
    L = paged.lib()
    assert L.mpg_bytes(config(**more)) == 0 and b"mpg_bytes: lists of" in L.mkv_last_error()
    h = ctypes.c_void_p(1)
    assert L.mpg_create(ctypes.byref(h), config(**more), None, None, None) == -7 and h.value is None
    assert b"mpg_create: lists of" in L.mkv_last_error()
    more["tokens"] = more["seqs"] = 100
    assert L.mpg_bytes(config(**more)) > 0
