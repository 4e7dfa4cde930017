"""The paged cache's Python binding: what it keeps, and what it refuses by itself."""
import copy
import ctypes
import pickle

import pytest
import torch

from mechta_amd import paged


def test_pages_are_refused_after_close():
    """The tensors over the pool given before are of memory that is free now: none is given again."""
    kv = paged.PagedKv.__new__(paged.PagedKv)  # (as after close() on a device)
    kv._owner = paged._Handle()
    kv._views = {(0, paged.K): "a tensor over the pool"}
    kv.close()
    with pytest.raises(paged.MkvError, match="NULL handle"):
        kv.pages(0, paged.K)


@pytest.mark.gpu
def test_pages_are_refused_after_close_on_the_device(torch_gpu):
    kv = paged.PagedKv(1, 2, 1, 64, 4, page=32, seqs=1)
    assert kv.pages(0, paged.V).shape[0] == 4 and kv.pages(0, paged.K) is kv.pages(0, paged.K)
    kv.close()
    for which in (paged.K, paged.V):
        with pytest.raises(paged.MkvError, match="NULL handle"):
            kv.pages(0, which)

def test_a_copied_rope_goes_by_its_own_turns():
    """Copies and pickles (a model's configuration on its way to another process) hold no address of another object."""
    rope = paged.Rope(64, layout="interleaved", base=5e5, scaling="yarn", factor=4.0, original=4096)
    for other in (copy.copy(rope), copy.deepcopy(rope), pickle.loads(pickle.dumps(rope))):
        assert other._ptr == ctypes.addressof(other._turns)
        assert bytes(other._turns) == bytes(rope._turns) and other.freqs() == rope.freqs() and other.dim == 64


@pytest.mark.parametrize("past", [1 << 31, 1 << 32, (1 << 32) + 64, -(1 << 31) - 1])
def test_numbers_past_32_bits_are_refused(past, monkeypatch):
    """The C ABI's ints would hold their low 32 bits: another layer, sequence or length."""
    class Library:  # none of these calls may get as far
        def __getattr__(self, name):
            return lambda *a: pytest.fail(f"reached {name}")

    kv = paged.PagedKv.__new__(paged.PagedKv)
    kv._owner, kv._views = paged._Handle(), {}
    kv._h, kv._lib = kv._owner.ptr, Library()
    kv.kv_heads = kv.q_heads = 1
    kv.head_dim, kv.device = 64, torch.device("cpu")
    kv.dtype = torch.float16
    k = torch.zeros(1, 1, 64, dtype=torch.float16)
    monkeypatch.setattr(paged, "lib", Library)
    for call in (lambda: kv.length(past), lambda: kv.table(past), lambda: kv.set_len(past, 0), lambda: kv.set_len(0, past),
                 lambda: kv.pages(past, 0), lambda: kv.pages(0, past), lambda: kv.read_rows(past, 0, 0, 0, 1, k),
                 lambda: kv.read_rows(0, past, 0, 0, 1, k), lambda: kv.read_rows(0, 0, past, 0, 1, k),
                 lambda: kv.read_rows(0, 0, 0, past, past + 1, k), lambda: kv.append(past, k, k),
                 lambda: kv.attend(past, k, out=k.clone()), lambda: paged.Rope(past),
                 lambda: paged.Rope(64, scaling="yarn", factor=2.0, original=past),
                 lambda: paged._config(1, 2, 1, 64, 8, 32, past, 200, paged.F16, 64),
                 lambda: paged._config(1, 2, 1, 64, 8, 32, 3, past, paged.F16, 64)):
        with pytest.raises(ValueError, match="32 bits"):
            call()


@pytest.mark.parametrize("shape", [((1 << 32) + 1, 1, 64), (1, (1 << 32) + 1, 64), (1, 1, (1 << 32) + 64)])
def test_rows_past_32_bits_are_refused(shape):
    x = torch.zeros(1, 1, 1, device="meta").expand(shape)
    with pytest.raises(ValueError, match="32 bits"):
        paged.rotate(x, torch.empty(0, dtype=torch.int32, device="meta"), paged.Rope(64), out=x)


@pytest.mark.gpu
def test_one_token_of_odd_strides(torch_gpu):
    """A token cut from a row of another width is as good as one that was not; q may be rotated in place."""
    heads, group, dim = 2, 3, 64
    with paged.PagedKv(1, heads * group, heads, dim, 4, page=32, seqs=2, rope=paged.Rope(dim)) as kv:
        x = torch.randn(1, heads * (group + 2) * dim + 3, device="cuda").half()
        assert x.stride(0) % 8

        def parts(x):
            a = x[:, :heads * (group + 2) * dim].unflatten(1, (-1, dim))
            return a[:, :heads], a[:, heads:2 * heads], a[:, 2 * heads:]

        ones, got = torch.ones(80, heads, dim, device="cuda").half(), []
        kv.begin([0, 1], [40, 40])
        kv.append(0, ones, ones)
        for seq, y in enumerate((x, x[:, :-3].clone())):
            kv.begin([seq], [1])
            k, v, q = parts(y)
            r = kv.append(0, k, v, q)
            got.append((r, kv.attend(0, r, gate=q), kv.attend(0, q), kv.read_rows(0, 0, seq), kv.read_rows(0, 1, seq)))
            assert kv.append(0, k, v, q, q_out=q) is q and torch.equal(q, r)
        assert all(torch.equal(a, b) for a, b in zip(*got))


def test_rotate_refuses_rows_that_lie_on_each_other():
    """Two threads would write one place, or rotate it twice."""
    lib, turns = paged.lib(), paged.Rope(64)._ptr
    # rows, heads, strides of out; x elsewhere and in place
    for rows, heads, row, head in [(2, 1, 0, 64), (1, 2, 64, 0), (2, 3, 192, 63), (2, 3, -63, 64), (2, 2, 64, 64), (2, 2, 64, -64),
                                   (5, 1, 1, 0)]:
        for x in (64, 1 << 20):
            assert lib.mpg_rotate(turns, 0, rows, heads, 64, x, row, head, 64, 64, row, head, None) == -1, (rows, heads, row, head)
            assert b"on each other" in lib.mkv_last_error()
