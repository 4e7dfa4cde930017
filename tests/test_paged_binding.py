"""The paged cache's Python binding: what it keeps, and what it refuses by itself."""
import copy
import ctypes
import pickle

import pytest

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
