"""Forks of a prompt beside chunks on the GPU, where few rows and what the forks share go among the chunks' tiles, against the plain
64-bit form (tests/paged_reference.py). test_paged_share_chunks.py asserts that they go there."""
import pytest

from tests.test_gpu_paged_shared import Forest, pg  # noqa: F401
from tests.test_paged_share_chunks import BESIDE_CHUNKS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("name", BESIDE_CHUNKS)
def test_what_forks_share_among_a_chunks_tiles(torch_gpu, pg, name, typ):  # noqa: F811
    torch = torch_gpu
    heads, group, dim, page, prompt, forks, own, tokens, chunks, window = BESIDE_CHUNKS[name]
    f = Forest(torch, pg, heads, group, dim, typ, page, pages=(prompt + forks * (own + 300) + 6000) // page + 100, window=window)
    f.grow([0], [prompt])
    f.fork([0] * (forks - 1), list(range(1, forks)))
    f.grow(list(range(forks)), [own] * forks)
    others = list(range(forks, forks + len(chunks)))
    f.grow(others, [c[1] for c in chunks])
    f.begin(list(range(forks)) + others, [tokens] * forks + [c[0] for c in chunks], True)
    q = f.rnd(sum(f.batch[1]), heads * group, dim)
    out = f.check(q=q, what=name)
    assert torch.equal(out, f.kv.attend(0, q))
    f.check(sinks=torch.randn(heads * group, generator=f.g, device="cuda"), gate=True, what=name)
