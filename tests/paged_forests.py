"""Batches of forks by how their work is cut: every sequence by itself, what they share in tiles of 32 rows beside their own, or in
a chunk's tiles. test_paged_share.py asserts that they go there, test_gpu_paged_shared.py runs them."""

# name: kv_heads, group, dim, page, prompt, forks, own part up to, tokens in turn, window, kinds of the shared tiles (none: apart)
FORESTS = {
    "short prompts, apart": (2, 4, 128, 64, 700, 4, 40, [1], 0, ()),
    "samples, tiles of 32": (4, 8, 128, 64, 9000, 4, 100, [1], 0, (1,)),
    "samples, tiles of 32, 64": (8, 4, 64, 32, 3000, 24, 200, [1], 0, (1,)),
    "samples, tiles of 32, 256": (2, 8, 256, 64, 5000, 12, 90, [1], 0, (1,)),
    "samples, tiles of 128": (4, 8, 128, 64, 6000, 50, 300, [1], 0, (2,)),
    "samples, tiles of 128, 256": (2, 8, 256, 32, 7000, 30, 90, [1], 0, (2,)),
    "verifies, tiles of 128, 256": (1, 16, 256, 128, 12000, 16, 150, [4, 4, 4, 2], 0, (2,)),
    "verifies, tiles of 256, 64": (2, 8, 64, 64, 16000, 40, 500, [4], 0, (3,)),
    "verifies, tiles of 128": (1, 8, 128, 64, 14000, 60, 200, [4], 0, (2,)),
    "some verify, some generate": (2, 5, 128, 128, 8000, 17, 150, [1, 4, 2], 0, (1,)),
    "a window inside the prompt": (2, 8, 128, 32, 6000, 40, 300, [1, 2], 3000, (2,)),
    "a window's edge inside the tiles": (4, 8, 128, 64, 5000, 60, 1400, [1], 4500, (2,)),
    "a window past the prompt": (2, 8, 128, 64, 2000, 9, 1000, [1], 33, ()),
    "chunks beside generation": (2, 4, 128, 64, 9000, 30, 100, [1, 1, 1, 1, 1, 130, 1], 0, (2,)),
    "one query head a head": (3, 1, 64, 256, 9000, 40, 300, [1, 3], 0, (1,)),
}
