"""Batches of the paged cache by the kernels their work goes to: few rows (tiles of 16 and 32), chunks (tiles of 128 and 256
rows), whole and split over the keys. test_paged_book.py asserts that they go there, test_gpu_paged_shapes.py runs them."""

# name: dim, kv_heads, group, window, [(new tokens, length)], kind of tile, split over the keys
UNEVEN = [(1, 100 * i * i + 50) for i in range(1, 9)] * 8
SHAPES = {
    "one token, many splits": (128, 1, 8, 0, [(1, 20000)], 0, True),
    "four tokens, many splits": (256, 2, 8, 0, [(4, 9000)], 1, True),
    "uneven tokens, tiles of a third of the places": (64, 1, 4, 0, UNEVEN[:8] * 11, 0, True),
    "uneven tokens": (128, 4, 4, 0, UNEVEN, 0, True),
    "uneven pairs of tokens": (256, 4, 5, 0, [(2, n + 1) for _, n in UNEVEN + UNEVEN[:16]], 0, True),
    "many short ones": (64, 8, 2, 0, [(1, n) for n in range(1, 60)], 0, False),
    "few rows, many of their splits": (64, 1, 64, 0, [(4, 3000)], 2, True),
    "chunk of 40, many splits": (128, 2, 8, 0, [(40, 9001)], 2, True),
    "chunk of 200, nine splits": (64, 1, 16, 0, [(200, 9001)], 2, True),
    "decodes among chunks": (128, 4, 8, 513, [(700, 700), (256, 3001), (33, 97)] + [(1, 400 * i + 5) for i in range(10)], 2, False),
    "decodes among chunks, split": (256, 2, 8, 0, [(1, 1003), (300, 2000), (4, 1001), (300, 2011), (1, 5), (2, 999)], 2, True),
    "decodes among a short chunk": (64, 4, 8, 0, [(1, 30), (100, 300)] + [(1, 37 * i + 1) for i in range(10)], 2, False),
    "last round of chunks cut": (128, 4, 8, 0, [(1050, 8000)], 2, True),
    "prompt of small tiles": (256, 2, 8, 700, [(1037, 1037)], 2, False),
    "prompts of large tiles, 64": (64, 8, 16, 4096, [(163, 164), (185, 185)], 3, False),
    "prompts of large tiles, 128": (128, 8, 16, 100, [(107, 107), (95, 111), (159, 159), (73, 73)], 3, False),
    "prompts of large tiles, 256": (256, 8, 16, 513, [(291, 291), (222, 222), (112, 112), (85, 85)], 3, False),
    "large tiles split, 64": (64, 8, 4, 0, [(116, 116), (48, 10219), (41, 41), (141, 141)], 3, True),
    "large tiles split, 128": (128, 2, 8, 4096, [(42, 42), (831, 2932), (399, 1065), (41, 41)], 3, True),
    "large tiles split, 256": (256, 2, 8, 0, [(96, 30066), (968, 968)], 3, True),
}
