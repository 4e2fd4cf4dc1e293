"""Batches that reach the long plans of the 16-bit cache's attention, and what each is there for: ``tests/test_attention16_cuts.py``
holds them to it on the host, ``tests/test_gpu_kv16_plans.py`` runs them."""

# name: (heads, kv heads, head size, page size, [(length, rows)], what the plan has to be)
PLANS = {
    # eight waves for 128 columns' tokens, nothing to join: an even and an odd number of tiles, a last tile of one token
    "eight waves": (28, 4, 128, 64, [(1777, 1777)], {"parts": 2, "combine": 0, "tile_longest": 28}),
    "eight waves, odd": (28, 4, 128, 32, [(1600, 1600)], {"parts": 2, "combine": 0, "tile_longest": 25}),
    "eight waves, one more": (28, 4, 128, 128, [(1601, 1601)], {"parts": 2, "combine": 0, "tile_longest": 26}),
    "eight waves, kv heads": (16, 16, 128, 16, [(2500, 2500)], {"parts": 2, "combine": 0, "tile_longest": 40}),
    "eight waves, heads of 64": (14, 2, 64, 16, [(2500, 2500)], {"parts": 2, "combine": 0, "tile_longest": 40}),
    "eight waves behind a context": (28, 4, 128, 16, [(5000, 1300)], {"parts": 2, "combine": 0, "tile_longest": 79}),
    "eight waves, several": (28, 4, 128, 64, [(700, 600), (600, 600), (1900, 580)], {"parts": 2, "combine": 1, "tile_longest": 30}),
    # four waves, whole: the longest prompts', past the 64 pages that a lane each has
    "whole": (28, 4, 128, 16, [(2500, 2500)], {"parts": 1, "combine": 0, "tile_longest": 40, "tile_sums": 0}),
    "whole, kv heads": (16, 16, 128, 64, [(4100, 4100)], {"parts": 1, "combine": 0, "tile_longest": 65, "tile_sums": 0}),
    "whole, heads of 64": (12, 12, 64, 16, [(5500, 5500)], {"parts": 1, "combine": 0, "tile_longest": 86, "tile_sums": 0}),
    "whole, several": (28, 4, 128, 16, [(1500, 900), (3000, 1700)], {"parts": 1, "combine": 1, "tile_longest": 47, "tile_sums": 0}),
    # split along the tokens, items of more pages than a lane each has
    "split": (28, 4, 128, 16, [(20000, 600)], {"parts": 1, "combine": 1, "tile_longest": 105, "tile_sums": 1}),
    "split, heads of 64": (14, 2, 64, 16, [(16000, 400), (9000, 333)], {"parts": 1, "combine": 1, "tile_sums": 1}),
}
