"""Sizes of dense products that take the paths their tests are for.  (tokens, k, results a row)"""

# 4 bits, more than 128 tokens: some or all tiles are split among the pairs of a cluster.  The first three have no other tiles.
SPLIT_PRODUCTS = [(512, 12288, 4096), (130, 4096, 513), (300, 8224, 1000), (2500, 8192, 2048)]
SPLIT_GATED = [(200, 8192, 1024), (200, 8192, 1056), (129, 6176, 96), (1300, 8192, 2048)]
# Up to 128 tokens: more tiles of 128 results than blocks at once (two an SM up to 64 tokens), so that a block takes several
SEVERAL_A_BLOCK_PRODUCTS = [(8, 96, 70000), (30, 352, 70000), (60, 96, 70001), (100, 288, 40000)]
SEVERAL_A_BLOCK_GATED = [(8, 96, 40032), (30, 160, 40000), (60, 96, 40064), (100, 288, 40000)]
