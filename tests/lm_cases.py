"""Sizes at which the wide kernels of the language-model products run with
several tiles per worker, each with the tile width that the library is to take
for it (test_lm_dispatch.py), and their check on the GPU (test_lm_tiles_gpu.py).

A ragged-n case: lengths of the groups, m, k.
"""

# Last half-tiles of 16, 48, 80 and 112 tokens: an odd number of staged pieces
# of 16 columns per tile, 512 tiles of 128 columns for 148 workers, one slice of k.
ODD_PIECES = dict(lengths=[16, 48, 80, 112] * 4, m=4096, k=64)
