"""Sizes that reach every kernel of the language-model products, most with
several tiles per worker: checked on the GPU (test_lm_tiles_gpu.py), with the
tile widths they are there for, which the library has to choose on 148 SMs
(test_lm_dispatch.py).
"""

# Last half-tiles of 16, 48, 80 and 112 tokens: an odd number of staged pieces
# of 16 columns per tile, 512 tiles of 128 columns for 148 workers, one slice of k.
ODD_PIECES = dict(name="odd pieces", lengths=[16, 48, 80, 112] * 4, m=4096, k=64, bf16=128, fp8=128)

# Prompts: pairs of CTAs on 256 x 256 tiles. Groups end inside either half of a
# tile, after 16, 48 and 192 columns of it; one is empty.
PROMPTS = [
    dict(name="one slice", lengths=[1040, 0, 1072, 1984], m=4096, k=64, bf16=256, fp8=256),
    dict(name="ragged slices", lengths=[1040, 0, 1072, 1984], m=4096, k=136, bf16=256, fp8=256),
    # Nothing a multiple of anything; weights, tokens and results of odd rows.
    dict(name="odd", lengths=[2999, 1, 0, 1303, 777, 33], m=1999, k=391, bf16=256, fp8=256),
    # Whole tiles of 128 and 256 tokens, and ends just past them.
    dict(name="edges", lengths=[256, 128, 257, 129, 1024, 1025, 511, 513], m=4112, k=272, bf16=256,
         fp8=256),
    # Several chunks of k, and more than four blocks of scales.
    dict(name="deep", lengths=[700, 0, 1500, 900], m=3000, k=1100, bf16=256, fp8=256),
    dict(name="one group", lengths=[3333], m=3000, k=328, bf16=256, fp8=256),
]

# Decoding: the thin kernels, alone and in clusters that share k.
DECODING = [
    dict(name="few", lengths=[1, 0, 9, 17, 2, 4] * 6, m=1999, k=136, bf16=16, fp8=16),
    dict(name="few, deep", lengths=[2, 7, 0, 5] * 6, m=2000, k=4200, bf16=16, fp8=16),
    dict(name="some", lengths=[12, 1, 33, 0, 7, 15] * 4, m=1999, k=328, bf16=32, fp8=32),
    dict(name="idle SMs", lengths=[64, 1, 0, 63, 65, 40], m=700, k=2100, bf16=64, fp8=64),
]

RAGGED = [ODD_PIECES] + PROMPTS + DECODING

# Gradients of weights: m, n.
GRADIENTS = [(1536, 1000), (1177, 1003)]

# Orthogonalised matrices: rows, columns, batch.
ORTHOGONAL = [(1290, 1030, 4), (770, 515, 8), (1500, 1001, 2), (1020, 1530, 2), (530, 1500, 2),
              (1290, 520, 2), (1290, 515, 1), (270, 1500, 2), (200, 300, 2), (770, 510, 1), (512, 513, 4)]
