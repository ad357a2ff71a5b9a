"""Sizes of projections with adapters at which the inputs are taken in several parts, by how the call is launched.  The plans are checked on the
CPU (tests/test_product_splits.py), so that a change of plan shows that a path has lost its test on the GPU (tests/test_gpu_product_splits.py)."""

# rows, outputs, inputs, adapters, rank: the main product's parts are summed up by a kernel of their own
JOINED = [(1, 300, 4096, 5, 24), (1, 1030, 4104, 5, 256), (17, 300, 4104, 5, 64), (17, 1030, 4096, 40, 16), (96, 300, 4096, 40, 40),
          (96, 1030, 4104, 5, 24), (600, 130, 4104, 7, 16)]
# and where it takes the adapters as more inputs: 128 x 64 tiles, 256 x 128 tiles, 256 x 128 tiles with rows left for smaller ones
MANY = [(700, 4096, 2056, 10, 24), (500, 5000, 4096, 5, 64), (3000, 4200, 1032, 11, 72), (3100, 4200, 4096, 11, 16), (4200, 4096, 2056, 11, 64),
        (4200, 4096, 4104, 5, 8)]
# groups, entries, outputs, inputs of products by expert, and the rows of their tiles
GROUPS = [(1024, 5000, 100, 72, 64), (1024, 60000, 300, 72, 128), (1024, 470000, 256, 64, 256)]
