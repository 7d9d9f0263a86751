"""Steps of drafted tokens that between them take every kernel of esda_tree_decode, with K and V apart and one, with
a merge and without: test_tree_forms.py pins the kernel of each on the host, test_tree_forms_gpu.py runs them."""

ONE = 2 ** 31 - 32  # split_rows of a single piece
SHORT, BATCH = [60, 150, 3], [90, 0, 33, 70, 95]
# D, query heads, kv heads, nodes, lengths, room of a sequence in rows, split_rows -> the kernel's kind, query rows of a
# workgroup, waves, pieces; with K and V apart and as one
BOTH = [
    ((128, 8, 2, 4, SHORT, 176, ONE), "run 16 4 one"), ((128, 8, 2, 4, [500, 601], 640, 0), "run 16 4 split"),
    ((128, 8, 2, 12, [300, 41], 640, 0), "run 16 4 split"),  # three workgroups of the same keys
    ((128, 16, 1, 20, [100, 7], 160, ONE), "run 32 4 one"), ((128, 16, 1, 20, [600], 640, 0), "run 32 4 split"),
    ((128, 64, 4, 64, BATCH, 160, 0), "tile 128 4 one"), ((128, 64, 4, 64, [1200, 0, 33, 700, 95], 1280, 0), "tile 128 4 split"),
    ((256, 8, 2, 4, SHORT, 176, ONE), "run 16 4 one"), ((256, 8, 2, 4, [500, 601], 640, 0), "run 16 4 split"),
    ((256, 8, 1, 7, [100, 7], 160, ONE), "tile 64 8 one"), ((256, 16, 2, 20, [601, 40], 640, 0), "tile 64 8 split"),
    ((256, 64, 4, 64, BATCH, 160, 0), "tile 128 8 one"), ((256, 64, 4, 64, BATCH, 160, 96), "tile 128 8 split"),
    ((512, 8, 2, 4, SHORT, 176, ONE), "run 16 4 one"), ((512, 8, 2, 4, [500, 601], 640, 0), "run 16 4 split"),
    ((512, 16, 1, 20, [100, 3], 160, ONE), "tile 64 4 one"), ((512, 16, 1, 20, [600], 640, 0), "tile 64 4 split"),
    ((512, 64, 4, 64, BATCH, 160, 0), "tile 128 8 one"), ((512, 64, 4, 64, BATCH, 160, 96), "tile 128 8 split"),
    ((512, 64, 4, 12, [1200, 300], 1280, 0), "tile 128 8 split"),
]
# 64 query rows of 512 dims, which one tile holds: of four waves for K = V, of eight for K and V apart
SHARED = [((512, 16, 2, 8, [9000, 700], 20000, ONE), "tile 64 4 one"), ((512, 16, 2, 8, [9000, 700], 20000, 0), "tile 64 4 split")]
APART = [((512, 8, 1, 7, [3000, 1], 8992, ONE), "tile 128 8 one"), ((512, 8, 1, 7, [3000, 1], 8992, 0), "tile 128 8 split")]
STEPS = [(step, shared, form) for shared in (False, True) for step, form in BOTH + (SHARED if shared else APART)]
