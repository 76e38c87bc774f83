"""Sizes at which the gated linear map's products run on each of their tiles, and those tiles as the plan's rule has to
choose them: (dtype, N, H, F) -> (v and g, x's gradient, the weights' gradients), columns by rows; v's and g's columns
count as two, OWN a kernel of its own. SHARED: those at which the last round's tiles of product 1 or 2 are shared out. Read by the test that runs them on the device and by the one that holds the rule to them."""

LARGE, MEDIUM, FLAT, OWN = (256, 256), (128, 128), (256, 32), (0, 0)

TILES = {
    ("float32", 1030, 776, 4610): (LARGE, LARGE, LARGE),
    ("bfloat16", 1030, 776, 4610): (LARGE, LARGE, LARGE),
    ("bfloat16", 1030, 832, 4616): (LARGE, LARGE, LARGE),
    ("bfloat16", 1100, 520, 3330): (LARGE, MEDIUM, MEDIUM),
    ("float32", 300, 136, 700): (MEDIUM, MEDIUM, MEDIUM),
    ("bfloat16", 300, 136, 700): (MEDIUM, MEDIUM, MEDIUM),
    ("float32", 30, 520, 600): (OWN, OWN, MEDIUM),
    ("bfloat16", 30, 520, 600): (OWN, FLAT, MEDIUM),
}

# (N, H, F) -> product, its tiles that a workgroup does alone, all
SHARED = {(4100, 1032, 6600): (2, 256, 260), (13300, 1031, 2056): (1, 256, 260)}
