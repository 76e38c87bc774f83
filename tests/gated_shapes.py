"""Sizes at which the gated linear map's products run on each of their tiles, and those tiles as the plan's rule has to
choose them: (dtype, N, H, F) -> (v and g, x's gradient, the weights' gradients), columns by rows; v's and g's columns count
as two. Read by the test that runs them on the device and by the one that holds the rule to them."""

LARGE, MEDIUM, FLAT = (256, 256), (128, 128), (256, 32)

TILES = {
    ("float32", 1030, 776, 4610): (LARGE, LARGE, LARGE),
    ("bfloat16", 1030, 776, 4610): (LARGE, LARGE, LARGE),
    ("bfloat16", 1030, 832, 4616): (LARGE, LARGE, LARGE),
    ("bfloat16", 1100, 520, 3330): (LARGE, MEDIUM, MEDIUM),
    ("float32", 300, 136, 700): (MEDIUM, MEDIUM, MEDIUM),
    ("bfloat16", 300, 136, 700): (MEDIUM, MEDIUM, MEDIUM),
    ("float32", 30, 520, 600): (FLAT, FLAT, MEDIUM),
    ("bfloat16", 30, 520, 600): (FLAT, FLAT, MEDIUM),
}
