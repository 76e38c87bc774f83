"""Sizes at which linear cross entropy's products run on each of their tiles, and those tiles as the plan's rule has to
choose them: (dtype, N, H, V, reduction) -> (logits, hidden's gradient, weight's gradient), columns by rows. Read by the
test that runs them on the device and by the one that holds the rule to them."""

LARGE, MEDIUM, FLAT, FEW32, MORE32 = (256, 256), (128, 128), (256, 32), (128, 32), (128, 64)

TILES = {
    # 256 x 256 everywhere: W in planes, packed (a width that is no multiple of 64, of 8) and where it is
    ("float32", 1030, 776, 9001, "mean"): (LARGE, LARGE, LARGE),
    ("float32", 1029, 779, 9001, "none"): (LARGE, LARGE, LARGE),
    ("bfloat16", 1030, 776, 9001, "mean"): (LARGE, LARGE, LARGE),
    ("bfloat16", 1029, 779, 9001, "sum"): (LARGE, LARGE, LARGE),
    ("bfloat16", 1100, 832, 9001, "none"): (LARGE, LARGE, LARGE),
    # dz in two planes
    ("bfloat16", 256, 1032, 33001, "none"): (LARGE, LARGE, LARGE),
    ("bfloat16", 200, 1032, 27001, "none"): (MEDIUM, LARGE, MEDIUM),
    ("bfloat16", 30, 520, 6001, "none"): (FLAT, FLAT, MEDIUM),
    # the others beside them
    ("float32", 700, 136, 7001, "mean"): (MEDIUM, MEDIUM, MEDIUM),
    ("float32", 30, 8, 1100003, "mean"): (FLAT, FLAT, MEDIUM),
    ("float32", 30, 523, 6001, "mean"): (FEW32, FEW32, MEDIUM),
    ("float32", 300, 523, 6001, "mean"): (MORE32, MORE32, MEDIUM),
    ("bfloat16", 700, 136, 7001, "mean"): (MEDIUM, MEDIUM, MEDIUM),
    ("bfloat16", 30, 520, 6001, "mean"): (FLAT, FLAT, MEDIUM),
}
