"""Shapes of the experts' products that the kernels on CTA pairs are to take, in the forward pass too: ``test_grouped_rules.py`` holds them to the rule in
``csrc/mmoe_grouped_few.cu`` for the 148 multiprocessors of a B200, ``test_gpu_grouped_pairs.py`` computes them."""

SMS = 148
BF16, E4M3 = 0, 4
LINEAR, GATED = 0, 1

# blocks and their parts in 16 bits: (rows, experts, hidden, inter); no width is whole stages of 64, nor whole tiles
BLOCKS = {
    "values": (241, 6, 1416, 1352),
    "replays": (600, 4, 1032, 520),
    "bad ends": (400, 3, 1416, 712),
    "strides": (300, 3, 1928, 968),
}
# (rows, experts, width, channels)
PROJECTIONS = {"room": (700, 2, 72, 1176)}
# 8 bits: (rows, experts, width, channels; of a gated one, gate and up rows together)
EIGHT_BITS = {
    "values": (640, 6, 272, 528),
    "replays": (600, 4, 272, 288),
    "bad ends": (400, 3, 144, 144),
    "room": (700, 2, 80, 67),
}


def products():
    """``(type, kind, rows, experts, channels, width)`` of every forward product of the above."""
    for rows, experts, hidden, inter in BLOCKS.values():
        yield BF16, GATED, rows, experts, inter, hidden
        yield BF16, LINEAR, rows, experts, hidden, inter
        yield BF16, LINEAR, rows, experts, 2 * inter, hidden
    for rows, experts, width, channels in PROJECTIONS.values():
        yield BF16, LINEAR, rows, experts, channels, width
    for rows, experts, width, channels in EIGHT_BITS.values():
        yield E4M3, LINEAR, rows, experts, channels, width
        if channels % 16 == 0:
            yield E4M3, GATED, rows, experts, channels // 2, width
