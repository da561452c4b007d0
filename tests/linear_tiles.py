"""Sizes whose products take the linear kernel's tiles in every way, and the tiles they are there for: (columns of the
tile, whether the sum is split), 256 columns being a pair of CTAs on 256 rows; None where a size is not there for it."""

PAIR, PAIR_SPLIT, ONE, ONE_SPLIT = (256, False), (256, True), (128, False), (128, True)
# (M, K, N): forward, dx, dweight, in 16-bit types with an activation
SIZES = {
    (2500, 1536, 2048): (PAIR, PAIR, PAIR),             # whole 16-byte rows: everything by TMA
    (2000, 1300, 1900): (PAIR, PAIR, PAIR),             # ragged rows: operands copied, stores and residual by element
    (3000, 1029, 2101): (PAIR, PAIR, PAIR),              # odd ones
    (5000, 600, 2000): (PAIR, PAIR, PAIR_SPLIT),
    (20000, 512, 1024): (PAIR, PAIR, PAIR_SPLIT),
    (300, 8200, 2100): (PAIR_SPLIT, PAIR, PAIR),
    (40, 4096, 8192): (ONE_SPLIT, ONE_SPLIT, PAIR),
    (4096, 2048, 512): (ONE, PAIR, PAIR_SPLIT),
    (70001, 24, 20): ((64, False), (64, False), (64, True)),
}
