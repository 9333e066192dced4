"""Sizes of fp8 products, one at least for each kernel that products take on 256 compute units, with rows, contraction and columns
off the tiles' sizes: (rows, contraction, columns), output type, x laid out before, the kernel and that of the rows behind the last
whole tiles."""
from pillarnet_lts_amd._lib import (PN_DTYPE_BF16 as BF16, PN_DTYPE_F32 as F32, PN_FP8_DIRECT_32 as D32, PN_FP8_DIRECT_64 as D64,
                                    PN_FP8_PAIR as PAIR, PN_FP8_TILE_64 as T64, PN_FP8_TILE_128 as T128)

CASES = [
    ((500, 3136, 256), BF16, 0, D32, 0), ((500, 3136, 256), F32, 0, D32, 0),            # x laid out on the way
    ((1000, 1000, 256), BF16, 0, D64, 0), ((1000, 1000, 256), F32, 0, D64, 0),
    ((512, 3136, 256), BF16, 1, D32, 0), ((104, 1160, 52), F32, 1, D32, 0),
    ((1439, 1290, 65), BF16, 1, D64, 0), ((1439, 1290, 65), F32, 1, D64, 0),
    ((2104, 1160, 69), BF16, 1, T64, 0), ((897, 1160, 8205), BF16, 1, T64, 0),          # ... several tiles a workgroup
    ((777, 1160, 900), F32, 1, T64, 0), ((7713, 1930, 1029), F32, 1, T64, 0),
    ((1031, 1160, 1030), BF16, 1, T128, 0), ((8728, 1160, 1799), BF16, 1, T128, 0),
    ((2312, 1160, 2312), F32, 1, T128, 0), ((1860, 1160, 8744), F32, 1, T128, 0),
    ((902, 1160, 8707), BF16, 1, PAIR, 0), ((5253, 1160, 7692), BF16, 1, PAIR, 0),
    ((3589, 5000, 1800), F32, 1, PAIR, 0), ((6314, 5129, 2200), F32, 1, PAIR, 0),
    ((4100, 1000, 2040), BF16, 0, PAIR, 0), ((4100, 1000, 2040), F32, 0, PAIR, D32),    # whole tiles and the rows behind them
    ((5129, 1160, 6314), BF16, 1, PAIR, D32), ((3589, 1160, 8967), BF16, 1, PAIR, D64),
    ((6284, 1160, 5126), BF16, 1, PAIR, T64), ((4484, 1160, 7222), BF16, 1, PAIR, T128),
    ((8197, 1160, 1991), F32, 1, PAIR, D32), ((7259, 1160, 2246), F32, 1, PAIR, D64), ((2124, 1160, 7691), F32, 1, PAIR, T64),
]
# training steps: the kernels of y, dx and dweight
TRAIN = [((512, 3136, 256), F32, (D32, T64, T64)), ((512, 3136, 256), BF16, (D32, T128, T64)),
         ((5129, 2200, 6314), BF16, (PAIR | D32 << 4, PAIR, PAIR))]


def products(m, k, n, dtype):
    """(rows, columns, contraction, output type) of a training step's three products, fp32 weights."""
    return (m, n, k, dtype), (m, k, n, dtype), (n, k, m, F32)
