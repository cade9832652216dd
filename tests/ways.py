"""Every form of the product and weight gradient kernels, with a ragged shape that runs in it, and a query of how a shape runs.

A product's form: rows and columns of a tile, blocks of K staged (0: the few rows' kernel), whether K goes in parts.  A weight
gradient's: rows and columns of a tile, whether its rows go straight into LDS, whether the tokens go in parts, and, where they
do not go straight, whether a row has less than 8 elements."""
import ctypes

PRODUCTS = {                                          # form: (M, N, K)
    (8, 8, 0, False): (5, 70, 700),
    (16, 16, 0, False): (9, 900, 300),
    (32, 32, 0, False): (20, 300, 1000),
    (64, 32, 0, False): (50, 2100, 700),
    (64, 64, 4, False): (100, 1501, 1000),
    (64, 64, 4, True): (100, 257, 4100),
    (64, 128, 4, False): (600, 3000, 4100),
    (64, 128, 4, True): (1575, 562, 7541),
    (128, 128, 2, False): (2040, 4090, 520),
    (128, 128, 2, True): (750, 1380, 3200),
    (128, 128, 4, False): (1000, 3000, 700),
    (128, 128, 4, True): (510, 1076, 3214),
    (128, 192, 4, False): (1200, 3300, 900),
    (256, 256, 2, False): (2200, 3700, 600),
}
GRADIENTS = {                                         # form: (tokens, N, K)
    (64, 64, 0, False, True): (70, 7, 40),
    (64, 64, 0, True, True): (5000, 7, 400),
    (64, 64, 0, False, False): (333, 1501, 1000),
    (64, 64, 0, True, False): (3001, 65, 300),
    (128, 128, 0, False, False): (1000, 1501, 1500),
    (128, 128, 0, True, False): (3000, 1031, 1000),
    (64, 64, 1, False, False): (200, 300, 500),
    (64, 64, 1, True, False): (3001, 600, 300),
    (128, 128, 1, False, False): (1000, 1500, 1500),
    (128, 128, 1, True, False): (3001, 1030, 1000),
    (256, 192, 1, False, False): (333, 4000, 3000),
    (256, 256, 1, False, False): (100, 1300, 8600),
}


def _ask(fn, *args):
    way = (ctypes.c_int * 4)()
    assert fn(*args, way) == 0, args
    return tuple(way)


def product(lib, M, N, K):
    rows, outputs, stages, parts = _ask(lib.z1_product8_way, M, N, K)
    return rows, outputs, stages, parts > 1


def gradient(lib, T, N, K, whole_dwords):
    rows, columns, direct, parts = _ask(lib.z1_weight_grad8_way, T, N, K, int(whole_dwords))
    return rows, columns, direct, parts > 1, not direct and N < 8
