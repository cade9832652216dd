"""The forms in which matrices of a size are orthogonalised, and a size for each (z1_orthogonalize_way)."""
import ctypes

PRODUCTS = ('A', 'square', 'X')


def forms(lib, count, m, n, precise):
    """What a size takes: ('small', fragments to a wave, rows of fragments, whether pairs), or for each product
    its tile, whether quarters take the rest, whether the summed axis is cut, and the blocks staged."""
    way = (ctypes.c_int * 12)()
    assert lib.z1_orthogonalize_way(count, m, n, precise, way) == 0
    if way[0] == 0:
        return {('small', way[1], (min(m, n) + 31) // 32, way[2])}
    return {(PRODUCTS[i], way[4 * i], way[4 * i + 1] > 0, way[4 * i + 2] > 1, way[4 * i + 3]) for i in range(3)}


# (count, m, n)
FAST = [(2, 20, 31), (2, 60, 61), (2, 72, 65), (2, 1, 428), (2, 103, 35), (2, 99, 68), (2, 106, 98), (151, 206, 195),
        (11, 630, 577), (1, 1980, 7200), (1, 1497, 3635), (28, 694, 698), (110, 426, 660), (51, 658, 807), (2, 1025, 2),
        (1, 3198, 40), (12, 1602, 1643), (3, 1263, 1033), (1, 2116, 967), (5, 1156, 1333), (18, 1109, 775), (13, 1072, 922),
        (2, 20, 200), (2, 40, 90)]
PRECISE = [(2, 20, 31), (2, 35, 33), (2, 1, 291), (2, 33, 106), (2, 77, 69), (97, 210, 217), (59, 204, 196), (1, 3422, 1936),
           (1, 1960, 1518), (56, 418, 485), (12, 1731, 1744), (101, 467, 402), (2, 1, 897), (1, 1052, 1), (7, 390, 1166),
           (100, 199, 67), (49, 337, 386), (57, 530, 457), (159, 479, 151),
           (2, 526, 1294), (1, 3753, 1477), (289, 223, 206)]
