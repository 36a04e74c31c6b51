"""Sizes (rows, K, N) that take each kernel of linear8 and of its weight's gradient, and which one the library says it takes."""
import ctypes as C

import self_forcing_amd as sfa

# 256-row tiles: a half last strip and pipelines of 1, 2, 4 and 5 stages, a strip of 204 rows, whole strips
TILE_256 = {(4200, 100, 5003): 1, (4200, 200, 5000): 1, (4200, 390, 5003): 1, (4200, 640, 5003): 1, (4300, 300, 5003): 0, (4352, 300, 5000): 0}
# 128-row tiles: pipelines of 1, 2, 3, 4 and 5 stages, whole strips and one of 74 rows
TILE_128 = [(2304, 100, 2101), (2304, 200, 2100), (2250, 300, 2101), (2304, 390, 2101), (2250, 640, 2101)]
NO_TILE = [(528, 512, 256), (600, 200, 130), (12, 256, 64)]
# the weight's gradient, 256 x 256 tiles: one part, rows from one to nineteen steps with and without a last one that is not whole;
# several parts.  K of 3900, 1408: the last tile has one block.  N of 4001, 1501, 1029: rows of dy end inside a piece of 8 channels
WGRAD_256 = {(1, 3900, 4001): 1, (32, 4096, 4000): 1, (33, 3900, 4001): 1, (97, 3900, 4000): 1, (130, 4001, 4001): 1, (161, 3900, 4001): 1,
             (600, 3000, 3001): 1, (600, 3900, 4008): 1, (4680, 1500, 1501): 6, (4680, 1536, 1536): 6, (8000, 1408, 1029): 8}


def product_plan(M, K, N):
    """(rows of a tile or 0, whether the last strip is half)"""
    a, b = C.c_int32(0), C.c_int32(0)
    sfa.lib.check(sfa.lib.load().sfm_linear8_plan(M, N, K, C.byref(a), C.byref(b)))
    return a.value, b.value


def wgrad_plan(M, K, N):
    """(channels of a tile, parts of the rows)"""
    a, b = C.c_int32(0), C.c_int32(0)
    sfa.lib.check(sfa.lib.load().sfm_linear8_wgrad_plan(M, N, K, C.byref(a), C.byref(b)))
    return a.value, b.value
