"""The kernels that the sizes of the GPU tests take, with 256 compute units, and the refusals of the queries."""
import ctypes as C

import pytest

from linear8_sizes import NO_TILE, TILE_128, TILE_256, WGRAD_256, product_plan, wgrad_plan
from self_forcing_amd import lib as L


def test_products():
    for size, half in TILE_256.items():
        assert product_plan(*size) == (256, half), size
    for size in TILE_128:
        assert product_plan(*size) == (128, 0), size
    for size in NO_TILE:
        assert product_plan(*size) == (0, 0), size
    # a chunk through the block's layers
    assert [product_plan(4680, *s) for s in ((1536, 8960), (8960, 1536), (1536, 4608), (1536, 1536))] == [(256, 1), (128, 0), (256, 1), (128, 0)]


def test_weights_gradients():
    for size, parts in WGRAD_256.items():
        assert wgrad_plan(*size) == (256, parts), size
    assert [wgrad_plan(4680, *s) for s in ((1536, 8960), (8960, 1536), (1536, 4608), (1536, 1536))] == [(256, 1), (256, 1), (256, 2), (256, 6)]


@pytest.mark.parametrize("query", ["sfm_linear8_plan", "sfm_linear8_wgrad_plan"])
def test_refusals(query):
    n, ask = C.c_int32(0), getattr(L.load(), query)
    for args, code in (((4, 4, 4, None, C.byref(n)), -1), ((4, 4, 4, C.byref(n), None), -1), ((0, 4, 4, C.byref(n), C.byref(n)), -3),
                       ((4, 1 << 23, 4, C.byref(n), C.byref(n)), -3)):
        assert ask(*args) == code
