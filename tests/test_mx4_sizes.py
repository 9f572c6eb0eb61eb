"""The sizes that the GPU tests multiply reach every kernel of the 4-bit products (mx4_sizes.py); a planner that sends them elsewhere fails here."""
import ctypes

import pytest

import mx4_sizes
from test_mx4_index import index, planned  # noqa: F401 (a fixture)


def tiles(k):
    return -(-k // 256)


def together(index, sizes):  # noqa: F811
    return index.together(((ctypes.c_int64 * 3) * len(sizes))(*((ctypes.c_int64 * 3)(m, n, tiles(k)) for m, n, k in sizes)), len(sizes), 256)


@pytest.mark.parametrize("shape,kernel,parts", mx4_sizes.ALONE, ids=str)
def test_products_alone(index, shape, kernel, parts):  # noqa: F811
    batch, m, n, k = shape
    assert planned(index, m, n, tiles(k), batch)[:2] == (kernel, parts)


@pytest.mark.parametrize("sizes,kernel", mx4_sizes.TOGETHER, ids=str)
def test_products_together(index, sizes, kernel):  # noqa: F811
    assert together(index, sizes) == kernel


def test_all_kernels_are_reached():
    alone = {(kernel, parts) for _, kernel, parts in mx4_sizes.ALONE}
    assert {k for k, p in alone if p == 1} == set(range(8)) == {k for _, k in mx4_sizes.TOGETHER} - {mx4_sizes.APART}
    for kernel in (mx4_sizes.TILES_32, mx4_sizes.TILES_64, mx4_sizes.TILES_64_128, mx4_sizes.TILES_128):
        assert {p for k, p in alone if k == kernel} >= {2, 4, 8}, kernel
    # (of one and of several batches, where a batch's part of C begins elsewhere)
    assert {kernel for (batch, *_), kernel, _ in mx4_sizes.ALONE if batch > 1} == set(range(8))
    assert {parts for (batch, *_), _, parts in mx4_sizes.ALONE if batch > 1} >= {1, 8}
    # rows, columns and contractions that end inside a tile
    for (_, m, n, k), kernel, _ in mx4_sizes.ALONE:
        assert k % 256 and (m % 32 or n % 32)


@pytest.mark.parametrize("sizes", [*mx4_sizes.TOGETHER_IN_PARTS, *([(t, n, k), (t, k, n), (n, k, t)] for t, k, n in mx4_sizes.STEPS_IN_PARTS)], ids=str)
def test_sets_that_need_a_workspace(index, sizes):  # noqa: F811
    assert together(index, sizes) == mx4_sizes.APART and max(planned(index, m, n, tiles(k))[1] for m, n, k in sizes) > 1
