"""Sizes beyond what one launch counts (its work-items in 32 bits) are refused as sizes, in front of it."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT
from test_mx4_host import FAKE, INT8, lib, mx, norm, operand, recorded, refused  # noqa: F401 (fixtures)

MOST = 1 << 32      # work-items that no launch has


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    at = tmp_path_factory.mktemp("limits")
    (at / "index.cpp").write_text('#include <cstdint>\n#include "index_math.h"\nextern "C" int fits(int64_t b, int t) { return ti8::idx::grid_fits(b, t); }\n'
                                  'extern "C" int norm_rows(int64_t d) { return ti8::idx::mx4_norm_rows(d); }\n')
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "triton-int8_amd", "csrc"), "-o", str(at / "index.so"), str(at / "index.cpp")], check=True)
    out = ctypes.CDLL(str(at / "index.so"))
    out.fits.argtypes, out.norm_rows.argtypes = [ctypes.c_int64, ctypes.c_int], [ctypes.c_int64]
    return out


@pytest.mark.parametrize("threads", [64, 128, 256, 512])
def test_what_a_launch_takes(index, threads):
    for blocks in (-1, 0, 1, MOST // threads - 1, MOST // threads, MOST // threads + 1, 1 << 31, 1 << 40):
        assert bool(index.fits(blocks, threads)) == (0 < blocks and blocks * threads < MOST), blocks


def most_rows(dim):
    return (1 << 24) - 1 if dim > 1024 else (1 << 26) - 4


@pytest.mark.parametrize("dim", [8, 512, 1024, 1032, 2048, 16384])
def test_rows_of_the_norm(lib, index, dim):  # noqa: F811
    per = index.norm_rows(dim)
    assert index.fits(-(-most_rows(dim) // per), 256) and not index.fits(-(-(most_rows(dim) + 1) // per), 256)
    for rows in (most_rows(dim) + 1, 1 << 28, (1 << 28) + 1):
        for to in (dict(mx4=mx(lib, rows, dim)), *([dict(mx4=lib.Mx4(), **{**INT8, "ldq": dim, "group": g}) for g in (0, 128)] if dim % 128 == 0 else [])):
            refused(lib, "ti8_rmsnorm_quant", 2, "rows", norm(lib, rows=rows, dim=dim, ldx=dim, ldr=dim, ldh=dim, **to), None)


@pytest.mark.parametrize("rows,cols", [(1 << 28, 512), ((1 << 28) - 31, 512), (1 << 25, 4096), (1 << 28, 1 << 28)])
def test_quantisers(lib, rows, cols):  # noqa: F811
    by_rows, by_columns = mx(lib, rows, cols), mx(lib, cols, rows)
    refused(lib, "ti8_mx4_quant", 2, "elements", operand(lib, ldx=cols, rows=rows, cols=cols, by_rows=by_rows), 1, None)
    refused(lib, "ti8_mx4_dequant", 2, "elements", by_rows, rows, cols, FAKE, cols, None)
    if rows * cols > 1 << 37:
        refused(lib, "ti8_mx4_quant", 2, "elements", operand(lib, ldx=cols, rows=rows, cols=cols, by_columns=by_columns), 1, None)
        refused(lib, "ti8_mx4_quant", 2, "elements", operand(lib, ldx=cols, rows=rows, cols=cols, by_rows=by_rows, by_columns=by_columns), 1, None)


@pytest.mark.parametrize("rows,cols,group", [(1 << 28, 128, 0), (1 << 23, 4096, 128), (1 << 28, 1 << 20, 0), (1 << 15, 1 << 20, 0)])
def test_dequant_row(lib, rows, cols, group):  # noqa: F811
    refused(lib, "ti8_dequant_row", 2, "elements", FAKE, cols, FAKE, rows, cols, group, FAKE, cols, None)


def test_products(lib):  # noqa: F811
    """Output tiles of 256 x 256 by 512 threads at most: from 2^39 elements of C on there are too many."""
    a, n = mx(lib, 1 << 28, 256), 1 << 14
    refused(lib, "ti8_mx4_gemm_nt", 2, "elements", a, 0, mx(lib, n, 256), 0, FAKE, n, 0, 1, 1 << 28, n, 256, 0, None, 0, None)


@pytest.mark.parametrize("dim,to", [(8, "mx4"), (1024, "int8"), (2048, "mx4")])
def test_rows_of_the_norm_from_python(recorded, dim, to):  # noqa: F811
    """(Rows that share their memory: none of it is read.)"""
    T, calls = recorded
    w, one = torch.zeros(dim, dtype=torch.bfloat16), torch.zeros(1, dim, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="rows"):
        T.ops.rmsnorm_quant(one.expand(most_rows(dim) + 1, -1), w, 1e-5, to=to)
    assert not calls
