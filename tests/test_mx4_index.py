"""Index arithmetic of the 4-bit products and quantisers (csrc/index_math.h), compiled for the host, and what their compiled code waits for."""
import ctypes
import os
import re
import subprocess

import pytest

from conftest import ROOT
from test_kernel_resources import VMEM, kernel_bodies, loops

CODE = r"""
#include <cstdint>
#include "index_math.h"
using namespace ti8::idx;
extern "C" int64_t range(int64_t block, int64_t blocks) { return xcd_range(block, blocks); }
extern "C" void part(int p, int parts, int nk, int* out) { const Mx4Part q = mx4_part(p, parts, nk); out[0] = q.first; out[1] = q.tiles; }
extern "C" void plan(int64_t M, int64_t N, int64_t nk, int64_t batch, int cus, double* out) { const Mx4Plan p = mx4_plan(M, N, nk, batch, cus); out[0] = p.kernel; out[1] = p.parts; out[2] = p.us; }
extern "C" int together(const int64_t (*sizes)[3], int count, int cus) { return mx4_plan_together(sizes, count, cus); }
extern "C" int pick(int block, int first1, int first2, int count) { return gemm_multi_pick(block, first1, first2, count); }
extern "C" int swizzle(int row) { return (int)mx4_chunk_swizzle(row); }
extern "C" int chunk(int wave, int octet, int waves) { return mx4_col_chunk(wave, octet, waves); }
extern "C" int row(int r, int rows) { return mx4_row(r, rows); }
extern "C" int behind(int stages, int loads, int scales) { return mx4_behind(stages, loads, scales); }
extern "C" int64_t tiles(int64_t c) { return mx4_tiles(c); }
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    at = tmp_path_factory.mktemp("mx4_index")
    (at / "index.cpp").write_text(CODE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "triton-int8_amd", "csrc"), "-o", str(at / "index.so"), str(at / "index.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "index.so"))
    for name in ("range", "tiles"):
        getattr(lib, name).restype, getattr(lib, name).argtypes = ctypes.c_int64, [ctypes.c_int64] * (2 if name == "range" else 1)
    lib.plan.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_int, ctypes.POINTER(ctypes.c_double)]
    return lib


@pytest.mark.parametrize("blocks", [*range(1, 34), 255, 256, 257, 1000, 2047])
def test_ranges_of_the_xcds_are_a_permutation(index, blocks):
    to = [index.range(b, blocks) for b in range(blocks)]
    assert sorted(to) == list(range(blocks))
    for xcd in range(min(8, blocks)):       # (workgroups go round the XCDs: each has one range without a gap)
        mine = to[xcd::8]
        assert mine == list(range(mine[0], mine[0] + len(mine)))


def test_parts_of_a_contraction_cover_it(index):
    out = (ctypes.c_int * 2)()
    for nk in range(1, 70):
        for parts in range(1, min(nk, 8) + 1):
            at = 0
            for p in range(parts):
                index.part(p, parts, nk, out)
                assert out[0] == at and out[1] >= 1
                at += out[1]
            assert at == nk


def planned(index, m, n, nk, batch=1, cus=256):
    out = (ctypes.c_double * 3)()
    index.plan(m, n, nk, batch, cus, out)
    return int(out[0]), int(out[1]), out[2]


SIZES = [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 200, 333, 512, 1000, 4096, 5000, 14336, 100000, 1 << 28]


@pytest.mark.parametrize("cus", [256, 32, 304])
def test_every_product_has_a_kernel(index, cus):
    """Only up to 32 rows go to the kernels for few, up to 64 to tiles of 32; parts are no more than K tiles, and one where a launch of all tiles has no room for more."""
    tile = {2: (32, 64), 3: (64, 64), 4: (128, 128), 5: (128, 128), 6: (256, 256), 7: (64, 128)}
    for m in SIZES:
        for n in SIZES:
            for nk in (1, 2, 3, 4, 8, 16, 56, 1000, 1 << 14):
                for batch in (1, 5, 65535):
                    kernel, parts, us = planned(index, m, n, nk, batch, cus)
                    assert 0 <= kernel <= 7 and 1 <= parts <= 8 and parts <= nk and 0 < us < 1e30, (m, n, nk, batch)
                    assert kernel > 1 or (m <= 16 * (kernel + 1) and -(-n // 16) * batch <= cus)
                    assert kernel != 2 or m <= 64
                    if parts > 1:
                        bm, bn = tile[kernel]
                        assert -(-m // bm) * -(-n // bn) * batch * parts <= cus


def test_products_together_have_a_kernel_for_all_of_them(index):
    shapes = [(m, n, nk) for m in (1, 16, 17, 32, 33, 64, 65, 700, 8192) for n in (1, 1000, 4096, 14336) for nk in (1, 16, 56)]
    seen = set()
    for i, a in enumerate(shapes):
        for b in shapes[i:]:
            for sizes in ([a, b], [a, b, a]):
                flat = ((ctypes.c_int64 * 3) * len(sizes))(*((ctypes.c_int64 * 3)(*s) for s in sizes))
                kernel, most = index.together(flat, len(sizes), 256), max(s[0] for s in sizes)
                seen.add(kernel)
                assert -1 <= kernel <= 7
                assert kernel not in (0, 1) or most <= 16 * (kernel + 1)
                assert kernel != 2 or most <= 64
    assert seen == {-1, 0, 1, 2, 3, 4, 5, 6, 7}


def test_workgroups_find_their_product(index):
    for counts in ((8, 16, 8), (8, 8), (24,), (8, 8, 800)):
        first = [sum(counts[:i]) for i in range(4)]
        for b in range(sum(counts)):
            which = index.pick(b, first[1], first[2], len(counts))
            assert first[which] <= b < first[which] + counts[which]


def test_rows_stay_inside(index):
    for rows in (1, 2, 31, 256):
        assert [index.row(r, rows) for r in range(256)] == [min(r, rows - 1) for r in range(256)]


def test_chunks_lie_apart(index):
    """A row's eight pieces of 16 bytes trade places; the same piece of eight rows side by side lies in eight places, and so it is for the pieces of the columns' waves."""
    assert all(index.swizzle(r) in range(8) and index.swizzle(r) == index.swizzle(r + 32) for r in range(256))
    for first in range(0, 256, 8):
        for piece in range(8):
            assert len({piece ^ index.swizzle(first + r) for r in range(8)}) == 8
    for waves in (2, 4, 8):
        for octet in range(32):
            assert sorted(index.chunk(w, octet, waves) for w in range(waves)) == list(range(waves))


def loads_of(bm, bn, wm, wn):
    waves = wm * wn
    return (bm + bn) // 8 // waves, -(-(bm // 32) // waves) + -(-(bn // 32) // waves)


@pytest.mark.parametrize("loads,scales", [(12, 6), (8, 3), (4, 2), (1, 1), (9, 4), (8, 2)])
@pytest.mark.parametrize("stages", [2, 3, 4])
def test_a_tile_is_there_when_it_is_read(index, stages, loads, scales):
    """The order in which the loop with steps asks for codes and scales, and how many loads may be on their way at its two waits: a tile is read behind the wait that
    its codes and scales are in front of, from the first tile on."""
    queue, first = [], loads // 2
    queue += [("s", 0)] * scales + [("s", 1)] * scales
    for t in range(stages - 1):
        queue += [("c", t)] * loads + [("s", t + 2)] * scales
    queue += [("c", stages - 1)] * first

    def arrived(in_flight, tile):
        done = queue[:len(queue) - in_flight]
        return done.count(("c", tile)) == loads and done.count(("s", tile)) == scales

    assert arrived(index.behind(stages, loads, scales) + first, 0)
    for kt in range(40):
        queue += [("c", kt + stages - 1)] * (loads - first) + [("s", kt + stages + 1)] * scales
        assert arrived(index.behind(stages, loads, scales), kt + 1)
        queue += [("c", kt + stages)] * first


KERNELS = {"Li32ELi64ELi1ELi2ELi4E": (32, 64, 1, 2, 4), "Li64ELi64ELi2ELi2ELi4E": (64, 64, 2, 2, 4), "Li64ELi128ELi2ELi2ELi4E": (64, 128, 2, 2, 4), "Li128ELi128ELi2ELi2ELi3E": (128, 128, 2, 2, 3),
           "Li128ELi128ELi2ELi2ELi2E": (128, 128, 2, 2, 2), "Li256ELi256ELi2ELi4ELi2E": (256, 256, 2, 4, 2)}


@pytest.fixture(scope="module")
def bodies(tmp_path_factory):
    at = tmp_path_factory.mktemp("mx4_asm")
    return {source: kernel_bodies(source + ".hip", at, "_kernel") for source in ("mx4_gemm", "mx4_quant")}


def test_kernels_keep_out_of_scratch_memory(bodies):
    for name, body in ((n, b) for all_ in bodies.values() for n, b in all_.items()):
        assert re.search(r"\.amdhsa_private_segment_fixed_size 0\b", body), name


def test_the_loops_wait_for_what_they_issue(bodies, index):
    """Each turn of a tile's loop asks for one K tile, straight into LDS, and leaves as many loads on their way as were asked for behind the tile that is read next."""
    found = 0
    for name, body in bodies["mx4_gemm"].items():
        shape = next((v for k, v in KERNELS.items() if k in name), None)
        if shape is None:
            assert "few_rows" in name or "join" in name, name
            continue
        found += 1
        bm, bn, wm, wn, stages = shape
        loads, scales = loads_of(bm, bn, wm, wn)
        whole = bm // wm // 32 * (bn // wn // 32) <= 4
        loop = max((x for x in loops(body) if "v_mfma" in x), key=len)
        assert loop.count("v_mfma") == body.count("v_mfma"), name
        turns = 2 if whole else 1       # (tiles to a turn of the loop)
        issued = re.findall(r"^\s*" + VMEM + r"([^\n]*)", loop, flags=re.M)
        assert len(issued) == turns * (loads + scales) and all("lds" in op for op, _ in issued), (name, len(issued))
        behind = (stages - 2) * (loads + scales) if whole else index.behind(stages, loads, scales)
        waits = [int(v) for v in re.findall(r"s_waitcnt[^\n]*vmcnt\((\d+)\)", loop)]
        assert waits == [behind] * turns, (name, waits, behind)
        assert len(re.findall(r"^\s*s_barrier", loop, flags=re.M)) == turns
        assert "scratch_" not in loop
        # what runs ahead
        ahead = body[:body.index(loop)]
        waits = [int(v) for v in re.findall(r"s_waitcnt[^\n]*vmcnt\((\d+)\)[^\n]*\n(?:\s*;[^\n]*\n|\s*\n)*\s*s_barrier", ahead)]
        assert waits == [(stages - 1) * (loads + scales) if whole else behind + loads // 2], (name, waits)
        asked = re.findall(r"^\s*" + VMEM, ahead, flags=re.M)
        assert len(asked) == (stages * (loads + scales) if whole else (stages + 1) * scales + (stages - 1) * loads + loads // 2) and all("lds" in a for a in asked), name
    assert found == 2 * len(KERNELS)      # (one product to a launch, and several)
