"""Index arithmetic of the 4-bit cache's kernels (csrc/index_math.h), compiled for the host, at sizes that the entry points take, and what their code holds."""
import ctypes
import os
import re
import subprocess

import pytest

from conftest import ROOT
from test_kernel_resources import kernel_bodies

CODE = r"""
#include <cstdint>
#include "index_math.h"
extern "C" int first_row(int entry, int older, int group) { return ti8::idx::cache4_first_row(entry, older, group); }
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    at = tmp_path_factory.mktemp("cache4_index")
    (at / "index.cpp").write_text(CODE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "triton-int8_amd", "csrc"), "-o", str(at / "index.so"), str(at / "index.cpp")], check=True)
    return ctypes.CDLL(str(at / "index.so"))


@pytest.mark.parametrize("group,length,count", [
    (1, 5, 2), (4, 700, 40), (128, (1 << 24) + 1000, 1), (128, (1 << 30), 70), (4096, (1 << 19) + 70000, 1), (4096, 1 << 20, 3), (4096, 1 << 30, 1 << 18), (7, 3, 9)])
def test_first_row_that_sees_an_entry(index, group, length, count):
    """Every row sees the entries in front of the tokens' own, however many there are; of the others those from their own token on."""
    older = length - count
    entries = sorted({e for e in (0, 1, length // 3, older - 1, older, older + 1, older + count // 2, length - 1, length + 30) if 0 <= e})
    for entry in entries:
        assert index.first_row(entry, older, group) == max(entry - older, 0) * group


def test_weights_are_added_to_and_never_stored(tmp_path):
    """Two sequences may name a page: nothing between a weight's load and its store gets lost if it is neither loaded nor stored."""
    bodies = kernel_bodies("cache4_attention.hip", tmp_path, "weights_kernel")
    assert len(bodies) == 2
    for name, body in bodies.items():
        assert re.search(r"^\s*global_atomic_add_f32 ", body, flags=re.M) and not re.search(r"^\s*(global|buffer|flat)_store", body, flags=re.M), name


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 3e38, -2e38])
def test_scales_that_are_refused(scale):
    """With one that is no number all entries would get the same, without a word."""
    import triton_int8_amd
    lib, fake = triton_int8_amd._lib, 0x10000
    cache = lib.Cache4(pool=fake, table=fake, weights=fake, pages=8, kv_heads=2, page_size=64, head_dim=128, batch=3, table_pages=4, table_stride=4)
    assert lib.lib().ti8_cache4_attention(cache, fake, None, 5, 8, fake, 2048, 256, 128, scale, 0, fake, fake, fake, 1 << 40, None) == 2
    assert b"scale" in lib.lib().ti8_last_error()
