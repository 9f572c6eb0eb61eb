"""The 4-bit cache without a GPU: what the entry points refuse, how the entries are shared out, where they lie, and what the kernels' code holds."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from conftest import ROOT
from oracle import cache4 as oracle
from test_kernel_resources import VMEM, kernel_bodies, kernel_resources, loops

CSRC = os.path.join(ROOT, "triton-int8_amd", "csrc")
FAKE = 0x10000      # a 16-byte aligned "device pointer"; validation never dereferences it


@pytest.fixture(scope="module")
def lib():
    import triton_int8_amd
    return triton_int8_amd._lib


def _cache(lib, **other):
    fields = dict(pool=FAKE, table=FAKE, weights=FAKE, pages=8, kv_heads=2, page_size=64, head_dim=128, batch=3, table_pages=4, table_stride=4)
    return lib.Cache4(**{**fields, **other})


CACHES = [
    (dict(pool=None), 1, "required"), (dict(table=None), 1, "required"), (dict(head_dim=96), 2, "head_dim"), (dict(page_size=48), 2, "page_size"),
    (dict(page_size=8), 2, "page_size"), (dict(page_size=512), 2, "page_size"), (dict(batch=0), 2, "batch"), (dict(batch=65536), 2, "batch"),
    (dict(kv_heads=0), 2, "kv_heads"), (dict(pages=0), 2, "pages"), (dict(pages=1 << 31), 2, "pages"), (dict(table_pages=0), 2, "table_pages"),
    (dict(table_pages=1 << 25, table_stride=1 << 25), 2, "table_pages"), (dict(table_stride=3), 2, "table_stride"), (dict(pool=FAKE + 8), 3, "aligned"),
    (dict(table=FAKE + 2), 3, "4-byte"), (dict(weights=FAKE + 1), 3, "4-byte"),
]


@pytest.mark.parametrize("other,code,msg", CACHES, ids=str)
@pytest.mark.parametrize("entry", ["append", "read", "attention", "evict"])
def test_caches_that_are_refused(lib, entry, other, code, msg):
    c, l = _cache(lib, **other), lib.lib()
    rows = FAKE, 2048, 256, 128
    rc = {"append": lambda: l.ti8_cache4_append(c, FAKE, None, 5, *rows, *rows, None),
          "read": lambda: l.ti8_cache4_read(c, FAKE, None, 5, FAKE, FAKE, None),
          "attention": lambda: l.ti8_cache4_attention(c, FAKE, None, 5, 8, *rows, 1.0, 0, FAKE, FAKE, FAKE, 1 << 40, None),
          "evict": lambda: l.ti8_cache4_evict(c, FAKE, FAKE, 4, 4, 100, 10, FAKE, FAKE, None)}[entry]()
    assert rc == code and msg in l.ti8_last_error().decode() and f"ti8_cache4_{entry}" in l.ti8_last_error().decode()


ROWS = (FAKE, 2048, 256, 128)


@pytest.mark.parametrize("name,args,code,msg", [
    ("append", (None, None, 5, *ROWS, *ROWS, None), 1, "starts"), ("append", (FAKE, None, 0, *ROWS, *ROWS, None), 2, "tokens"),
    ("append", (FAKE, None, 1 << 31, *ROWS, *ROWS, None), 2, "tokens"), ("append", (FAKE, None, 5, None, 0, 0, 0, *ROWS, None), 1, "k is required"),
    ("append", (FAKE, None, 5, *ROWS, FAKE + 2, 0, 0, 0, None), 3, "v must be"), ("append", (FAKE, None, 5, FAKE, 4, 0, 0, *ROWS, None), 3, "multiples of 8"),
    ("read", (FAKE, None, 5, FAKE, None, None), 1, "v is required"), ("read", (FAKE, None, 5, FAKE + 4, FAKE, None), 3, "aligned"),
    ("read", (None, None, 5, FAKE, FAKE, None), 1, "starts"),
    ("attention", (FAKE, None, 0, 8, *ROWS, 1.0, 0, FAKE, FAKE, FAKE, 1 << 40, None), 2, "tokens"),
    ("attention", (FAKE, None, 5, 7, *ROWS, 1.0, 0, FAKE, FAKE, FAKE, 1 << 40, None), 2, "multiple of kv_heads"),
    ("attention", (FAKE, None, 1 << 24, 64, *ROWS, 1.0, 0, FAKE, FAKE, FAKE, 1 << 40, None), 2, "launch"),
    ("attention", (None, None, 5, 8, *ROWS, 1.0, 0, FAKE, FAKE, FAKE, 1 << 40, None), 1, "lengths"),
    ("attention", (FAKE, None, 5, 8, *ROWS, 1.0, 0, None, FAKE, FAKE, 1 << 40, None), 1, "out"),
    ("attention", (FAKE, None, 5, 8, *ROWS, 1.0, 0, FAKE, FAKE, None, 1 << 40, None), 1, "workspace"),
    ("attention", (FAKE, None, 5, 8, *ROWS, 1.0, 0, FAKE, FAKE, FAKE, 100, None), 2, "bytes of workspace"),
    ("attention", (FAKE, None, 5, 8, FAKE, 2044, 256, 128, 1.0, 0, FAKE, FAKE, FAKE, 1 << 40, None), 3, "multiples of 8"),
    ("attention", (FAKE, None, 5, 8, *ROWS, 1.0, 0, FAKE + 8, FAKE, FAKE, 1 << 40, None), 3, "aligned"),
    ("attention", (FAKE, None, 100, 8, FAKE, 8, 1 << 26, 128, 1.0, 1, FAKE, FAKE, FAKE, 1 << 40, None), 2, "stride"),
    ("attention", (FAKE, None, 100, 8, FAKE, 8, 128, 1 << 29, 1.0, 1, FAKE, FAKE, FAKE, 1 << 40, None), 2, "stride"),
    ("evict", (None, FAKE, 4, 4, 100, 10, FAKE, FAKE, None), 1, "lengths"), ("evict", (FAKE, FAKE, 4, 4, 0, 0, FAKE, FAKE, None), 2, "keep"),
    ("evict", (FAKE, FAKE, 4, 4, 257, 0, FAKE, FAKE, None), 2, "keep"), ("evict", (FAKE, FAKE, 4, 4, 100, 101, FAKE, FAKE, None), 2, "recent"),
    ("evict", (FAKE, FAKE, 4, 3, 100, 10, FAKE, FAKE, None), 2, "new_stride"), ("evict", (FAKE, FAKE, 4, 4, 100, 10, None, FAKE, None), 1, "kept"),
])
def test_arguments_that_are_refused(lib, name, args, code, msg):
    l = lib.lib()
    assert getattr(l, "ti8_cache4_" + name)(_cache(lib, table_pages=64, table_stride=64), *args) == code
    assert msg in l.ti8_last_error().decode(), l.ti8_last_error()


def test_weights_are_required_where_they_are_used(lib):
    l, c = lib.lib(), _cache(lib, weights=None)
    assert l.ti8_cache4_attention(c, FAKE, None, 5, 8, *ROWS, 1.0, 1, FAKE, FAKE, FAKE, 1 << 40, None) == 1
    assert l.ti8_cache4_evict(c, FAKE, FAKE, 4, 4, 100, 10, FAKE, FAKE, None) == 1


def test_workspace_sizes(lib):
    size = lambda tokens, heads, **o: lib.lib().ti8_cache4_attention_workspace(_cache(lib, **o), tokens, heads)
    assert size(1, 8, table_pages=64, table_stride=64) > 0 and size(1, 8) == 0          # (short sequences have a workgroup each)
    assert size(1, 7) == -1 and size(0, 8) == -1 and size(1, 8, head_dim=80) == -1
    assert size(1 << 24, 64) == -1          # more rows than a launch takes
    assert size(1, 2, batch=65535, table_pages=1 << 18, table_stride=1 << 18) == -1


def test_the_oracle_rounds_to_the_nearest_code():
    """Against a search over all codes and, for the scale, over all exponents."""
    gen = torch.Generator().manual_seed(0)
    x = (torch.randn(400, 32, generator=gen) * torch.exp(4 * torch.randn(400, 1, generator=gen))).bfloat16()
    x[0], x[1, 1:], x[2] = 0.0, 0.0, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4)
    codes, scales = oracle.encode(x)
    value = oracle.decode(codes, scales)
    every = torch.cat((oracle.MAGNITUDES, -oracle.MAGNITUDES))
    for row, s, v in zip(x.double(), scales[:, 0], value):
        unit, top = 2.0 ** (int(s) - 127), float(row.abs().max())
        assert top <= 6 * unit and (top > 3 * unit or int(s) == 1)
        assert torch.equal((row - v).abs(), (row[:, None] - every * unit).abs().amin(1))
    assert value[2].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0] * 4          # halfway: the even code


# ---- how the kernels find their places -----------------------------------------------------------------------------

WALK = r"""
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>
#include "index_math.h"
using namespace ti8::idx;
extern "C" int walk_share(int units, int groups, char* msg) {
    const Share s = share_out(units, groups);
    if (s.groups > groups || s.groups > units || s.groups < 1) { sprintf(msg, "%d workgroups of %d for %d units", s.groups, groups, units); return 1; }
    int at = 0;
    for (int w = 0; w < s.groups; ++w) {
        const int begin = share_begin(s, w), end = share_begin(s, w + 1);
        if (begin != at || end <= begin || end - begin > units / s.groups + 1) { sprintf(msg, "workgroup %d has %d to %d", w, begin, end); return 1; }
        for (int u = begin; u < end; ++u)
            if (share_of(s, u) != w) { sprintf(msg, "unit %d is %d's, not %d's", u, w, share_of(s, u)); return 1; }
        at = end;
    }
    if (at != units) { sprintf(msg, "%d of %d units", at, units); return 1; }
    return 0;
}
// step_kernel's walk over its share and join_kernel's search for the parts: every unit of every head once, a head that nobody has whole in parts that
// are found again, in places that nobody else writes
extern "C" int walk_step(const int* lengths, int batch, int heads, int most, int extra, char* msg) {
    std::vector<int> per(batch), before(batch + 1, 0);
    for (int b = 0; b < batch; ++b) {
        per[b] = cache4_units(lengths[b], CACHE4_UNIT);
        before[b + 1] = before[b] + (per[b] + extra) * heads;
    }
    const Share s = share_out(before[batch], most);
    std::vector<std::vector<int>> done(batch * heads);
    for (int i = 0; i < batch * heads; ++i) done[i].assign(per[i / heads], 0);
    std::vector<int> part(2 * s.groups, -1), whole(batch * heads, 0);
    for (int w = 0; w < s.groups; ++w) {
        const int begin = share_begin(s, w), end = share_begin(s, w + 1);
        int b = 0;
        while (before[b + 1] <= begin) ++b;
        const int in = (begin - before[b]) % (per[b] + extra);
        int h = (begin - before[b]) / (per[b] + extra), unit = imax(in - extra, 0);
        for (int left = end - begin - imax(extra - in, 0); left > 0;) {
            if (b >= batch || h >= heads) { sprintf(msg, "workgroup %d goes on to sequence %d head %d", w, b, h); return 1; }
            const int n = imin(left, per[b] - unit), pair = b * heads + h;
            for (int u = unit; u < unit + n; ++u) ++done[pair][u];
            if (n == per[b]) ++whole[pair];
            else {
                int& slot = part[2 * w + (unit == 0)];
                if (slot >= 0) { sprintf(msg, "workgroup %d writes a part twice", w); return 1; }
                slot = pair;
            }
            left -= n + extra;
            unit = 0;
            if (++h == heads && left > 0) { h = 0; ++b; }
        }
    }
    for (int pair = 0; pair < batch * heads; ++pair) {
        for (size_t u = 0; u < done[pair].size(); ++u)
            if (done[pair][u] != 1) { sprintf(msg, "unit %zu of pair %d is done %d times", u, pair, done[pair][u]); return 1; }
        const int b = pair / heads, begin = before[b] + pair % heads * (per[b] + extra) + extra;
        const int first = share_of(s, begin), last = share_of(s, begin + per[b] - 1);
        if ((first == last) != (whole[pair] == 1)) { sprintf(msg, "pair %d: whole %d, workgroups %d to %d", pair, whole[pair], first, last); return 1; }
        for (int w = first; w <= last && first != last; ++w) {
            int& slot = part[2 * w + (w == first)];
            if (slot != pair) { sprintf(msg, "pair %d finds workgroup %d's part of pair %d", pair, w, slot); return 1; }
            slot = -1;
        }
    }
    for (size_t i = 0; i < part.size(); ++i)
        if (part[i] >= 0) { sprintf(msg, "the part %zu of pair %d is nobody's", i, part[i]); return 1; }
    return 0;
}
extern "C" int walk_place(int pairs, int blocks, char* msg) {
    const int64_t grid = round8(pairs) * blocks;
    std::vector<int> seen((size_t)round8(pairs) * blocks, 0);
    for (int64_t w = 0; w < grid; ++w) {
        const AttentionPlace p = cache4_place((uint32_t)w, pairs, blocks);
        if (p.pair < 0 || p.pair >= round8(pairs) || p.block < 0 || p.block >= blocks || p.pair % 8 != w % 8) { sprintf(msg, "workgroup %lld: pair %d block %d", (long long)w, p.pair, p.block); return 1; }
        if (seen[(size_t)p.pair * blocks + p.block]++) { sprintf(msg, "pair %d block %d twice", p.pair, p.block); return 1; }
    }
    return 0;
}
// bytes of a page: every entry's codes and scales in places of their own, all of the page used
extern "C" int walk_page(int page, int dim, char* msg) {
    std::vector<char> used(cache4_block_bytes(page, dim), 0);
    if (1 << log2_of(page) != page) { sprintf(msg, "log2 of %d", page); return 1; }
    for (int row = 0; row < page; ++row)
        for (int values = 0; values < 2; ++values) {
            const int at[2] = {cache4_codes(page, dim, values, row), cache4_scales(page, dim, values, row)}, bytes[2] = {dim / 2, dim / 32};
            for (int i = 0; i < 2; ++i) {
                if (at[i] % bytes[i]) { sprintf(msg, "row %d is misaligned", row); return 1; }
                for (int x = 0; x < bytes[i]; ++x)
                    if (at[i] + x >= (int)used.size() || used[at[i] + x]++) { sprintf(msg, "byte %d of row %d", at[i] + x, row); return 1; }
            }
        }
    for (char u : used)
        if (!u) { sprintf(msg, "unused bytes"); return 1; }
    return 0;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    at = tmp_path_factory.mktemp("cache4")
    (at / "walk.cpp").write_text(WALK)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", str(at / "walk.so"), str(at / "walk.cpp")], check=True)
    so, msg = ctypes.CDLL(str(at / "walk.so")), ctypes.create_string_buffer(512)

    def run(name, *args):
        assert getattr(so, name)(*args, msg) == 0, msg.value
    return run


def test_units_are_shared_out(walk):
    for units in (1, 2, 7, 255, 256, 257, 768, 769, 5000, 99991):
        for groups in (1, 2, 3, 255, 256, 512, 768, 1024):
            walk("walk_share", units, groups)


def test_every_unit_is_done_once_and_every_part_found(walk):
    extra = int(re.search(r"constexpr int EXTRA = (\d+);", open(os.path.join(CSRC, "cache4_attention.hip")).read()).group(1))
    gen = torch.Generator().manual_seed(0)
    for batch in (1, 2, 5, 63, 64, 65, 130, 200):
        for top in (1, 128, 129, 3000, 70000):
            lengths = [int(x) for x in torch.randint(0, top + 1, (batch,), generator=gen)]
            for heads in (1, 3, 8):
                for most in (1, 100, 512, 768):
                    walk("walk_step", (ctypes.c_int * batch)(*lengths), batch, heads, most, extra)
    walk("walk_step", (ctypes.c_int * 16)(*([0] * 16)), 16, 32, 768, extra)


def test_row_blocks_are_placed_once(walk):
    for pairs in (1, 7, 8, 9, 16, 100):
        for blocks in (1, 2, 5, 64):
            walk("walk_place", pairs, blocks)


def test_pages_are_used_up(walk):
    for page in (16, 32, 64, 128, 256):
        for dim in (64, 128):
            walk("walk_page", page, dim)


# ---- the kernels' code ----------------------------------------------------------------------------------------------

def test_kernels_do_not_spill(tmp_path):
    for source, most in (("cache4.hip", 128), ("cache4_attention.hip", 256)):
        kernels = kernel_resources(source, tmp_path)
        assert len(kernels) >= 7
        for name, v in kernels.items():
            assert v["private_segment_fixed_size"] == 0 and v["next_free_vgpr"] <= most, (name, v)
    step = {k: v["next_free_vgpr"] for k, v in kernels.items() if "step_kernel" in k}
    assert all(n <= 168 for k, n in step.items() if re.search("ILi(64|128)ELi1ELb0E", k)), step          # three workgroups per CU
    assert all(n <= 128 for k, n in step.items() if "ILi64ELi1ELb1E" in k) and len(step) == 8, step      # two of eight waves
    assert all(v["next_free_vgpr"] <= 128 for k, v in kernels.items() if "weights_kernel" in k)       # two of eight waves


def test_weights_kernel_waits_for_what_it_issues(tmp_path):
    """The walk over many rows waits with vmcnt(n) for its own tile while the next one's n loads may be in flight: it has to issue exactly n loads between
    two waits, all of them to LDS, and nothing else.  Behind the walk everything is waited for, so that no load lands in the LDS of another workgroup."""
    for name, body in kernel_bodies("cache4_attention.hip", tmp_path, "weights_kernel").items():
        per_tile = 3 if "ILi128E" in name else 2
        walks = [loop for loop in loops(body) if re.search(rf"s_waitcnt vmcnt\({per_tile}\) lgkmcnt\(0\)\s*\n(?:\s*;[^\n]*\n|\s*\n)*\s*s_barrier", loop)]
        assert walks, name
        inner = min(walks, key=len)
        issued = re.findall(r"^\s*" + VMEM + r"([^\n]*)", inner, flags=re.M)
        assert len(issued) == per_tile and all("_lds_" in op or rest.rstrip().endswith("lds") for op, rest in issued), (name, issued)
        assert len(re.findall(r"vmcnt\(", inner)) == 1, name         # nothing else in the walk waits for loads
        behind = body[body.index(inner) + len(inner):]
        assert re.search(r"s_waitcnt vmcnt\(0\)", behind), name
