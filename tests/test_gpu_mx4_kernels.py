"""Every kernel of the 4-bit products, alone and several to a launch, whole and in parts, in both types; results lie in larger buffers, of which nothing else is written.

Operands are random codes with scales of a half, one and two: products are multiples of 2^-4, and where the sum of their magnitudes is below 2^20 every partial sum, in any
order, is a number of fp32.  So results are exact, however long the contraction: one tile too few, too many or of another turn shows."""
import pytest
import torch

import mx4_sizes
from conftest import bits_equal, make_gen
from oracle import mx4 as oracle

pytestmark = pytest.mark.gpu
FILL = 7.0


@pytest.fixture(scope="module")
def M(dev):
    import triton_int8_amd
    if torch.cuda.get_device_properties(dev).multi_processor_count != 256:
        pytest.skip("the sizes reach the kernels on 256 compute units")
    return triton_int8_amd.mx4


def codes_of(gen, dev, rows, k):
    """Random codes and scales [rows, k] in 4 bits, zeros behind k."""
    tiles = -(-k // 256)
    codes = torch.randint(0, 256, (rows, tiles * 128), dtype=torch.uint8, generator=gen, device=dev)
    codes[:, (k + 1) // 2:] = 0
    if k % 2:
        codes[:, k // 2] &= 15
    return codes, torch.randint(126, 129, (tiles, rows, 8), dtype=torch.uint8, generator=gen, device=dev)


def sample(rows, most=300):
    """All rows, or those at the ends of tiles and some between."""
    if rows <= most:
        return torch.arange(rows)
    ends = [r for t in range(0, rows + 256, 256) for r in (t - 1, t, t + 31, t + 32, t + 64, t + 128) if 0 <= r < rows] + [rows - 2, rows - 1]
    return torch.tensor(sorted({*ends, *torch.randint(0, rows, (most - 100,), generator=make_gen(rows)).tolist()}))


def equal(got, want, mag):
    assert mag.max() < 2 ** 20
    wrong = got.cpu() != want.to(got.dtype)
    assert not wrong.any(), (int(wrong.sum()), wrong.nonzero()[:4].tolist())


def check(got, a, b, k):
    """[rows of A, rows of B] against the sums, at the sampled rows."""
    at_a, at_b = sample(a[0].shape[0]), sample(b[0].shape[0])
    va, vb = (oracle.values(codes[at.to(codes.device)].cpu(), scales[:, at.to(codes.device)].cpu(), k) for (codes, scales), at in ((a, at_a), (b, at_b)))
    equal(got[at_a.to(got.device)][:, at_b.to(got.device)], *oracle.gemm_nt(va, vb))


class Result:
    """C [batch, M, N] inside a filled buffer, rows and batches further apart than need be."""

    def __init__(self, batch, m, n, wide, dev):
        self.batch, self.m, self.n = batch, m, n
        self.all = torch.full((5 + batch * (m + 2), n + 5), FILL, dtype=torch.float32 if wide else torch.bfloat16, device=dev)
        self.c = self.inside(self.all)
        self.ldc, self.bsc = n + 5, (m + 2) * (n + 5)

    def inside(self, t):
        return t[3:3 + self.batch * (self.m + 2)].view(self.batch, self.m + 2, self.n + 5)[:, :self.m, 2:2 + self.n]

    def alone(self):
        """Nothing around C has been written."""
        around = self.all.clone()
        self.inside(around).fill_(FILL)
        return bool((around == FILL).all())


class Workspace:
    """So many bytes at an address of so many's alignment, with others around them."""

    def __init__(self, need, dev):
        self.need, self.all = need, torch.full((need + 1024,), 0xA5, dtype=torch.uint8, device=dev)
        self.at = self.all.data_ptr() + 512

    def alone(self):
        return bool((self.all[:512] == 0xA5).all() and (self.all[512 + self.need:] == 0xA5).all())


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("wide", [False, True], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape,kernel,parts", mx4_sizes.ALONE, ids=str)
def test_alone(M, dev, shape, kernel, parts, wide):
    batch, m, n, k = shape
    gen = torch.Generator(device=dev).manual_seed(m + n + k)
    a, b = codes_of(gen, dev, batch * m, k), codes_of(gen, dev, batch * n, k)
    da, db = M._operand(*a, "A")[2], M._operand(*b, "B")[2]
    out, lib = Result(batch, m, n, wide, dev), M._lib
    need = lib.lib().ti8_mx4_gemm_nt_workspace(batch, m, n, k)
    assert need == (parts * batch * m * n * 4 if parts > 1 else 0)
    space = Workspace(need, dev)
    lib.call("ti8_mx4_gemm_nt", da, m if batch > 1 else 0, db, n if batch > 1 else 0, out.c.data_ptr(), out.ldc, out.bsc, batch, m, n, k, int(wide), space.at, need, stream())
    assert out.alone() and space.alone()
    for i in range(batch):
        part = lambda t, r: (t[0][i * r:(i + 1) * r], t[1][:, i * r:(i + 1) * r])  # noqa: E731
        check(out.c[i], part(a, m), part(b, n), k)
    whole = lambda t, r: (t[0].view(batch, r, -1) if batch > 1 else t[0], t[1])  # noqa: E731
    got = M.gemm_nt(*whole(a, m), *whole(b, n), out_dtype=torch.float32 if wide else torch.bfloat16)
    assert bits_equal(got.view(batch, m, n), out.c)


@pytest.mark.parametrize("first", [0, 1], ids=["bf16 first", "fp32 first"])
@pytest.mark.parametrize("sizes,kernel", mx4_sizes.TOGETHER + [(s, mx4_sizes.APART) for s in mx4_sizes.TOGETHER_IN_PARTS], ids=str)
def test_together(M, dev, sizes, kernel, first):
    gen = torch.Generator(device=dev).manual_seed(len(sizes) + first)
    lib, problems, kept = M._lib, (M._lib.Mx4GemmProblem * len(sizes))(), []
    for i, (m, n, k) in enumerate(sizes):
        a, b, out = codes_of(gen, dev, m, k), codes_of(gen, dev, n, k), Result(1, m, n, (i + first) % 2, dev)
        problems[i] = lib.Mx4GemmProblem(M._operand(*a, "A")[2], M._operand(*b, "B")[2], out.c.data_ptr(), out.ldc, m, n, k, (i + first) % 2)
        kept.append((a, b, out))
    need = lib.lib().ti8_mx4_gemm_nt_multi_workspace(problems, len(sizes))
    assert (need > 0) == (kernel == mx4_sizes.APART and any(lib.lib().ti8_mx4_gemm_nt_workspace(1, *s) > 0 for s in sizes))
    assert need > 0 or sizes not in mx4_sizes.TOGETHER_IN_PARTS
    space = Workspace(need, dev)
    lib.call("ti8_mx4_gemm_nt_multi", problems, len(sizes), space.at, need, stream())
    made = M.gemm_nt_multi([(*a, *b) for a, b, _ in kept])
    assert space.alone()
    for i, ((a, b, out), (m, n, k)) in enumerate(zip(kept, sizes)):
        assert out.alone(), i
        check(out.c[0], a, b, k)
        assert bits_equal(made[i], out.c[0].bfloat16())     # (rounded once, here or there)


def graphed(T, run, sets):
    """Two graphs of a call, replayed in turn with other inputs and eager work between them."""
    want = [[t.clone() for t in run(*s)] for s in sets]
    steps = [T.GraphedStep(run, *sets[0]) for _ in range(2)]
    for turn in range(4):
        for step in steps:
            got = step(*sets[turn % len(sets)])
            torch.cuda.synchronize()
            assert all(bits_equal(a, b) for a, b in zip(got, want[turn % len(sets)])), turn
            run(*sets[(turn + 1) % len(sets)])


@pytest.mark.parametrize("sizes", mx4_sizes.TOGETHER_IN_PARTS, ids=str)
def test_captured_products_in_parts(M, dev, sizes):
    import triton_int8_amd as T
    gen = torch.Generator(device=dev).manual_seed(1)
    sets = [[t for m, n, k in sizes for t in (*codes_of(gen, dev, m, k), *codes_of(gen, dev, n, k))] for _ in range(2)]
    graphed(T, lambda *t: tuple(M.gemm_nt_multi([t[i:i + 4] for i in range(0, len(t), 4)])), sets)


@pytest.mark.parametrize("shape", [s for s, _, parts in mx4_sizes.ALONE if parts > 1 and s[1] * s[3] < 1 << 23], ids=str)
def test_captured_product_in_parts(M, dev, shape):
    import triton_int8_amd as T
    batch, m, n, k = shape
    gen = torch.Generator(device=dev).manual_seed(2)
    sets = [[*codes_of(gen, dev, batch * m, k), *codes_of(gen, dev, batch * n, k)] for _ in range(2)]
    whole = lambda t, r: t.view(batch, r, -1) if batch > 1 else t  # noqa: E731
    graphed(T, lambda a, sa, b, sb: (M.gemm_nt(whole(a, m), sa, whole(b, n), sb),), sets)


@pytest.mark.parametrize("tokens,k,n", mx4_sizes.STEPS_IN_PARTS + [(1000, 1024, 2560), (100, 300, 200), (1, 1, 1), (2050, 2050, 777)])
def test_steps(M, dev, tokens, k, n):
    """A step's outputs and workspace in larger buffers; those in parts captured, too.  (Numbers that are codes: 4 bits hold them as they are, by rows and by columns.)"""
    import triton_int8_amd as T
    gen, lib = make_gen(tokens), M._lib
    sets = [[(oracle.MAGNITUDES[torch.randint(0, 8, s, generator=gen)] * (1 - 2 * torch.randint(0, 2, s, generator=gen))).bfloat16().to(dev) for s in ((tokens, k), (n, k), (tokens, n))]
            for _ in range(2)]
    x, w, dy = sets[0]
    need = lib.lib().ti8_mx4_linear_fwd_bwd_workspace(tokens, k, n)
    space = Workspace(need, dev)
    outs = [torch.full((r * c + 512,), FILL, dtype=torch.bfloat16, device=dev) for r, c in ((tokens, n), (tokens, k), (n, k))]
    lib.call("ti8_mx4_linear_fwd_bwd", x.data_ptr(), k, w.data_ptr(), k, dy.data_ptr(), n, *(o.data_ptr() + 2 * 255 for o in outs), tokens, k, n, space.at, need, stream())
    assert space.alone() and all(bool((o[:255] == FILL).all() and (o[-257:] == FILL).all()) for o in outs)
    made = M.linear_fwd_bwd(x, w, dy)
    for o, m, (a, b) in zip(outs, made, ((x, w), (dy, w.t()), (dy.t(), x.t()))):
        assert bits_equal(o[255:-257].view(m.shape), m)
        at_a, at_b = sample(a.shape[0], 200), sample(b.shape[0], 200)
        equal(m[at_a.to(dev)][:, at_b.to(dev)], *oracle.gemm_nt(a[at_a.to(dev)].cpu().double(), b[at_b.to(dev)].cpu().double()))
    if (tokens, k, n) in mx4_sizes.STEPS_IN_PARTS:
        graphed(T, M.linear_fwd_bwd, sets)
