"""4-bit tensors, their products and the norm at sizes whose offsets pass 32 bits: what lies at the ends is what a call for that part alone gives."""
import pytest
import torch

from conftest import bits_equal, make_gen
from oracle import mx4 as oracle
from test_gpu_mx4 import close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import triton_int8_amd
    return triton_int8_amd


def normal(dev, rows, cols, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev)
    for part in x.split(1 << 17):
        part.normal_(generator=gen)
    return x


def test_quantisers(T, dev):
    rows, cols = (1 << 20) + 300, 4100          # 8.6 GB
    x = normal(dev, rows, cols)
    q, s, qt, st = T.mx4.quant_row_col_t(x)
    for at in (0, rows - 70):
        part, scales = T.mx4.quant_row(x[at:at + 70])
        assert bits_equal(q[at:at + 70], part) and bits_equal(s[:, at:at + 70], scales)
        assert bits_equal(T.mx4.dequant(q, s, cols)[at:at + 70], T.mx4.dequant(part, scales, cols))
    at = rows // 256 * 256 - 256
    part, scales = T.mx4.quant_col_t(x[at:])
    assert bits_equal(qt[:, at // 2:], part) and bits_equal(st[at // 256:], scales)
    del q, s, qt, st
    q, s = T.mx4.quant_row(x)
    part, scales = T.mx4.quant_row(x[-70:])
    assert bits_equal(q[-70:], part) and bits_equal(s[:, -70:], scales)


@pytest.mark.parametrize("m,n,k", [(70001, 40003, 32), ((1 << 22) + 77, 9, 2048), (9, (1 << 22) + 77, 2048)], ids=["result", "A", "B"])
def test_products(T, dev, m, n, k):
    """Results, or codes of an operand, of more than 2^32 bytes."""
    a, b = normal(dev, m, k), normal(dev, n, k, seed=1)
    rows, cols = (torch.tensor(sorted({0, 1, size // 2, size - 2, size - 1})) for size in (m, n))
    got = T.mx4.gemm_nt(*T.mx4.quant_row(a), *T.mx4.quant_row(b))
    want, mag = oracle.gemm_nt(oracle.rounded(a[rows.to(dev)].cpu()), oracle.rounded(b[cols.to(dev)].cpu()))
    close(got[rows.to(dev)][:, cols.to(dev)], want, mag, k)


@pytest.mark.parametrize("to", ["mx4", "int8"])
def test_norm(T, dev, to):
    rows, dim = (1 << 20) + 3, 4224
    x, r = normal(dev, rows, dim), normal(dev, rows, dim, seed=1)
    w = torch.rand(dim, generator=make_gen(2)).bfloat16().to(dev)
    q, s, rstd, h = T.ops.rmsnorm_quant(x, w, 1e-5, residual=r, to=to)
    for at in (0, rows // 2, rows - 5):
        part = slice(at, at + 5)
        p, t, u, v = T.ops.rmsnorm_quant(x[part], w, 1e-5, residual=r[part], to=to)
        assert bits_equal(q[part], p) and bits_equal(s[:, part] if to == "mx4" else s[part], t) and bits_equal(rstd[part], u) and bits_equal(h[part], v)
    if to == "int8":
        y = T.ops.dequant_row(q, s)
        assert bits_equal(y[-5:], T.ops.dequant_row(q[-5:], s[-5:]))
