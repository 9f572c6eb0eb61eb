"""Quantisers, their inverses and the norm write into larger buffers, rows and tiles further apart than need be: the bits of the public calls, and nothing around them."""
import ctypes

import pytest
import torch

from conftest import bits_equal, make_gen, randn_bf16
from test_gpu_mx4 import tensor

pytestmark = pytest.mark.gpu
FILL = 0xA5


@pytest.fixture(scope="module")
def T():
    import triton_int8_amd
    return triton_int8_amd


class Room:
    """[rows][cols] of a type inside a filled buffer: `apart` more elements between rows, `ahead` in front."""

    def __init__(self, dev, rows, cols, dtype=torch.uint8, apart=0, ahead=512):
        self.size = torch.empty((), dtype=dtype).element_size()
        self.rows, self.cols, self.ld, self.ahead = rows, cols, cols + apart, ahead
        self.all = torch.full(((ahead + rows * self.ld + 512) * self.size,), FILL, dtype=torch.uint8, device=dev)
        self.t = self.inside(self.all).view(dtype) if self.size == 1 else self.all.view(dtype)[ahead:ahead + rows * self.ld].view(rows, self.ld)[:, :cols]
        self.at = self.all.data_ptr() + ahead * self.size

    def inside(self, flat):
        row = self.ld * self.size
        return flat[self.ahead * self.size:][:self.rows * row].view(self.rows, row)[:, :self.cols * self.size]

    def alone(self):
        around = self.all.clone()
        self.inside(around).fill_(FILL)
        return bool((around == FILL).all())


class Mx4Room:
    """A tensor in 4 bits with room between its rows of codes and its tiles of scales."""

    def __init__(self, T, dev, rows, cols):
        self.tiles = -(-cols // 256)
        self.codes, self.scales = Room(dev, rows, self.tiles * 128, apart=48), Room(dev, self.tiles, rows * 8, apart=24)
        self.c = T._lib.Mx4(self.codes.at, self.scales.at, self.codes.ld, self.scales.ld)

    def is_just(self, codes, scales):
        return (torch.equal(self.codes.t, codes.reshape(self.codes.t.shape)) and torch.equal(self.scales.t, scales.reshape(self.tiles, -1)) and self.codes.alone() and self.scales.alone())


def stream():
    return torch.cuda.current_stream().cuda_stream


SIZES = [(1, 1), (2, 31), (33, 255), (64, 512), (65, 777), (255, 24), (257, 40), (300, 1000), (1001, 1016), (1, 5000), (5000, 1), (6185, 5641)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("ways", ["rows", "columns", "both"])
def test_quantisers(T, dev, rows, cols, ways):
    x = tensor(make_gen(rows + cols), rows, cols).to(dev)
    apart = torch.full((rows, cols + 3), float("nan"), dtype=torch.bfloat16, device=dev)     # (what lies between the rows of x is not read)
    apart[:, :cols] = x
    by_rows, by_columns = Mx4Room(T, dev, rows, cols), Mx4Room(T, dev, cols, rows)
    nothing = T._lib.Mx4()
    operand = T._lib.Mx4Operand(apart.data_ptr(), cols + 3, rows, cols, nothing if ways == "columns" else by_rows.c, nothing if ways == "rows" else by_columns.c)
    T._lib.call("ti8_mx4_quant", operand, 1, stream())
    if ways != "columns":
        assert by_rows.is_just(*T.mx4.quant_row(x))
        y = Room(dev, rows, cols, torch.bfloat16, apart=5, ahead=513)
        T._lib.call("ti8_mx4_dequant", by_rows.c, rows, cols, y.at, y.ld, stream())
        assert bits_equal(y.t, T.mx4.dequant(*T.mx4.quant_row(x), cols)) and y.alone()
    if ways != "rows":
        assert by_columns.is_just(*T.mx4.quant_col_t(x))


@pytest.mark.parametrize("sizes", [[(33, 255), (300, 1000)], [(1001, 1016), (2, 31), (257, 40)], [(6185, 3641), (5, 7), (2050, 4100)]], ids=str)
def test_several_operands(T, dev, sizes):
    xs = [tensor(make_gen(i), r, c).to(dev) for i, (r, c) in enumerate(sizes)]
    rooms = [(Mx4Room(T, dev, r, c), Mx4Room(T, dev, c, r)) for r, c in sizes]
    operands = (T._lib.Mx4Operand * len(sizes))(*(T._lib.Mx4Operand(x.data_ptr(), c, r, c, a.c, b.c) for x, (r, c), (a, b) in zip(xs, sizes, rooms)))
    T._lib.call("ti8_mx4_quant", operands, len(sizes), stream())
    for x, (a, b) in zip(xs, rooms):
        assert a.is_just(*T.mx4.quant_row(x)) and b.is_just(*T.mx4.quant_col_t(x))


@pytest.mark.parametrize("rows,dim", [(1, 8), (3, 264), (5, 512), (7, 520), (4, 1024), (2, 1032), (9, 2048), (3, 4104), (33, 4096), (2, 8200), (2, 16384)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("to", ["mx4", "row", "group"])
def test_norm(T, dev, rows, dim, residual, to):
    if to != "mx4" and dim % 128:
        dim = -(-dim // 128) * 128
    gen = make_gen(rows + dim)
    x, r, w = randn_bf16(gen, rows, dim).to(dev), randn_bf16(gen, rows, dim).to(dev), randn_bf16(gen, dim).to(dev)
    groups = dim // 128 if to == "group" else 1
    h, rstd, q, s = Room(dev, rows, dim, torch.bfloat16, apart=8), Room(dev, 1, rows, torch.float32), Room(dev, rows, dim, torch.int8, apart=8), Room(dev, rows, groups, torch.float32)
    mx = Mx4Room(T, dev, rows, dim)
    a = T._lib.RmsnormQuantArgs(x=x.data_ptr(), ldx=dim, w=w.data_ptr(), rstd=rstd.at, rows=rows, dim=dim, eps=1e-5, group=128 if to == "group" else 0, inv_mode=T.ops.INV_RCP_OF_SCALE)
    if residual:
        a.residual, a.ldr, a.h, a.ldh = r.data_ptr(), dim, h.at, h.ld
    if to == "mx4":
        a.mx4 = mx.c
    else:
        a.q, a.ldq, a.s, a.qflags = q.at, q.ld, s.at, T.ops.Q_CLAMP
    T._lib.call("ti8_rmsnorm_quant", ctypes.byref(a), stream())
    want = T.ops.rmsnorm_quant(x, w, 1e-5, residual=r if residual else None, to="mx4" if to == "mx4" else "int8", group=128 if to == "group" else 0)
    assert torch.equal(rstd.t[0], want[2]) and rstd.alone()
    assert h.alone() and (not residual or bits_equal(h.t, want[3]))
    if to == "mx4":
        assert mx.is_just(*want[:2])
    else:
        assert torch.equal(q.t, want[0]) and torch.equal(s.t, want[1].view(rows, groups)) and q.alone() and s.alone()
        y = Room(dev, rows, dim, torch.bfloat16, apart=8)
        T._lib.call("ti8_dequant_row", q.at, q.ld, s.at, rows, dim, 128 if to == "group" else 0, y.at, y.ld, stream())
        assert bits_equal(y.t, T.ops.dequant_row(*want[:2])) and y.alone()
