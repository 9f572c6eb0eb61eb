"""Tensors in 4 bits with shared scales in plain torch on the CPU: their codes, scales and values, products in float64, and the norm in front of them.

No counterpart in the reference.  Format: ``include/ti8.h``, ti8_mx4."""
import torch

from .cache4 import MAGNITUDES


def quant_row(x):
    """bf16 [rows, cols] -> (codes uint8 [rows, tiles * 128], scales uint8 [tiles, rows, 8])."""
    x = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % 256))
    g = x.unflatten(-1, (-1, 32))
    lost = ~g.isfinite().all(-1, keepdim=True)
    g = torch.where(lost, 0.0, g)
    mantissa, exponent = torch.frexp(g.abs().amax(-1, keepdim=True))        # amax = mantissa 2^exponent, 0.5 <= mantissa < 1
    e = torch.where(mantissa == 0, -126, exponent - 3 + (mantissa > 0.75)).clamp(-126, 125)      # 6 = 0.75 2^3
    g = g.clamp(-1.5 * 2.0 ** 127, 1.5 * 2.0 ** 127)
    away = ((g.abs() / torch.exp2(e.double())).unsqueeze(-1) - MAGNITUDES).abs()
    nearest = away == away.amin(-1, keepdim=True)
    even = nearest & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1, keepdim=True), even, nearest).byte().argmax(-1) + 8 * torch.signbit(g)
    code = code.flatten(-2).byte()
    scale = torch.where(lost, 255, e + 127).squeeze(-1).byte()
    return code[:, 0::2] | (code[:, 1::2] << 4), scale.unflatten(-1, (-1, 8)).transpose(0, 1).contiguous()


def values(codes, scales, cols):
    """float64 [rows, cols]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    v = MAGNITUDES[(c & 7).long()] * torch.where(c >= 8, -1.0, 1.0)
    e = scales.transpose(0, 1).flatten(1)
    s = torch.where(e == 255, float("nan"), torch.exp2(e.double() - 127))
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)[:, :cols]


def rounded(x):
    """The values of bf16 rows in 4 bits, float64."""
    return values(*quant_row(x), x.shape[1])


def gemm_nt(a, b):
    """(A B^T, sum of the magnitudes of the products) of values."""
    return a @ b.transpose(-1, -2), a.abs() @ b.abs().transpose(-1, -2)


def norm(x, weight, eps, residual=None):
    """(y, rstd float64, h): the norm's result before it is quantised."""
    h = x if residual is None else (x.double() + residual.double()).bfloat16()
    rstd = 1.0 / torch.sqrt(h.double().square().mean(-1) + eps)
    n = (h.float() * rstd.float().unsqueeze(-1)).bfloat16()
    return (n.float() * weight.float()).bfloat16(), rstd, h
