"""Linear layers in 4-bit floating point with shared scales (csrc/mx4_quant.hip, csrc/mx4_gemm.hip; no counterpart in the reference).

A tensor in 4 bits is a pair: ``codes`` uint8 [.., rows, tiles * 128] and ``scales`` uint8 [tiles, all rows, 8], tiles = ceil(columns / 256).  Two codes
to a byte (the format of the 4-bit cache: magnitudes 0 .5 1 1.5 2 3 4 6 and a sign); 32 neighbours along the contraction share a power of two, the smallest
by which the largest of them is at most 6.  ``include/ti8.h`` has it to the bit.  Groups with an infinity or a NaN stand for NaN.

The functions take bf16 tensors on the current GPU, enqueue on torch's current stream and may be captured into a graph.  They give no gradients:
:class:`Mx4Linear` does, with every product of forward and backward in 4 bits.
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .ops import _natively, _need, _no_tangent, _stream, _unrecorded

__all__ = ["Mx4Linear", "Mx4LinearFunction", "dequant", "gemm_nt", "gemm_nt_multi", "linear_fwd_bwd", "linears", "quant_col_t", "quant_row", "quant_row_col_t"]

TILE = 256                  # elements of a row that take 128 bytes of codes and 8 scales
MOST_ROWS = 1 << 28
MOST_CONTRACTED = 1 << 22


def _tiles(cols):
    return -(-cols // TILE)


def _here(t):
    return ops._on_gpu(t) and t.get_device() == torch._C._cuda_getDevice()


def _bf16(x, name, dim=None):
    _unrecorded("a call in 4 bits")
    _need(isinstance(x, torch.Tensor) and x.dtype == torch.bfloat16 and _here(x), f"{name} must be a bfloat16 tensor on the current GPU")
    _need(x.dim() >= 1 and x.numel() > 0 and dim in (None, x.dim()), f"{name} must be a non-empty tensor" + ("" if dim is None else f" of {dim} dimensions"))
    _no_tangent(x, name)


def _empty(rows, cols, device, lead=None):
    """Room for a tensor in 4 bits, and its C description."""
    tiles = _tiles(cols)
    codes = torch.empty((*((rows,) if lead is None else lead), tiles * 128), dtype=torch.uint8, device=device)
    scales = torch.empty((tiles, rows, 8), dtype=torch.uint8, device=device)
    return codes, scales, _lib.Mx4(codes.data_ptr(), scales.data_ptr(), tiles * 128, rows * 8)


def _quant(x, by_rows, by_columns):
    """x [R, C] with dense rows or dense columns."""
    if x.stride(1) != 1 and x.shape[1] > 1:
        if x.stride(0) == 1 and x.stride(1) >= x.shape[0]:      # the transpose of a tensor with dense rows: its columns are rows there
            made = _quant(x.t(), by_columns, by_rows)
            return made[1], made[0]
        x = x.contiguous()
    R, C = x.shape
    ldx = C if R == 1 else x.stride(0)
    if ldx < C:         # rows that overlap, as those of a tensor that is expanded over them
        x = x.clone(memory_format=torch.contiguous_format)
        ldx = C
    _need(max(R, C) <= MOST_ROWS, f"a tensor in 4 bits has up to 2^28 rows and columns, got {R} x {C}")
    rows = _empty(R, C, x.device) if by_rows else None
    cols = _empty(C, R, x.device) if by_columns else None
    nothing = _lib.Mx4()
    _lib.call("ti8_mx4_quant", _lib.Mx4Operand(x.data_ptr(), ldx, R, C, nothing if rows is None else rows[2], nothing if cols is None else cols[2]), 1, _stream())
    return None if rows is None else rows[:2], None if cols is None else cols[:2]


def quant_row(x):
    """``x`` bf16 [.., cols] in 4 bits, groups along the last dim: ``(codes, scales)``."""
    made = _natively("mx4_quant", x, 1, 0)
    if made is not None:
        return tuple(made)
    _bf16(x, "x")
    codes, scales = _quant(x.reshape(-1, x.shape[-1]), True, False)[0]
    return codes.view(*x.shape[:-1], codes.shape[-1]), scales


def quant_col_t(x):
    """The transpose of ``x`` [R, C] in 4 bits, groups along its columns: ``quant_row(x.T)`` without the transpose in bf16."""
    made = _natively("mx4_quant", x, 0, 1)
    if made is not None:
        return tuple(made)
    _bf16(x, "x", 2)
    return _quant(x, False, True)[1]


def quant_row_col_t(x):
    """``(codes, scales)`` of ``x`` [R, C] and of its transpose from one read: the same bits as :func:`quant_row` and :func:`quant_col_t`."""
    made = _natively("mx4_quant", x, 1, 1)
    if made is not None:
        return tuple(made)
    _bf16(x, "x", 2)
    rows, cols = _quant(x, True, True)
    return *rows, *cols


def _operand(codes, scales, name):
    """Codes [rows, bytes] or [batch, rows, bytes] with their scales as the kernels read them: (codes, scales, C description)."""
    _unrecorded("a call in 4 bits")
    _need(isinstance(codes, torch.Tensor) and codes.dtype == torch.uint8 and codes.dim() in (2, 3) and codes.numel() > 0 and codes.shape[-1] % 128 == 0 and _here(codes),
          f"codes of {name} must be a uint8 tensor [rows, tiles * 128] or [batch, rows, tiles * 128] on the current GPU")
    tiles, rows = codes.shape[-1] // 128, codes.shape[:-1].numel()
    _need(isinstance(scales, torch.Tensor) and scales.dtype == torch.uint8 and scales.shape == (tiles, rows, 8) and _here(scales),
          f"scales of {name} must be a uint8 tensor {(tiles, rows, 8)} on the current GPU")
    if codes.dim() == 3 or codes.stride(1) != 1 or codes.data_ptr() % 16 or (rows > 1 and (codes.stride(0) % 16 or codes.stride(0) < codes.shape[1])):
        if not codes.is_contiguous() or codes.data_ptr() % 16:
            codes = codes.clone(memory_format=torch.contiguous_format)
    ld = codes.shape[-1] if codes.dim() == 3 or rows == 1 else codes.stride(0)
    if scales.stride(2) != 1 or (rows > 1 and scales.stride(1) != 8) or scales.data_ptr() % 8 or (tiles > 1 and (scales.stride(0) % 8 or scales.stride(0) < rows * 8)):
        scales = scales.clone(memory_format=torch.contiguous_format)
    return codes, scales, _lib.Mx4(codes.data_ptr(), scales.data_ptr(), ld, rows * 8 if tiles == 1 else scales.stride(0))


def dequant(codes, scales, cols):
    """The values, bf16 [.., cols], that codes [.., tiles * 128] and scales stand for (exact)."""
    y = _natively("mx4_dequant", codes, scales, cols)
    if y is not None:
        return y
    _unrecorded("a call in 4 bits")
    _need(isinstance(codes, torch.Tensor) and codes.dim() >= 1 and codes.numel() > 0, "codes must be a non-empty uint8 tensor [.., tiles * 128]")
    _need(isinstance(cols, int) and cols > 0 and codes.shape[-1] == _tiles(cols) * 128, f"{cols} columns have {_tiles(cols) * 128 if isinstance(cols, int) else '?'} bytes of codes, got {codes.shape[-1]}")
    flat = codes.reshape(-1, codes.shape[-1])
    flat, scales, q = _operand(flat, scales, "the tensor")
    _need(flat.shape[0] <= MOST_ROWS, "a tensor in 4 bits has up to 2^28 rows")
    y = torch.empty((*codes.shape[:-1], cols), dtype=torch.bfloat16, device=codes.device)
    _lib.call("ti8_mx4_dequant", q, flat.shape[0], cols, y.data_ptr(), cols, _stream())
    return y


def gemm_nt(A, sA, B, sB, out_dtype=torch.bfloat16):
    """``A B^T`` of tensors in 4 bits: A [M, ..] or [batch, M, ..], B [N, ..] (that all batches share) or [batch, N, ..]; bf16 or float32, [M, N] or [batch, M, N].
    Added up in fp32 in a fixed order and rounded once."""
    wide = out_dtype is torch.float32
    if wide or out_dtype is torch.bfloat16:
        out = _natively("mx4_gemm_nt", A, sA, B, sB, 1 if wide else 0)
        if out is not None:
            return out
    _need(out_dtype in (torch.bfloat16, torch.float32), f"out_dtype must be bfloat16 or float32, got {out_dtype}")
    A, sA, a = _operand(A, sA, "A")
    B, sB, b = _operand(B, sB, "B")
    _need(A.shape[-1] == B.shape[-1], f"A has {A.shape[-1] // 128} tiles along the contraction, B {B.shape[-1] // 128}")
    _need(B.dim() == 2 or (A.dim() == 3 and A.shape[0] == B.shape[0]), f"batches do not fit: A {tuple(A.shape)}, B {tuple(B.shape)}")
    M, N, batch, K = A.shape[-2], B.shape[-2], 1 if A.dim() == 2 else A.shape[0], A.shape[-1] * 2
    _need(max(M, N) <= MOST_ROWS and K <= MOST_CONTRACTED, f"a product takes up to 2^28 rows and contracts up to 2^22 elements, got {M}, {N} and {K}")
    out = torch.empty((M, N) if A.dim() == 2 else (batch, M, N), dtype=out_dtype, device=A.device)
    rows_a, rows_b = M, N if B.dim() == 3 else 0
    if rows_b == 0:         # one weight for all batches: their rows are rows of one product
        M, batch = M * batch, 1
    _need(batch <= 65535 and M <= MOST_ROWS, f"a product takes up to 65535 batches and 2^28 rows, got {batch} and {M}")
    need = _lib.lib().ti8_mx4_gemm_nt_workspace(batch, M, N, K)
    workspace = torch.empty((need,), dtype=torch.uint8, device=A.device) if need > 0 else None
    _lib.call("ti8_mx4_gemm_nt", a, rows_a if batch > 1 else 0, b, rows_b if batch > 1 else 0, out.data_ptr(), N, M * N, batch, M, N, K, int(wide),
              None if workspace is None else workspace.data_ptr(), need, _stream())
    return out


def gemm_nt_multi(problems):
    """Up to three products ``(A, sA, B, sB)`` of matrices, in one launch where that is faster: a list of bf16 matrices.  What :func:`gemm_nt` gives, but for the order
    in which contractions are added up."""
    _need(1 <= len(problems) <= 3, f"between 1 and 3 products, got {len(problems)}")
    for p in problems:
        _need(len(p) == 4, "a product is (codes of A, scales of A, codes of B, scales of B)")
    made = _natively("mx4_gemm_nt_multi", *[t for p in problems for t in p])
    if made is not None:
        return made
    descs, outs, keep = (_lib.Mx4GemmProblem * len(problems))(), [], []
    for i, (A, sA, B, sB) in enumerate(problems):
        A, sA, a = _operand(A, sA, "A")
        B, sB, b = _operand(B, sB, "B")
        _need(A.dim() == B.dim() == 2 and A.shape[1] == B.shape[1], f"need matrices of as many tiles along the contraction, got codes {tuple(A.shape)} and {tuple(B.shape)}")
        M, N, K = A.shape[0], B.shape[0], A.shape[1] * 2
        _need(max(M, N) <= MOST_ROWS and K <= MOST_CONTRACTED, f"a product takes up to 2^28 rows and contracts up to 2^22 elements, got {M}, {N} and {K}")
        outs.append(torch.empty((M, N), dtype=torch.bfloat16, device=A.device))
        descs[i] = _lib.Mx4GemmProblem(a, b, outs[-1].data_ptr(), N, M, N, K, 0)
        keep.append((A, sA, B, sB))     # (copies stay alive until the launch is queued)
    need = _lib.lib().ti8_mx4_gemm_nt_multi_workspace(descs, len(problems))
    workspace = torch.empty((need,), dtype=torch.uint8, device=outs[0].device) if need > 0 else None
    _lib.call("ti8_mx4_gemm_nt_multi", descs, len(problems), None if workspace is None else workspace.data_ptr(), need, _stream())
    return outs


def _fit(X2, W, dY2=None):
    _need(W.dim() == 2 and X2.shape[1] == W.shape[1] and (dY2 is None or tuple(dY2.shape) == (X2.shape[0], W.shape[0])),
          f"shapes do not fit: X {tuple(X2.shape)}, W {tuple(W.shape)}" + ("" if dY2 is None else f", dY {tuple(dY2.shape)}"))


def _dense_rows(x):
    """x itself where its rows are dense and do not overlap, else a copy."""
    return x if (x.stride(1) == 1 or x.shape[1] == 1) and x.stride(0) >= x.shape[1] else x.clone(memory_format=torch.contiguous_format)


def linear_fwd_bwd(X, W, dY):
    """One forward and backward of a layer, every product in 4 bits: ``(Y, dX, dW)`` for X bf16 [.., K], W bf16 [N, K] and dY bf16 [.., N].  The operands of
    dX = dY W are in 4 bits along N, those of dW = dY^T X along the tokens."""
    made = _natively("mx4_linear_fwd_bwd", X, W, dY)
    if made is not None:
        return tuple(made)
    K, N = X.shape[-1], W.shape[0]
    X2, dY2 = X.reshape(-1, K), dY.reshape(-1, N)
    _fit(X2, W, dY2)
    if X2.shape[0] == 0:    # nothing to multiply: empty Y and dX, a zero weight gradient (as torch.nn.functional.linear gives)
        return X.new_empty((*X.shape[:-1], N)), torch.empty_like(X), torch.zeros_like(W)
    for t, name in ((X2, "X"), (W, "W"), (dY2, "dY")):
        _bf16(t, name)
    X2, W, dY2 = (_dense_rows(t) for t in (X2, W, dY2))
    T, dev = X2.shape[0], X2.device
    need = _lib.lib().ti8_mx4_linear_fwd_bwd_workspace(T, K, N)
    _need(need >= 0, f"a step takes up to 2^22 tokens and features, got {T}, {K} and {N}")
    Y, dX, dW = (torch.empty(shape, dtype=torch.bfloat16, device=dev) for shape in ((T, N), (T, K), (N, K)))
    workspace = ops._workspace(need, dev)
    _lib.call("ti8_mx4_linear_fwd_bwd", X2.data_ptr(), X2.stride(0), W.data_ptr(), W.stride(0), dY2.data_ptr(), dY2.stride(0), Y.data_ptr(), dX.data_ptr(), dW.data_ptr(), T, K, N,
              workspace.data_ptr(), need, _stream())
    return Y.view(*X.shape[:-1], N), dX.view(X.shape), dW


def _column_sum(x):
    """``x.sum(0)`` of a bf16 matrix of any width, added up in fp32."""
    cols = x.shape[1]
    return ops.column_sum(x if cols % 32 == 0 else torch.nn.functional.pad(x, (0, -cols % 32)))[:cols]


def _products(codes, scales, views, shape):
    """Outputs [*shape, features] for an input in 4 bits and the forward's views of several weights: three to a launch."""
    ys = [y for i in range(0, len(views), 3) for y in gemm_nt_multi([(codes, scales, *v) for v in views[i:i + 3]])]
    return tuple(ys) if len(shape) == 1 else tuple(y.view(*shape, y.shape[1]) for y in ys)


class Mx4LinearFunction(torch.autograd.Function):
    """The products of one x with several weights, each ``x W^T`` with all of its operands, and those of its gradients, in 4 bits; x is quantised once.
    The backward reads what the forward quantised: neither x nor the weights are kept."""

    @staticmethod
    def forward(ctx, x, *weights):
        x2 = x.reshape(-1, x.shape[-1])
        for w in weights:
            _bf16(w, "weight", 2)
            _fit(x2, w)
        ctx.shape, ctx.features = x.shape, [w.shape[0] for w in weights]
        ctx.set_materialize_grads(False)
        if x2.shape[0] == 0:
            return tuple(x.new_empty((*x.shape[:-1], n)) for n in ctx.features)
        _bf16(x, "x")
        kept, views = [], []
        if any(ctx.needs_input_grad[1:]):
            xq, xs, *kept = quant_row_col_t(x2)
        else:
            xq, xs = quant_row(x2)
        for w in weights:
            if ctx.needs_input_grad[0]:
                q, s, *transposed = quant_row_col_t(w)
                kept += transposed
            else:
                q, s = quant_row(w)
            views.append((q, s))
        ctx.save_for_backward(*kept)
        return _products(xq, xs, views, x.shape[:-1])

    @staticmethod
    @once_differentiable
    def backward(ctx, *dys):
        wants_x, wants = ctx.needs_input_grad[0], ctx.needs_input_grad[1:]
        kept = ctx.saved_tensors
        K, tokens = ctx.shape[-1], ctx.shape[:-1].numel()
        x, of_weights = kept[:2 * any(wants)], kept[2 * any(wants):]
        dx, dws = None, [None] * len(dys)
        # the last layer's part first, as autograd adds up those of separate calls
        for i in reversed(range(len(dys))):
            if dys[i] is None or not (wants_x or wants[i]):     # (an output that nobody uses: its weight has no gradient)
                continue
            if tokens == 0:
                dx, dws[i] = dys[i].new_empty((0, K)), dys[i].new_zeros((ctx.features[i], K)) if wants[i] else None
                continue
            _no_tangent(dys[i], "a gradient")
            d = dys[i].reshape(tokens, ctx.features[i])
            made = _natively("mx4_quant", d, int(wants_x), int(wants[i]))
            rows, cols = _quant(d, wants_x, wants[i]) if made is None else (made[:2], made[-2:])
            made = gemm_nt_multi(([(*rows, *of_weights[2 * i:2 * i + 2])] if wants_x else []) + ([(*cols, *x)] if wants[i] else []))
            if wants_x:
                dx = made[0] if dx is None else dx.add_(made[0])
            if wants[i]:
                dws[i] = made[-1]
        return (dx.view(ctx.shape) if wants_x and dx is not None else None, *dws)


class _BiasFunction(torch.autograd.Function):
    """y + bias, with the bias's gradient added up in fp32 by launches that a graph may hold."""

    @staticmethod
    def forward(ctx, y, bias):
        return y + bias

    @staticmethod
    @once_differentiable
    def backward(ctx, d):
        d2 = d.reshape(-1, d.shape[-1])
        db = None
        if ctx.needs_input_grad[1]:
            _no_tangent(d, "a gradient")
            # (a sum with a bias of another type has that type: not for the kernel)
            db = d2.new_zeros(d2.shape[1:]) if d2.shape[0] == 0 else _column_sum(d2) if d2.dtype == torch.bfloat16 else d2.sum(0)
        return d, db


def _with_bias(y, bias):
    """y + bias, also where the bias alone has a gradient."""
    return y if bias is None else _BiasFunction.apply(y, bias) if bias.requires_grad and torch.is_grad_enabled() else y + bias


def _served(codes, scales, shape, layers):
    """Outputs [*shape, out_features] of layers whose input is already in 4 bits."""
    ys = _products(codes, scales, [m.quantised() for m in layers], shape)
    biases = [m.bias for m in layers]       # (a module's attributes take a while)
    return tuple(map(_with_bias, ys, biases))


def linears(x, layers):
    """The outputs of several :class:`Mx4Linear` for the same x, which is quantised once, three products to a launch."""
    for m in layers:
        _need(x.shape[-1] == m.in_features, f"expected {m.in_features} input features, got {x.shape[-1]}")
    if forward_ad._current_level >= 0:
        for t in (x, *(t for m in layers for t in (m.weight, m.bias) if t is not None)):
            _need(forward_ad.unpack_dual(t).tangent is None, "a tensor with a tangent, which a layer in 4 bits does not carry on")
    if torch.is_grad_enabled() and (x.requires_grad or any(not m.packed and m.weight.requires_grad for m in layers)):
        _need(not any(m.packed for m in layers), "a packed layer serves the forward only: call it under torch.no_grad()")
        ys = Mx4LinearFunction.apply(x, *(m.weight for m in layers))
        return tuple(y if m.bias is None else _BiasFunction.apply(y, m.bias) for y, m in zip(ys, layers))
    if x.numel() == 0:
        return tuple(_with_bias(x.new_empty((*x.shape[:-1], m.out_features)), m.bias) for m in layers)
    return _served(*quant_row(x if x.dim() == 2 else x.reshape(-1, x.shape[-1])), x.shape[:-1], layers)


def _as_written(modules, cls, call):
    """Whether calls of these modules do just what their class does: no hooks, nothing replaced."""
    for m in modules:
        if type(m) is not cls:
            return False
    if torch.nn.modules.module._has_any_global_hook() or (cls.forward, cls.__call__, cls._call_impl) != call:
        return False
    for m in modules:
        own = m.__dict__
        if "forward" in own or "_call_impl" in own or m._compiled_call_impl is not None:
            return False
        if m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks:
            return False
    return True


class Mx4Linear(torch.nn.Module):
    """``torch.nn.Linear`` whose three products (Y, dX, dW) run in 4 bits.  Any number of features and tokens.

    A layer that only serves is packed (:meth:`pack`): it then keeps its weight in 4 bits, 17/32 of a byte per element, and gives the bf16 one up."""

    def __init__(self, in_features, out_features, bias=False, device=None, dtype=torch.bfloat16):
        super().__init__()
        _need(in_features > 0 and out_features > 0, "in_features and out_features must be positive")
        self.in_features, self.out_features = in_features, out_features
        self.weight = torch.nn.Parameter(torch.empty(out_features, in_features, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype)) if bias else None
        self.register_buffer("codes", None)
        self.register_buffer("scales", None)
        torch.nn.init.normal_(self.weight, std=0.02)

    @property
    def packed(self):
        return self.codes is not None

    @torch.no_grad()
    def pack(self):
        """The weight in 4 bits from here on, for the forward alone; returns the layer."""
        if not self.packed:
            self.codes, self.scales = quant_row(self.weight)
            self.weight = None
        return self

    def quantised(self):
        """The forward's view of the weight, ``(codes, scales)``: the packed one, or one made now."""
        codes = self.codes
        return quant_row(self.weight.detach()) if codes is None else (codes, self.scales)

    def forward(self, x):
        return linears(x, (self,))[0]

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, packed={self.packed}"


# the module's call, to be told from one that replaces part of it
_CALL = (Mx4Linear.forward, Mx4Linear.__call__, Mx4Linear._call_impl)


def all_as_written(layers):
    """Whether modules are :class:`Mx4Linear` whose calls do just what that does: then several may be one call."""
    return _as_written(layers, Mx4Linear, _CALL)
