"""A key / value cache in 4 bits, for serving: new tokens into it, attention over it, and a budget that is kept by dropping the
entries that got the least attention (csrc/cache4.hip, csrc/cache4_attention.hip; no counterpart in the reference).

The functions take the cache as the tensors that it consists of: ``pool`` uint8 [pages, kv_heads, page_size * (head_dim + head_dim // 16)] (see
``include/ti8.h`` for a page's layout), a page table int32 [batch, pages of a sequence], lengths int32 [batch] and, where attention is added up,
``weights`` float32 [pages, kv_heads, page_size].  :class:`Cache4` holds them for a batch of sequences.  Lengths, starts and counts are read on the
GPU only, so all of it may be captured into a graph.  There are no gradients: tensors that require one are refused while gradients are recorded, and
so are tensors with a tangent, and tracing.
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _lib, ops
from .ops import _need, _stream

__all__ = ["Cache4", "append", "attention", "evict", "page_bytes", "read"]


def page_bytes(page_size, head_dim):
    """Bytes that a page of one head takes: 4 bits per element of the keys and values and a byte per 32 of them."""
    return page_size * (head_dim + head_dim // 16)


def _on_this_gpu(t):
    return ops._on_gpu(t) and t.get_device() == torch._C._cuda_getDevice()


def _ints(t, name, batch):
    _need(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] == batch and t.is_contiguous() and _on_this_gpu(t),
          f"{name} must be a contiguous int32 tensor [{batch}] on the current GPU")
    return t.data_ptr()


def _table(t, name, batch):
    _need(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] == batch and t.shape[1] > 0 and _on_this_gpu(t)
          and (t.shape[1] == 1 or t.stride(1) == 1) and (batch == 1 or t.stride(0) >= t.shape[1]), f"{name} must be an int32 tensor [{batch}, pages] with dense rows on the current GPU")
    return t.data_ptr(), t.shape[1], t.shape[1] if batch == 1 else t.stride(0)


def _cache(pool, table, weights, head_dim, batch):
    """The C description of a cache."""
    _need(isinstance(pool, torch.Tensor) and pool.dtype == torch.uint8 and pool.dim() == 3 and pool.is_contiguous() and _on_this_gpu(pool),
          "pool must be a contiguous uint8 tensor [pages, kv_heads, bytes of a page] on the current GPU")
    pages, heads, block = pool.shape
    _need(head_dim in (64, 128), f"head_dim must be 64 or 128, got {head_dim}")
    page = block // (head_dim + head_dim // 16)
    _need(page in (16, 32, 64, 128, 256) and block == page_bytes(page, head_dim),
          f"{block} bytes are no page of 16, 32, 64, 128 or 256 entries of head_dim {head_dim}")
    if weights is not None:
        _need(isinstance(weights, torch.Tensor) and weights.dtype == torch.float32 and weights.shape == (pages, heads, page) and weights.is_contiguous()
              and _on_this_gpu(weights), f"weights must be a contiguous float32 tensor {(pages, heads, page)} on the current GPU")
        _no_gradient(weights, "weights")
    at, width, stride = _table(table, "table", batch)
    return _lib.Cache4(pool.data_ptr(), at, None if weights is None else weights.data_ptr(), pages, heads, page, head_dim, batch, width, stride)


def _no_gradient(t, name):
    _need(not (t.requires_grad and torch.is_grad_enabled()), f"{name} requires a gradient, which a cache does not give: call it under torch.no_grad()")
    _need(forward_ad._current_level < 0 or forward_ad.unpack_dual(t).tangent is None, f"{name} has a tangent, which a cache does not carry on")


def _rows(x, name):
    """bf16 [batch, tokens, heads, head_dim] as the kernels read it, and its strides."""
    _need(isinstance(x, torch.Tensor) and x.dtype == torch.bfloat16 and x.dim() == 4 and x.numel() > 0 and _on_this_gpu(x),
          f"{name} must be a non-empty bfloat16 tensor [batch, tokens, heads, head_dim] on the current GPU")
    _no_gradient(x, name)
    B, S, H, _ = x.shape
    sb, ss, sh, one = x.stride()
    sb, ss, sh = 0 if B == 1 else sb, 0 if S == 1 else ss, 0 if H == 1 else sh      # (of a dimension of one a stride means nothing)
    if one != 1 or (sb | ss | sh) & 7 or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        sb, ss, sh, _ = x.stride()
    return x, (sb, ss, sh)


def _natively(name, *args):
    """A call with its checks, allocations and launches made from C++, or None where it takes the Python way, which says what is wrong."""
    native = _lib.native()
    out = None if native is None else getattr(native, name)(*args, _stream())
    if type(out) is tuple:
        raise _lib.failed(*out)
    if out is None:
        ops._unrecorded("a call on a cache")
    return out


def append(pool, table, starts, k, v, counts=None, weights=None):
    """Keys and values of new tokens, bf16 [batch, tokens, kv_heads, head_dim], become entries ``starts[b]``, ``starts[b] + 1``, .. of each sequence;
    of sequence b the first ``counts[b]`` tokens (all of them without ``counts``).  The new entries' ``weights``, if given, become zero."""
    if _natively("cache4_append", pool, table, starts, k, v, counts, weights):
        return
    k, at_k = _rows(k, "k")
    v, at_v = _rows(v, "v")
    B, S, H, D = k.shape
    c = _cache(pool, table, weights, D, B)
    _need(v.shape == k.shape and H == c.kv_heads, f"shapes do not fit: k {tuple(k.shape)}, v {tuple(v.shape)}, {c.kv_heads} kv heads in the pool")
    _lib.call("ti8_cache4_append", c, _ints(starts, "starts", B), None if counts is None else _ints(counts, "counts", B), S,
              k.data_ptr(), *at_k, v.data_ptr(), *at_v, _stream())


def read(pool, table, starts, tokens, head_dim, counts=None):
    """The values that entries ``starts[b]`` .. of each sequence stand for: (keys, values), bf16 [batch, tokens, kv_heads, head_dim], zeros from the
    ``counts[b]``-th on and where the sequence's pages end."""
    made = _natively("cache4_read", pool, table, starts, counts, tokens, head_dim)
    if made is not None:
        return tuple(made)
    _need(isinstance(table, torch.Tensor) and table.dim() == 2 and table.shape[0] > 0, "table must be an int32 tensor [batch, pages]")
    _need(isinstance(tokens, int) and tokens > 0, f"tokens must be a positive number, got {tokens}")
    B = table.shape[0]
    c = _cache(pool, table, None, head_dim, B)
    k, v = (torch.empty((B, tokens, c.kv_heads, head_dim), dtype=torch.bfloat16, device=pool.device) for _ in range(2))
    _lib.call("ti8_cache4_read", c, _ints(starts, "starts", B), None if counts is None else _ints(counts, "counts", B), tokens, k.data_ptr(), v.data_ptr(), _stream())
    return k, v


def attention(pool, table, lengths, q, counts=None, scale=None, weights=None):
    """Attention of q bf16 [batch, tokens, heads, head_dim] over the cache, whose last entries are those of the queries' own tokens: of sequence b the
    first ``counts[b]`` rows are queries (all of them without ``counts``), and query i sees entries up to ``lengths[b] - counts[b] + i``.  ``heads``
    is a multiple of the pool's kv heads; neighbouring heads share one.  ``scale``: 1 / sqrt(head_dim) by default.

    Returns (out bf16 like q, lse float32 [batch, tokens, heads], the logarithms of the sums of the exponentials); rows that see nothing and rows that
    are no queries are zeros with an lse of -inf.  With ``weights``, every entry's probabilities over queries and heads are added to its weight; one whose page
    several sequences name gets those of all of them, in no fixed order (only there may the last bits differ from call to call)."""
    made = _natively("cache4_attention", pool, table, lengths, q, counts, weights, scale)
    if made is not None:
        return tuple(made)
    q, at_q = _rows(q, "q")
    B, S, H, D = q.shape
    c = _cache(pool, table, weights, D, B)
    _need(H % c.kv_heads == 0, f"{H} heads are no multiple of {c.kv_heads} kv heads")
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    _need(abs(scale) <= 2.0 ** 127, f"scale must be a number of up to 2^127 in magnitude, got {scale}")
    lengths = _ints(lengths, "lengths", B)
    counts = None if counts is None else _ints(counts, "counts", B)
    need = _lib.lib().ti8_cache4_attention_workspace(c, S, H)
    _need(need >= 0, f"{B} x {S} tokens of {H} heads over {c.table_pages * c.page_size} entries are more than a call takes")
    dev = q.device
    out, lse = torch.empty((B, S, H, D), dtype=torch.bfloat16, device=dev), torch.empty((B, S, H), dtype=torch.float32, device=dev)
    workspace = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
    _lib.call("ti8_cache4_attention", c, lengths, counts, S, H, q.data_ptr(), *at_q, scale, weights is not None,
              out.data_ptr(), lse.data_ptr(), workspace.data_ptr() if need else None, need, _stream())
    return out, lse


def evict(pool, table, lengths, weights, new_table, *, keep, recent):
    """Every sequence and kv head cut down to ``keep`` entries: the ``recent`` newest and the heaviest of the others by ``weights`` (among equals the
    older one), in their old order, with their weights, in the pages that ``new_table`` int32 [batch, pages] names.  Those must be
    others than the sequences' present ones, which are only read.  Sequences of up to ``keep`` entries move as they are.  Entries of pages that the pool does not
    have are not there: they are left out and do not count.

    Returns (kept int32 [batch, kv_heads, keep], which entry each of them was, -1 behind the last; the new lengths int32 [batch])."""
    made = _natively("cache4_evict", pool, table, lengths, weights, new_table, keep, recent)
    if made is not None:
        return tuple(made)
    _need(isinstance(table, torch.Tensor) and table.dim() == 2 and table.shape[0] > 0, "table must be an int32 tensor [batch, pages]")
    _need(isinstance(weights, torch.Tensor) and weights.dim() == 3 and isinstance(pool, torch.Tensor) and pool.dim() == 3 and weights.shape[2] > 0,
          "weights must be a float32 tensor [pages, kv_heads, page_size]")
    B, page = table.shape[0], weights.shape[2]
    c = _cache(pool, table, weights, pool.shape[2] // page * 16 // 17, B)
    at, width, stride = _table(new_table, "new_table", B)
    _need(isinstance(keep, int) and isinstance(recent, int) and 0 < keep <= width * page and 0 <= recent <= keep,
          f"need 0 <= recent <= keep and 0 < keep <= the {width * page} entries that new_table has room for, got keep={keep} recent={recent}")
    kept = torch.empty((B, c.kv_heads, keep), dtype=torch.int32, device=pool.device)
    new_lengths = torch.empty((B,), dtype=torch.int32, device=pool.device)
    _lib.call("ti8_cache4_evict", c, _ints(lengths, "lengths", B), at, width, stride, keep, recent, kept.data_ptr(), new_lengths.data_ptr(), _stream())
    return kept, new_lengths


class Cache4:
    """The cache of one attention layer for a batch of sequences of up to ``max_length`` entries each.

    ``budget``: the entries that :meth:`evict` cuts sequences down to; the pages for it, and the weights that :meth:`attend` adds up, are there only
    with it.  ``lengths`` int32 [batch] are the entries, ``positions`` int32 [batch] the tokens that went in, dropped ones among them (the next token's
    place in the text)."""

    def __init__(self, batch, max_length, kv_heads, head_dim, *, page_size=64, budget=None, device=None):
        _need(batch > 0 and max_length > 0 and kv_heads > 0, "batch, max_length and kv_heads must be positive")
        _need(head_dim in (64, 128) and page_size in (16, 32, 64, 128, 256), "head_dim must be 64 or 128 and page_size 16, 32, 64, 128 or 256")
        _need(budget is None or 0 < budget <= max_length, f"budget must be between 1 and max_length, got {budget}")
        device = torch.device("cuda") if device is None else torch.device(device)
        mine, spare = -(-max_length // page_size), 0 if budget is None else -(-budget // page_size)
        pages = batch * (mine + spare)
        self.max_length, self.budget, self.head_dim = max_length, budget, head_dim
        self.pool = torch.empty((pages, kv_heads, page_bytes(page_size, head_dim)), dtype=torch.uint8, device=device)
        self.weights = None if budget is None else torch.zeros((pages, kv_heads, page_size), dtype=torch.float32, device=device)
        self.table = torch.arange(batch * mine, dtype=torch.int32, device=device).view(batch, mine)
        self.spare = torch.arange(batch * mine, pages, dtype=torch.int32, device=device).view(batch, spare) if spare else None
        self._counts = torch.zeros((2, batch), dtype=torch.int32, device=device)
        self.lengths, self.positions = self._counts
        # entries and tokens of the longest sequence, as far as the host knows (all tokens of a call counted, replays of a graph not); see look()
        self.filled = self.seen = 0

    def look(self):
        """``filled`` and ``seen`` as the GPU has them, which is waited for."""
        self.filled, self.seen = self._counts.amax(1).tolist()

    def after(self, tokens, counts=None):
        """What ``filled`` and ``seen`` will be behind so many new tokens of every sequence (of sequence b ``counts[b]``), as the GPU has it; while a graph is
        recorded as the host has it."""
        if self.pool.is_cuda and torch.cuda.is_current_stream_capturing():
            return self.filled + tokens, self.seen + tokens
        return (self._counts + (tokens if counts is None else counts.clamp(0, tokens))).amax(1).tolist()

    def append(self, k, v, counts=None):
        """New tokens, bf16 [batch, tokens, kv_heads, head_dim], behind the entries of each sequence (of sequence b the first ``counts[b]``)."""
        tokens = k.shape[1]
        filled, seen = self.filled + tokens, self.seen + tokens
        if filled > self.max_length:        # before a call is refused: sequences may have got fewer tokens than the host counts
            filled, seen = self.after(tokens, counts)
        _need(filled <= self.max_length, f"{tokens} tokens are more than there is room for: a sequence would have {filled} entries of {self.max_length}")
        append(self.pool, self.table, self.lengths, k, v, counts=counts, weights=self.weights)
        self._counts.add_(tokens if counts is None else counts.clamp(0, tokens))        # (as the kernel takes them)
        self.filled, self.seen = filled, seen

    def take_back(self, tokens):
        """The newest tokens out again, as drafted ones that were rejected: so many of every sequence, or int32 [batch]; no more than it has entries.  What they gave
        to other entries' weights stays there."""
        if isinstance(tokens, int):
            self._counts.sub_(self.lengths.clamp(max=max(tokens, 0)))
            return
        _need(isinstance(tokens, torch.Tensor) and tokens.dtype == torch.int32 and tokens.shape == self.lengths.shape and tokens.device == self.lengths.device,
              f"tokens must be a number or an int32 tensor {tuple(self.lengths.shape)} on {self.lengths.device}")
        self._counts.sub_(self.lengths.minimum(tokens.clamp(min=0)))

    def reset(self, sequences=None):
        """All sequences empty again, or those that an index names (numbers, or bool [batch])."""
        if sequences is not None:
            self._counts[:, sequences] = 0
            return
        self._counts.zero_()
        self.filled = self.seen = 0

    def attend(self, q, counts=None, scale=None):
        """Attention of the last appended tokens' queries: see :func:`attention`."""
        return attention(self.pool, self.table, self.lengths, q, counts=counts, scale=scale, weights=self.weights)[0]

    def evict(self, recent):
        """Cut every sequence down to the budget, its ``recent`` newest entries among it; returns what :func:`evict` says was kept."""
        _need(self.budget is not None, "a cache without a budget drops nothing")
        kept, lengths = evict(self.pool, self.table, self.lengths, self.weights, self.spare, keep=self.budget, recent=recent)
        front = self.table[:, :self.spare.shape[1]]
        freed = front.clone()
        front.copy_(self.spare)
        self.spare.copy_(freed)
        self.lengths.copy_(lengths)
        self.filled = min(self.filled, self.budget)
        return kept
