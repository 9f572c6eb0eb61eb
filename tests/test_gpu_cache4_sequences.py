"""Cache4 and DecoderLayer.serve on sequences that grow by different numbers of tokens."""
import math

import pytest
import torch

from oracle import cache4 as oracle
from test_gpu_cache4 import C, _check_attention, _ints  # noqa: F401

pytestmark = pytest.mark.gpu


def test_counts_of_more_and_less_than_the_tokens(C, dev):
    """What counts of no sense add is what was written: no entry becomes visible that nobody wrote, and no sequence gets shorter."""
    gen = torch.Generator().manual_seed(1)
    cache = C.Cache4(3, 64, 2, 64, page_size=16, device=dev)
    cache.pool.fill_(255)         # scales that are no numbers
    k, v = (torch.randn(3, 12, 2, 64, generator=gen).bfloat16() for _ in range(2))
    q = torch.randn(3, 5, 2, 64, generator=gen).bfloat16()
    cache.append(k[:, :7].to(dev), v[:, :7].to(dev))
    cache.append(k[:, 7:].to(dev), v[:, 7:].to(dev), counts=_ints([40, -3, 2], dev))
    assert cache.lengths.tolist() == cache.positions.tolist() == [12, 7, 9]
    out, lse = C.attention(cache.pool, cache.table, cache.lengths, q.to(dev), counts=_ints([40, -3, 2], dev))
    want = oracle.attention(cache.pool.cpu(), cache.table.cpu(), [12, 7, 9], q, [5, 0, 2], 1 / math.sqrt(64), 16)
    assert bool(torch.isfinite(out).all())
    _check_attention(out, lse, want, 64, 12)
