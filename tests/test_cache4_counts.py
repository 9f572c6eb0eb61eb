"""What Cache4 knows of its sequences on the host, without a GPU: the launches are left out, the counts are those of the GPU."""
import pytest
import torch


@pytest.fixture
def C(monkeypatch):
    import triton_int8_amd as T
    monkeypatch.setattr(T.cache4, "append", lambda *args, **more: None)
    return T.cache4


def _cache(C, **more):
    return C.Cache4(3, 20, 2, 64, page_size=16, device="cpu", **more)


def _new(cache, tokens, counts=None):
    kv = torch.zeros(3, tokens, 2, 64, dtype=torch.bfloat16)
    cache.append(kv, kv, counts=None if counts is None else torch.tensor(counts, dtype=torch.int32))


def test_a_cache_refuses_what_has_no_room_and_nothing_else(C):
    """Sequences that got fewer tokens than a call has: the host's own numbers run ahead of them, and a call that has room is taken."""
    cache = _cache(C)
    for i in range(8):          # five drafted tokens at a time, of which one, two and none are new
        _new(cache, 5, [1, 2, 0])
    assert cache.lengths.tolist() == cache.positions.tolist() == [8, 16, 0]
    _new(cache, 5, [5, 4, 0])
    assert (cache.filled, cache.seen) == (20, 20) and cache.lengths.tolist() == [13, 20, 0]
    with pytest.raises(ValueError, match="room"):
        _new(cache, 5, [0, 1, 0])
    with pytest.raises(ValueError, match="room"):
        _new(cache, 1)
    assert cache.lengths.tolist() == [13, 20, 0]
    _new(cache, 7, [7, 0, 9])
    assert cache.lengths.tolist() == [20, 20, 7]
    cache.reset()
    _new(cache, 20)
    assert cache.lengths.tolist() == [20] * 3
    with pytest.raises(ValueError, match="room"):
        _new(cache, 1)


def test_the_host_can_look(C):
    cache = _cache(C)
    _new(cache, 6, [1, 0, 2])
    assert (cache.filled, cache.seen) == (6, 6)
    assert cache.after(6) == [8, 8] and cache.after(3, torch.tensor([3, 0, -1], dtype=torch.int32)) == [4, 4]
    cache.look()
    assert (cache.filled, cache.seen) == (2, 2)
    cache.lengths.fill_(1)      # as an eviction does
    cache.look()
    assert (cache.filled, cache.seen) == (1, 2)


def test_tokens_are_taken_back(C):
    cache = _cache(C)
    _new(cache, 8, [8, 2, 0])
    cache.take_back(1)
    assert cache.lengths.tolist() == cache.positions.tolist() == [7, 1, 0]
    cache.take_back(torch.tensor([3, 5, -2], dtype=torch.int32))
    assert cache.lengths.tolist() == cache.positions.tolist() == [4, 0, 0]
    cache.positions.add_(10)        # entries that an eviction dropped
    cache.take_back(9)
    assert cache.lengths.tolist() == [0, 0, 0] and cache.positions.tolist() == [10, 10, 10]
    for tokens in (1.0, torch.tensor([1, 1]), torch.tensor([1, 1, 1]), [1, 1, 1]):
        with pytest.raises(ValueError, match="tokens"):
            cache.take_back(tokens)
    _new(cache, 20)
    assert (cache.filled, cache.seen) == (20, 30)


@pytest.mark.parametrize("index", [1, [1], torch.tensor([False, True, False]), slice(1, 2)], ids=str)
def test_some_sequences_begin_again(C, index):
    cache = _cache(C)
    _new(cache, 20)
    cache.reset(index)
    assert cache.lengths.tolist() == cache.positions.tolist() == [20, 0, 20]
    _new(cache, 20, [0, 20, 0])
    assert cache.lengths.tolist() == [20, 20, 20]
