"""Forked caches on the host: a prefix that is set back and written again is not the one that was shared."""
import pytest
import torch

from qwen3_triton.inference import KVCache


def test_a_prefix_that_was_written_again():
    owner = object()
    k, v = ([torch.zeros((1, 2, 50, 128), dtype=torch.bfloat16) for _ in range(2)] for _ in range(2))
    cache = KVCache(k, v, 50, 1, owner)

    def append(n):   # what a forward does
        cache.admit(owner, 1, n)
        cache.write_from(cache.length)
        cache.length += n
    append(10)
    short = cache.fork(2, 5)
    append(20)
    long = cache.fork(3, 5)
    append(5)
    for forked in (short, long):
        forked.admit(owner, forked.batch_size, 5)
    cache.length = 30    # the shared positions still stand there
    long.admit(owner, 3, 5)
    append(1)
    long.admit(owner, 3, 5)
    cache.length = 29
    with pytest.raises(ValueError, match='no longer'):
        long.admit(owner, 3, 5)
    cache.length = 31    # nothing was written
    long.admit(owner, 3, 5)
    cache.length = 20
    append(1)
    append(14)           # other positions 20 .. 34
    with pytest.raises(ValueError, match='no longer'):
        long.admit(owner, 3, 5)
    long.reset()
    with pytest.raises(ValueError, match='no longer'):
        long.admit(owner, 3, 5)
    short.admit(owner, 2, 5)   # its ten have not been touched
    again = cache.fork(3, 5)
    again.admit(owner, 3, 5)
    cache.length = 12
    append(30)
    with pytest.raises(ValueError, match='no longer'):
        again.admit(owner, 3, 5)
    short.admit(owner, 2, 5)
    cache.length = 9
    append(1)
    with pytest.raises(ValueError, match='no longer'):
        short.admit(owner, 2, 5)
