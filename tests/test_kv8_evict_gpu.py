"""Eviction from the 8-bit cache where the other tests of it do not go."""
import pytest
import torch

from test_kv8_gpu import DEV, I8, I32, i32, random_cache, same, to_gpu
from open_ommx_serve_b200 import _lib, ommx_kv8_evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,status_wanted", [(100, 0), (-1, _lib.ST_BAD_LENGTH)])
def test_the_largest_list_of_kept_places(n, status_wanted):
    """Its last indexes lie next to 2^31; a sequence of fewer tokens keeps all, and what is behind its list is -1."""
    budget = 2 ** 31 - 1
    cache = random_cache(2, 1, 64, 64, I8)
    gpu, status = to_gpu(cache), i32([0])
    kept, len_out = torch.full((1, 1, budget), 7, dtype=I32, device=DEV), i32([1])
    ommx_kv8_evict(gpu["codes"], gpu["scales"], gpu["weight"], i32([[0, 1]]), i32([n]), kept, recent_tokens=budget, len_out=len_out, status=status)
    assert int(status) == status_wanted and len_out.tolist() == [n]
    held = max(n, 0)
    assert kept[0, 0, :held].tolist() == list(range(held))
    for part in kept[0, 0, held:].split(1 << 28):
        assert bool((part == -1).all())
    for name in cache:
        assert same(gpu[name], cache[name]), name
