"""Caches in pages at their edges: without pools, and with every bit of the rows set somewhere."""
import pytest
import torch

from test_pages_gpu import POOLS, Both

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
DEV = "cuda"


def test_a_cache_without_pools():
    """Tables, references and lengths as with pools; no row moves."""
    b = Both(POOLS[1], 30, 16, 6, 5)
    b.cache._cache.num_pools = 0
    b.call("reserve", [0, 1, 4], [37, 16, 5])
    b.set_length([37, 16, 0, 0, 5, 0])
    b.call("reserve", [0, 1], [64, 64])
    b.call("fork", [0, 0, 1], [2, 3, 5], [20, 37, 16])
    b.call("commit", [[0, 2, 9]] * 6, [3, 2, 0, 0, 0, 0])
    b.call("free", [2])
    b.call("compact")
    b.model.rows = {place: place for place in b.model.rows}  # (the model moved them)
    b.check()
