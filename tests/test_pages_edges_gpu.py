"""Caches in pages at their edges: without pools, and with every bit of the rows set somewhere."""
import pytest
import torch

from apertura_amd.pages import pages_read, pages_write
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


def _all_bits(b):
    """Every pattern of 16 bits in the pools, signs among them."""
    for pool, first in zip(b.pools, b.first):
        bits = torch.randint(-2 ** 15, 2 ** 15, pool.shape, dtype=torch.int32, device=DEV).to(torch.int16).view(BF)
        pool.copy_(bits)
        first.copy_(bits)
    return b


@pytest.mark.parametrize("order", [(0, 1, 2), (1, 2, 0)])
@pytest.mark.parametrize("pools", POOLS)
@pytest.mark.parametrize("R", [16, 64])
def test_every_bit_of_a_row_moves(pools, R, order):
    b = _all_bits(Both(pools, 50, R, 8, 8, order=order))
    b.call("reserve", [3, 0, 1, 2], [5 * R, 4 * R, R + 5, 2 * R])
    b.set_length([3 * R + 1, R - 2, R, 0, 0, 0, 0, 0])
    b.check()
    b.call("commit", [[0, 1, 4, 9]] * 8, [4, 3, 2, 1, 0, 0, 0, 0])
    b.check()
    b.call("fork", [0, 0, 1, 2], [4, 5, 6, 7], None)
    b.check()
    b.call("free", [0, 2])
    b.call("compact")
    b.check()


@pytest.mark.parametrize("planes,hkv,D,R", [(2, 3, 128, 16), (1, 2, 256, 64), (2, 1, 512, 32)])
def test_every_bit_of_a_row_goes_in_and_out(planes, hkv, D, R):
    n, B = 75, 2
    bits = lambda *shape: torch.randint(-2 ** 15, 2 ** 15, shape, dtype=torch.int32, device=DEV).to(torch.int16)
    most = (n + R - 1) // R + 1
    pool, rows = bits(planes, B * most, hkv, R, D), bits(planes, B, hkv, n, D)
    want = pool.clone()
    table = torch.randperm(B * most, device=DEV).to(torch.int32).view(B, most)
    row0 = torch.tensor([3, R - 1], dtype=torch.int32, device=DEV)
    for b, first in enumerate(row0.tolist()):
        for i in range(n):
            want[:, int(table[b, (first + i) // R]), :, (first + i) % R] = rows[:, b, :, i]
    pages_write(pool.view(BF), table, row0, rows.view(BF))
    assert torch.equal(pool, want)
    assert torch.equal(pages_read(pool.view(BF), table, row0, n).view(torch.int16), rows)
