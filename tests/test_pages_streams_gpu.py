"""A cache in pages beside streams: on another one than it was made on, behind what fills its tensors, and
its memory kept until that stream is through."""
import pytest
import torch

from apertura_amd._lib import EsdaError
from apertura_amd.pages import PagedCache

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
DEV = "cuda"


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _dirty():
    """Free memory of the allocator's holds a pattern that no cache starts with."""
    held = [torch.full((n,), 0x55, dtype=torch.uint8, device=DEV) for n in (1 << 15, 1 << 16, 1 << 17) for _ in range(16)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("given", [True, False])
def test_a_first_call_on_another_stream_waits_for_the_cache(given):
    """The workspace (and references that are counted) are filled on the stream the cache is made on."""
    pool = torch.randn((2, 8, 1, 16, 128), device=DEV).to(BF)
    want = pool.clone()
    table, length = _ints([[0, 1], [2, 3]]), _ints([10, 4])
    accept, count = _ints([[1, 3], [0, 5]]), _ints([2, 2])
    side = torch.cuda.Stream()
    _dirty()
    torch.cuda._sleep(20_000_000)
    cache = PagedCache([pool], table, length)
    if given:
        cache.commit(accept, count, stream=side)
        cache.reserve(_on_side(side, [1]), _on_side(side, [32]), stream=side)
    else:
        with torch.cuda.stream(side):
            cache.commit(accept, count)
            cache.reserve(_ints([1]), _ints([32]))
    torch.cuda.synchronize()
    for p, n, path in ((0, 10, [1, 3]), (2, 4, [0, 5])):
        for i, a in enumerate(path):
            want[:, p, :, n + i] = pool.new_tensor(0) + want[:, p, :, n + a]
    assert length.tolist() == [12, 6] and cache.left_out() == 0
    assert torch.equal(pool, want)
    assert table.tolist() == [[0, 1], [2, 3]] and cache.refs.tolist() == [1, 1, 1, 1, 0, 0, 0, 0]


def _on_side(side, x):
    with torch.cuda.stream(side):
        return _ints(x)


@pytest.mark.parametrize("given", [True, False])
def test_a_cache_s_memory_outlives_its_calls(given):
    """A cache dropped with work under way on another stream: its memory is not handed out before that is done."""
    pool = torch.zeros((1, 8, 1, 16, 128), dtype=BF, device=DEV)
    cache = PagedCache.empty([pool], 4, 2)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    held = {t.data_ptr(): t.numel() * t.element_size() for t in (cache.workspace, cache.table, cache.length, cache.refs)}
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        if not given:
            cache.compact()
    if given:
        cache.compact(stream=side)
    del cache
    again = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in held.values()]
    assert not set(held) & {t.data_ptr() for t in again}
    torch.cuda.synchronize()


def test_a_capture_on_a_stream_of_its_own():
    """The first call of a cache recorded into a graph, on the capture's stream."""
    pool = torch.randn((1, 8, 1, 16, 128), device=DEV).to(BF)
    table, length = torch.full((3, 2), -1, dtype=torch.int32, device=DEV), _ints([0, 0, 0])
    slots, rows = _ints([0, 2]), _ints([20, 5])
    cache = PagedCache([pool], table, length)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.free(slots)
        cache.reserve(slots, rows)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert table.tolist() == [[0, 1], [-1, -1], [2, -1]] and cache.refs.tolist() == [1, 1, 1, 0, 0, 0, 0, 0]
        cache.reserve(_ints([1]), _ints([1]))
        cache.free(_ints([1]))
        assert cache.left_out() == 0


def test_left_out_is_not_captured():
    """The count is read at once: a capture refuses it, and goes on."""
    pool = torch.randn((1, 8, 1, 16, 128), device=DEV).to(BF)
    cache = PagedCache.empty([pool], 3, 2)
    slots, rows = _ints([0, 9]), _ints([20, 20])
    cache.reserve(slots, rows)
    assert cache.left_out() == 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.free(slots)
        with pytest.raises(EsdaError) as refused:
            cache.left_out()
        cache.reserve(slots, rows)
    assert refused.value.code == 1 and "captured" in str(refused.value)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert cache.table.tolist() == [[0, 1], [-1, -1], [-1, -1]]
        assert cache.left_out() == 2 and cache.left_out() == 0
