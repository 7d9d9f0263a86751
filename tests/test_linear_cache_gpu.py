"""Steps of drafted tokens over linear caches, one after another, their accepted rows committed by
LinearCache: against 64 bits over rows that the test keeps itself."""
import random

import pytest
import torch

from _attn64 import attend64, check
from apertura_amd.tree import LinearCache, TreeCall, TreeStep, tree_decode
from test_tree_gpu import paths_of, random_parents

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
DEV = "cuda"


def _rows(shape, g):
    x = torch.randn(shape, device=DEV, generator=g)
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(BF)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("captured", [False, True])
def test_steps_and_their_commits(captured):
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    rng = random.Random(3)
    B, T, cap = 3, 9, 170
    heads = [(8, 2, 128, 2), (4, 1, 512, 1)]  # query heads, kv heads, dims, planes (1: K = V)
    start = [100, 0, 33]
    # (planes within sequences in memory: a stride between the sequences of a plane)
    caches = [torch.full((B, planes, hkv, cap, D), float("nan"), dtype=BF, device=DEV).transpose(0, 1) for _, hkv, D, planes in heads]
    rows = [[[_rows((hkv, n, D), g) for n in start] for _ in range(planes)] for _, hkv, D, planes in heads]
    for x, of in zip(caches, rows):
        for plane, seqs in zip(x, of):
            for b, n in enumerate(start):
                plane[b, :, :n] = seqs[b]
    cache = LinearCache(caches, _ints(start))
    accept, count, parent = _ints([[0] * 4] * B), _ints([0] * B), _ints([[-2] * T] * B)
    calls = []
    for x, (hq, hkv, D, planes) in zip(caches, heads):
        step = TreeStep.for_cache(x[0], hq, T, kv_shared=planes == 1, scale=D ** -0.5)
        q, kn, vn = (torch.zeros((B, T, h, D), dtype=BF, device=DEV) for h in (hq, hkv, hkv))
        calls.append((TreeCall(step, q, kn, None if planes == 1 else vn, x[0], x[-1], cache.length, parent=parent), q, kn, vn))

    def turn():
        for call, *_ in calls:
            call()
        cache.commit(accept, count)

    graph = None
    if captured:
        turn()  # (no nodes, nothing accepted)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            turn()
    for n in range(4):
        up = random_parents(B, T, n, 0.1)
        parent.copy_(up)
        paths = [paths_of(up[b].tolist()) for b in range(B)]
        taken = [rng.choice([p for p in paths[b] if p] or [[]])[:4] for b in range(B)]
        accept.copy_(_ints([(p + [0] * 4)[:4] for p in taken]))
        count.copy_(_ints([len(p) for p in taken]))
        for _, *tensors in calls:
            for x in tensors:
                x.copy_(_rows(x.shape, g))
        graph.replay() if captured else turn()
        torch.cuda.synchronize()
        for (call, q, kn, vn), of, (hq, hkv, D, planes), x in zip(calls, rows, heads, caches):
            G = hq // hkv
            for b in range(B):
                held = of[0][b].shape[1]
                seen = torch.zeros((T, held + T), dtype=torch.bool, device=DEV)
                for i, path in enumerate(paths[b]):
                    if path:
                        seen[i, :held] = True
                        seen[i, [held + j for j in path]] = True
                for h in range(hkv):
                    k = torch.cat([of[0][b][h], kn[b, :, h]])
                    v = torch.cat([of[-1][b][h], (kn if planes == 1 else vn)[b, :, h]])
                    o, bound = attend64(q[b, :, h * G:(h + 1) * G].reshape(T * G, D), k, v, seen.repeat_interleave(G, 0), D ** -0.5)
                    check(call.out[b, :, h * G:(h + 1) * G].reshape(T * G, D), o, bound, f"turn {n} sequence {b} kv head {h}")
                for plane, new in zip(range(planes), (kn, vn)):
                    of[plane][b] = torch.cat([of[plane][b], new[b, taken[b]].transpose(0, 1)], 1)
                    assert torch.equal(x[plane, b, :, :of[plane][b].shape[1]], of[plane][b])
        assert cache.length.tolist() == [of[0][b].shape[1] for b in range(B)]
    assert cache.left_out() == 0
    assert min(cache.length.tolist()) > 0


def test_rows_past_the_cache_are_left_out():
    x = torch.randint(-2 ** 15, 2 ** 15, (2, 3, 2, 40, 128), dtype=torch.int16, device=DEV)
    first = x.clone()
    cache = LinearCache([x.view(BF)], _ints([36, 38, 0]))
    cache.commit(_ints([[1, 3], [0, 2], [-1, 2]]), _ints([2, 2, 2]))
    assert cache.length.tolist() == [38, 38, 0] and cache.left_out() == 2 and cache.left_out() == 0
    first[:, 0, :, 36], first[:, 0, :, 37] = first[:, 0, :, 37].clone(), first[:, 0, :, 39].clone()
    assert torch.equal(x, first)
    cache.commit(_ints([[5], [0], [63]]), _ints([0, 1, 0]))
    assert cache.length.tolist() == [38, 39, 0] and cache.left_out() == 0 and torch.equal(x, first)


def test_beside_a_busy_stream():
    """tree_decode and commit on a side stream, which waits for the cache's making."""
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    x, q, kn = _rows((1, 2, 1, 40, 128), g), _rows((2, 3, 4, 128), g), _rows((2, 3, 1, 128), g)
    want, length = x.clone(), _ints([7, 30])
    accept, count = _ints([[0, 2], [1, 2]]), _ints([2, 1])
    step, side = TreeStep.for_cache(x[0], 4, 3, kv_shared=True, scale=0.1), torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)
    cache = LinearCache([x], length)
    tree_decode(step, q, kn, None, x[0], None, length, stream=side)
    cache.commit(accept, count, stream=side)
    torch.cuda.synchronize()
    want[0, 0, :, 7:10], want[0, 1, :, 30:33] = kn[0].transpose(0, 1), kn[1].transpose(0, 1)
    want[0, 0, :, 8], want[0, 1, :, 30] = kn[0, 2], kn[1, 1]
    assert length.tolist() == [9, 31] and cache.left_out() == 0 and torch.equal(x, want)
