"""Caches in pages as a serving loop uses them: prompts written, trees of drafted tokens attended and
committed on layers of two head shapes over one table, sequences forked, cut, ended, pages compacted, rows
read out again.  Every step is checked against 64 bits over rows that the test keeps itself."""
import random

import pytest
import torch

from _attn64 import attend64, check
from apertura_amd.decode import DecodeStep, decode_step
from apertura_amd.pages import PagedCache, pages_read, pages_write
from apertura_amd.rope import rope, rope_frequencies
from apertura_amd.tree import TreeCall, TreeStep
from test_tree_gpu import paths_of, random_parents

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
DEV = "cuda"


def _rows(shape, g, gain=1.0):
    x = torch.randn(shape, device=DEV, generator=g)
    return (gain * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(BF)


class Layer:
    """hq query and hkv kv heads; planes of one pool: K and V, or the K = V rows."""

    def __init__(self, hq, hkv, D, shared, window=0):
        self.hq, self.hkv, self.D, self.shared, self.window = hq, hkv, D, shared, window
        self.planes = 1 if shared else 2


class Serving:
    def __init__(self, layers, slots, pages, R, most, T, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)
        self.rng = random.Random(seed)
        self.layers, self.R, self.T, self.slots = layers, R, T, slots
        self.pools = [torch.full((x.planes, pages, x.hkv, R, x.D), float("nan"), dtype=BF, device=DEV) for x in layers]
        self.cache = PagedCache.empty(self.pools, slots, most)
        self.parent = torch.full((slots, T), -2, dtype=torch.int32, device=DEV)
        self.q = [torch.zeros((slots, T, x.hq, x.D), dtype=BF, device=DEV) for x in layers]
        self.new = [[torch.zeros((slots, T, x.hkv, x.D), dtype=BF, device=DEV) for _ in range(x.planes)] for x in layers]
        self.calls = []
        for x, pool, q, new in zip(layers, self.pools, self.q, self.new):
            step = TreeStep.for_pages(pool[0], self.cache.table, x.hq, T, window=x.window, kv_shared=x.shared, scale=x.D ** -0.5)
            self.calls.append(TreeCall(step, q, new[0], None if x.shared else new[1], pool[0], pool[-1], self.cache.length,
                                       table=self.cache.table, parent=self.parent))
        # what the test holds: rows[slot][layer][plane] is [hkv, length, D]
        self.rows = {}

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    def prompt(self, slot, n):
        """A prompt's rows, prefilled elsewhere, into its pages."""
        self.cache.reserve(self.ints([slot]), self.ints([n]))
        self.rows[slot] = []
        for x, pool in zip(self.layers, self.pools):
            rows = _rows((x.planes, 1, x.hkv, n, x.D), self.g)
            pages_write(pool, self.cache.table[slot:slot + 1], self.ints([0]), rows)
            self.rows[slot].append([rows[i, 0].clone() for i in range(x.planes)])
        self.cache.length[slot] = n

    def length(self, slot):
        return self.rows[slot][0][0].shape[1]

    def draft(self, replay=None):
        """One step of every live slot: drafted trees, attention on each layer, a path committed."""
        T, live = self.T, sorted(self.rows)
        parents = random_parents(self.slots, T, self.rng.randrange(10 ** 6), 0.15)
        for s in range(self.slots):
            if s not in self.rows:
                parents[s] = -2
        self.parent.copy_(parents)
        for q, new in zip(self.q, self.new):
            q.copy_(_rows(q.shape, self.g, 2.5))
            for t in new:
                t.copy_(_rows(t.shape, self.g))
        self.cache.reserve(self.ints(live), self.ints([self.length(s) + T for s in live]))
        accept = torch.zeros((self.slots, T), dtype=torch.int32)
        count = torch.zeros(self.slots, dtype=torch.int32)
        chosen = {}
        for s in live:
            paths = [p for p in paths_of(parents[s].tolist()) if p] or [[]]
            chosen[s] = self.rng.choice(paths)
            accept[s, :len(chosen[s])] = torch.tensor(chosen[s], dtype=torch.int32)
            count[s] = len(chosen[s])
        if replay is None:
            outs = [call() for call in self.calls]
            self.cache.commit(accept.to(DEV), count.to(DEV))
        else:
            graph, a, c = replay
            a.copy_(accept)
            c.copy_(count)
            graph.replay()
            outs = [call.out for call in self.calls]
        torch.cuda.synchronize()
        for i, (x, out, new) in enumerate(zip(self.layers, outs, self.new)):
            G = x.hq // x.hkv
            for s in range(self.slots):
                if s not in self.rows:
                    assert not bool(out[s].any()), "a slot without nodes"
                    continue
                n, paths = self.length(s), paths_of(parents[s].tolist())
                seen = torch.zeros((T, n + T), dtype=torch.bool, device=DEV)
                for j, path in enumerate(paths):
                    if path:
                        seen[j, max(0, n + len(path) - x.window) if x.window else 0:n] = True
                        seen[j, [n + k for k in path]] = True
                for h in range(x.hkv):
                    k, v = [torch.cat([self.rows[s][i][p][h], new[p][s, :, h]]) for p in (0, x.planes - 1)]
                    o, bound = attend64(self.q[i][s, :, h * G:(h + 1) * G].reshape(T * G, x.D), k, v, seen.repeat_interleave(G, 0),
                                        x.D ** -0.5)
                    check(out[s, :, h * G:(h + 1) * G].reshape(T * G, x.D), o, bound, f"layer {i} slot {s} kv head {h}")
        for s in live:
            for i, new in enumerate(self.new):
                for p, t in enumerate(new):
                    self.rows[s][i][p] = torch.cat([self.rows[s][i][p], t[s, chosen[s]].transpose(0, 1)], dim=1)
        self.check()

    def fork(self, src, dst, rows):
        self.cache.fork(self.ints(src), self.ints(dst), self.ints(rows))
        made = {d: [[t[:, :n].clone() for t in planes] for planes in self.rows[s]] for s, d, n in zip(src, dst, rows)}
        self.rows.update(made)
        self.check()

    def free(self, slots):
        self.cache.free(self.ints(slots))
        for s in slots:
            del self.rows[s]
        self.check()

    def compact(self):
        self.cache.compact()
        live = int((self.cache.refs > 0).sum())
        assert bool((self.cache.refs[:live] > 0).all())
        self.check()

    def check(self):
        """Lengths, and every row as its pages hold it."""
        assert self.cache.left_out() == 0
        lengths = self.cache.length.tolist()
        for s in range(self.slots):
            assert lengths[s] == (self.length(s) if s in self.rows else 0)
        for s in self.rows:
            for i, (x, pool) in enumerate(zip(self.layers, self.pools)):
                got = pages_read(pool, self.cache.table[s:s + 1], self.ints([0]), self.length(s))
                for p in range(x.planes):
                    assert torch.equal(got[p, 0].view(torch.int16), self.rows[s][i][p].contiguous().view(torch.int16)), (s, i, p)


LAYERS = [Layer(4, 2, 256, False), Layer(8, 1, 512, True), Layer(4, 2, 256, False, window=64)]


@pytest.mark.parametrize("R,T", [(16, 9), (64, 24)])
def test_a_serving_loop(R, T):
    print(f"\n[case] pages of {R}, {T} nodes", flush=True)
    s = Serving(LAYERS, slots=5, pages=5 * 300 // R + 30, R=R, most=400 // R + 2, T=T, seed=R)
    s.prompt(0, 100)
    s.prompt(3, 2 * R)
    s.draft()
    s.draft()
    s.fork([0, 3, 0], [1, 2, 4], [s.length(0), s.length(3), 50])  # samples, and one from an earlier turn
    s.draft()
    s.draft()
    s.free([3])
    s.fork([0], [0], [s.length(0) - 3])                           # a rewind
    s.compact()
    s.draft()
    s.fork([1, 0], [0, 1], [s.length(1), s.length(0)])            # two that change places
    s.prompt(3, 33)
    s.draft()
    s.free([0, 2])
    s.compact()
    s.draft()
    # a slot's rows, read out, are what the decode step over linear rows attends
    x, n = LAYERS[0], s.length(1)
    k, v = [torch.cat([p[0], torch.zeros((1, x.hkv, 1, x.D), dtype=BF, device=DEV)[0]], dim=1)[None].contiguous()
            for p in pages_read(s.pools[0], s.cache.table[1:2], s.ints([0]), n)]
    g = s.g
    q, kn, vn = _rows((1, x.hq, x.D), g, 2.5), _rows((1, x.hkv, x.D), g), _rows((1, x.hkv, x.D), g)
    out = decode_step(DecodeStep.for_cache(k, x.hq, scale=x.D ** -0.5), q, kn, vn, k, v, s.ints([n]))
    for h in range(x.hkv):
        o, bound = attend64(q[0, 2 * h:2 * h + 2], k[0, h], v[0, h], torch.ones((2, n + 1), dtype=torch.bool, device=DEV), x.D ** -0.5)
        check(out[0, 2 * h:2 * h + 2], o, bound, f"kv head {h}")


def test_a_captured_step():
    """Attention on every layer and the commit in one graph, replayed for step after step."""
    s = Serving(LAYERS, slots=3, pages=120, R=16, most=20, T=7, seed=3)
    s.prompt(0, 40)
    s.prompt(2, 90)
    s.draft()
    accept, count = torch.zeros((3, 7), dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for call in s.calls:
            call()
        s.cache.commit(accept, count)
    for turn in range(4):
        s.draft((graph, accept, count))
        if turn == 1:
            s.fork([0], [1], [s.length(0) - 2])
            s.compact()


def test_rotary_positions_of_a_tree():
    """A node's position is its sequence's length and its depth: a chain decoded token by token and the same
    chain drafted at once agree, rotated by rope()."""
    D, hq, hkv, n, T = 128, 8, 2, 50, 6
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    inv, _ = rope_frequencies(D, 10000.0, device=DEV)
    k0 = _rows((1, hkv, 64, D), g)
    v0 = _rows((1, hkv, 64, D), g)
    q, kn, vn = _rows((T, hq, D), g, 2.5), _rows((T, hkv, D), g), _rows((T, hkv, D), g)
    q, kn = rope(q, kn, n + torch.arange(T, device=DEV, dtype=torch.int32), inv)
    k, v = k0.clone(), v0.clone()
    step = DecodeStep.for_cache(k, hq, scale=D ** -0.5)
    one = torch.stack([decode_step(step, q[i:i + 1], kn[i:i + 1], vn[i:i + 1], k, v, torch.tensor([n + i], dtype=torch.int32, device=DEV))[0]
                       for i in range(T)])
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device=DEV)
    pool = torch.empty((2, 4, hkv, 16, D), dtype=BF, device=DEV)
    pages_write(pool, table, torch.zeros(1, dtype=torch.int32, device=DEV), torch.stack([k0, v0]))
    step = TreeStep.for_pages(pool[0], table, hq, T, scale=D ** -0.5)
    out = TreeCall(step, q[None].contiguous(), kn[None].contiguous(), vn[None].contiguous(), pool[0], pool[1],
                   torch.tensor([n], dtype=torch.int32, device=DEV), table=table)()
    err = (out[0].float() - one.float()).abs()
    assert float(err.max()) <= 2e-2 and float(err.mean()) <= 2e-3
    back = pages_read(pool, table, torch.zeros(1, dtype=torch.int32, device=DEV), 64)
    assert torch.equal(back[0].view(torch.int16), k.view(torch.int16)) and torch.equal(back[1].view(torch.int16), v.view(torch.int16))
