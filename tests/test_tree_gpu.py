"""GPU parity of esda_tree_decode against 64 bits (_attn64.py: the bound is derived there, per element).

Every row of the pool that no query may see is NaN: pages of nobody, rows behind a sequence's last, rows
before its window, pages that its table does not name.
"""
import pytest
import torch

from _attn64 import attend64, check
from apertura_amd.decode import DecodeStep, decode_step
from apertura_amd.pages import pages_status
from apertura_amd.tree import TreeCall, TreeStep, new_tree_workspace, tree_decode

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
DEV = "cuda"


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _rows(shape, g, gain=1.0):
    x = torch.randn(shape, device=DEV, generator=g)
    return (gain * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(BF)


def random_parents(B, T, seed, holes=0.0):
    """Parents of random trees; with `holes`, some nodes are none (and with them what hangs on them)."""
    g = torch.Generator().manual_seed(seed)
    up = torch.randint(1, 6, (B, T), generator=g)
    parent = torch.arange(T) - up
    parent = torch.where(parent < 0, -1, parent)
    if holes:
        parent = torch.where(torch.rand((B, T), generator=g) < holes, -2, parent)
    return parent.to(torch.int32)


def paths_of(parent):
    """Each node's path, itself last; [] for no node."""
    paths = []
    for i, p in enumerate(parent):
        paths.append([i] if p == -1 else paths[p] + [i] if 0 <= p < i and paths[p] else [])
    return paths


class Case:
    """lengths: committed rows of each sequence.  page 0: linear caches of `cap` rows."""

    def __init__(self, T, hq, hkv, D, lengths, page=16, shared=False, window=0, parent=None, cap=0, split_rows=0,
                 spare=0, gap=0, seed=0):
        g = _gen(seed)
        B = len(lengths)
        self.B, self.T, self.hq, self.hkv, self.D, self.page, self.shared, self.window = B, T, hq, hkv, D, page, shared, window
        self.lengths, self.parent = lengths, parent
        self.paths = [paths_of(list(range(-1, T - 1)) if parent is None else parent[b].tolist()) for b in range(B)]
        self.q, self.kn = _rows((B, T, hq, D), g, 2.5), _rows((B, T, hkv, D), g)
        self.vn = None if shared else _rows((B, T, hkv, D), g)
        R = page or cap
        most = (max(lengths) + T + R - 1) // R + spare if page else 1
        N = B * most + 2 if page else B
        # planes with room between pages and heads where `gap`
        shape = (N, hkv, R + gap, D)
        full = torch.full((1 if shared else 2, N + (1 if gap else 0)) + shape[1:], float("nan"), dtype=BF, device=DEV)
        self.full = full
        self.pool = full[:, :N, :, :R]
        self.table = torch.full((B, most), -1, dtype=torch.int32, device=DEV)
        ids = torch.randperm(N, device=DEV, generator=g) if page else torch.arange(N, device=DEV)
        for b, n in enumerate(lengths):
            for k in range((n + T + R - 1) // R if page else 1):
                self.table[b, k] = ids[b * most + k]
            first = max(0, n - window + 1) if window else 0
            for plane in self.pool:
                rows = _rows((hkv, max(0, n), D), g)
                rows[:, :first] = float("nan")
                for k in range((n + R - 1) // R):
                    part = rows[:, k * R:min(n, (k + 1) * R)]
                    plane[int(self.table[b, k]) if page else b, :, :part.shape[1]] = part
        self.length = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        kw = dict(window=window, kv_shared=shared, scale=D ** -0.5, split_rows=split_rows)
        self.step = TreeStep.for_pages(self.pool[0], self.table, hq, T, **kw) if page else \
            TreeStep.for_cache(self.pool[0], hq, T, **kw)

    def args(self):
        return dict(q=self.q, k_new=self.kn, v_new=self.vn, k_pages=self.pool[0], v_pages=self.pool[-1],
                    length=self.length, table=self.table if self.page else None,
                    parent=None if self.parent is None else self.parent.to(DEV))

    def run(self, **kw):
        print(f"\n[case] T={self.T} Hq={self.hq} Hkv={self.hkv} D={self.D} lengths={self.lengths[:6]} page={self.page} "
              f"window={self.window}", flush=True)
        before = self.full.clone()
        out = tree_decode(self.step, **self.args(), **kw)
        torch.cuda.synchronize()
        self.check(out, before)
        return out

    def row_of(self, full, plane, b, r):
        """[hkv, D] view of row r of sequence b."""
        if not self.page:
            return full[plane, b, :, r]
        return full[plane, int(self.table[b, r // self.page]), :, r % self.page]

    def exact(self, before, b):
        """(o, bound) [hkv, T, G, D] of sequence b."""
        T, G, R, n = self.T, self.hq // self.hkv, self.page or self.pool.shape[3], self.lengths[b]
        pages = self.table[b, :(n + R - 1) // R].long()
        held = [p[pages].transpose(0, 1).reshape(self.hkv, -1, self.D)[:, :n] if self.page else p[b, :, :n]
                for p in (before[0, :, :, :R], before[-1, :, :, :R])]
        seen = torch.zeros((T, n + T), dtype=torch.bool, device=DEV)
        for i, path in enumerate(self.paths[b]):
            if path:
                seen[i, max(0, n + len(path) - self.window) if self.window else 0:n] = True
                seen[i, [n + j for j in path]] = True
        outs = []
        for h in range(self.hkv):
            k = torch.cat([held[0][h], self.kn[b, :, h]])
            v = torch.cat([held[1][h], (self.kn if self.shared else self.vn)[b, :, h]])
            outs.append(attend64(self.q[b, :, h * G:(h + 1) * G].reshape(T * G, self.D), k, v, seen.repeat_interleave(G, 0),
                                 self.D ** -0.5))
        return [torch.stack(x).view(self.hkv, T, G, self.D) for x in zip(*outs)]

    def check(self, out, before, skipped=()):
        T, G = self.T, self.hq // self.hkv
        want = before.clone()
        for b, n in enumerate(self.lengths):
            if b in skipped:
                continue
            for i, path in enumerate(self.paths[b]):
                for plane, new in zip(range(len(want) if path else 0), (self.kn, self.vn)):
                    self.row_of(want, plane, b, n + i)[:] = new[b, i]
            o, bound = self.exact(before, b)
            check(out[b].view(T, self.hkv, G, self.D).transpose(0, 1), o, bound, f"sequence {b}")
        assert torch.equal(self.full.view(torch.int16), want.view(torch.int16)), "cache bytes"


HEADS = [(128, 8, 2, False), (128, 16, 1, True), (128, 2, 2, False), (256, 4, 2, False), (256, 5, 5, True), (512, 8, 1, True),
         (512, 4, 2, False)]


@pytest.mark.parametrize("lengths", [[0], [1], [15, 16], [17, 0, 33], [31, 32, 64, 5], [500, 3]])
@pytest.mark.parametrize("D,hq,hkv,shared", HEADS)
def test_single_tokens(D, hq, hkv, shared, lengths):
    Case(1, hq, hkv, D, lengths, 16, shared, seed=len(lengths)).run()


@pytest.mark.parametrize("T", [2, 3, 8, 17, 33, 64])
@pytest.mark.parametrize("D,hq,hkv,shared", HEADS)
def test_chains(D, hq, hkv, shared, T):
    Case(T, hq, hkv, D, [0, 1, 30, 129], 32, shared, seed=T).run()


@pytest.mark.parametrize("T", [2, 7, 16, 31, 64])
@pytest.mark.parametrize("D,hq,hkv,shared", HEADS)
def test_trees(D, hq, hkv, shared, T):
    Case(T, hq, hkv, D, [100, 0, 17], 16, shared, parent=random_parents(3, T, T), seed=T).run()
    Case(T, hq, hkv, D, [70, 3, 200, 9], 64, shared, parent=random_parents(4, T, T, 0.3), seed=T + 1).run()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 4096])
@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 2, False), (256, 4, 2, False), (512, 8, 1, True)])
def test_page_sizes(D, hq, hkv, shared, page):
    Case(5, hq, hkv, D, [page - 1, page, page + 1, 2 * page - 3], page, shared, seed=page).run()


@pytest.mark.parametrize("T,window", [(1, 1), (1, 16), (1, 33), (5, 5), (8, 40), (64, 64), (20, 100)])
@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 2, False), (256, 4, 2, False), (512, 8, 1, True)])
def test_windows(D, hq, hkv, shared, T, window):
    Case(T, hq, hkv, D, [0, 7, window, 300, 2 * window + 5], 16, shared, window, parent=random_parents(5, T, window), seed=T).run()
    Case(T, hq, hkv, D, [300, 95], 64, shared, window, seed=T).run()


@pytest.mark.parametrize("T", [1, 6, 40])
@pytest.mark.parametrize("D,hq,hkv,shared", HEADS)
def test_linear_caches(D, hq, hkv, shared, T):
    Case(T, hq, hkv, D, [0, 50, 333 - T], 0, shared, cap=333, seed=T).run()
    Case(T, hq, hkv, D, [77, 12], 0, shared, cap=201, window=64, parent=random_parents(2, T, 5), gap=3, seed=T).run()


@pytest.mark.parametrize("split_rows", [32, 64, 96, 1024, 2 ** 31 - 32])
@pytest.mark.parametrize("T", [1, 9, 33])
@pytest.mark.parametrize("D,hq,hkv,shared", HEADS)
def test_splits(D, hq, hkv, shared, T, split_rows):
    Case(T, hq, hkv, D, [700, 64, 0, 31], 16, shared, parent=random_parents(4, T, 3), split_rows=split_rows, spare=3, seed=T).run()


@pytest.mark.parametrize("T", [1, 12])
@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 2, False), (256, 4, 2, False), (512, 8, 1, True)])
def test_long_sequences(D, hq, hkv, shared, T):
    """Tables of more than 64 entries, more than 40 partials a row."""
    Case(T, hq, hkv, D, [5000, 2111], 16, shared, seed=T).run()
    Case(T, hq, hkv, D, [5000, 2111], 16, shared, split_rows=64, gap=1, seed=T).run()


@pytest.mark.parametrize("T", [1, 3, 30])
@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 2, False), (256, 4, 2, False), (512, 8, 1, True)])
def test_ragged_batches(D, hq, hkv, shared, T):
    """One sequence far longer than the others; tables with much more room than rows; more than 64
    sequences, the long one among the last."""
    Case(T, hq, hkv, D, [9000, 2, 20, 0, 77], 16, shared, parent=random_parents(5, T, 1), spare=300, seed=1).run()
    Case(T, hq, hkv, D, [n % 37 for n in range(130)] + [4000, 1], 16, shared, seed=2).run()


@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 8, False), (256, 8, 4, False), (512, 8, 1, True)])
def test_the_largest_batch(D, hq, hkv, shared):
    g = torch.Generator().manual_seed(3)
    Case(2, hq, hkv, D, torch.randint(0, 60, (256,), generator=g).tolist(), 16, shared, seed=5).run()


@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 32, 8, False), (256, 32, 16, False), (512, 32, 4, True)])
def test_serving_shapes(D, hq, hkv, shared):
    Case(1, hq, hkv, D, [1500, 2100, 4, 900, 37, 2048], 16, shared, seed=3).run()
    Case(63, hq, hkv, D, [1500, 37], 128, shared, parent=random_parents(2, 63, 9), seed=4).run()
    Case(24, hq, hkv, D, [1100, 37, 1024], 32, shared, 1024, parent=random_parents(3, 24, 9, 0.1), seed=4).run()


@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 2, False), (256, 4, 2, False), (512, 8, 1, True)])
def test_one_token_is_the_decode_step(D, hq, hkv, shared):
    """Over the same linear rows: each is within its bound of the exact values."""
    c = Case(1, hq, hkv, D, [200, 31, 0], 0, shared, cap=256, seed=6)
    k, v = c.pool[0].clone(), c.pool[-1].clone()
    step = DecodeStep.for_cache(k, hq, kv_shared=shared, scale=D ** -0.5)
    a = decode_step(step, c.q[:, 0], c.kn[:, 0], None if shared else c.vn[:, 0], k, k if shared else v, c.length)
    b = c.run()[:, 0]
    err = (a.float() - b.float()).abs()
    assert float(err.max()) <= 2e-2 and float(err.mean()) <= 2e-3
    assert torch.equal(k.view(torch.int16), c.pool[0].view(torch.int16))


@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("D,hq,hkv,shared", HEADS)
def test_pages_that_are_none_are_left_out(D, hq, hkv, shared, T):
    """Entries of committed rows outside the pool: the rows have no weight, nothing else changes."""
    c = Case(T, hq, hkv, D, [150, 40], 16, shared, seed=7)
    G = hq // hkv
    gone = [(0, 2, -1), (0, 5, c.pool.shape[1]), (1, 0, 2 ** 31 - 1)]
    missing = torch.zeros((2, 150 + T), dtype=torch.bool, device=DEV)
    held = [[torch.cat([plane[c.table[b, :10].clamp(min=0).long()].transpose(0, 1).reshape(hkv, -1, D)[:, :n], new[b].transpose(0, 1)], 1)
             for plane, new in zip((c.pool[0], c.pool[-1]), (c.kn, c.kn if shared else c.vn))] for b, n in enumerate(c.lengths)]
    for b, k, page in gone:
        c.table[b, k] = page
        missing[b, 16 * k:16 * k + 16] = True
    out = tree_decode(c.step, **c.args())
    for b, n in enumerate(c.lengths):
        seen = torch.ones((T, n + T), dtype=torch.bool, device=DEV).tril(n) & ~missing[b, :n + T]
        for h in range(hkv):
            o, bound = attend64(c.q[b, :, h * G:(h + 1) * G].reshape(T * G, D), held[b][0][h], held[b][1][h],
                                seen.repeat_interleave(G, 0), D ** -0.5)
            check(out[b, :, h * G:(h + 1) * G].reshape(T * G, D), o, bound, f"sequence {b} kv head {h}")


@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("D,hq,hkv,shared", HEADS)
def test_sequences_outside_their_cache_are_skipped(D, hq, hkv, shared, T):
    c = Case(T, hq, hkv, D, [20, 40, 33, 64, 5], 16, shared, seed=8)
    bad = {0: -1, 1: c.table.shape[1] * 16, 3: 2 ** 31 - 1}
    for b, n in bad.items():
        c.length[b] = n
    c.table[2, (33 + T - 1) // 16] = c.pool.shape[1]  # the last node's page
    out = torch.full_like(c.q, 7.0)
    ws = new_tree_workspace(c.step, DEV)
    before = c.full.clone()
    call = TreeCall(c.step, **c.args(), out=out, workspace=ws)
    call()
    torch.cuda.synchronize()
    assert bool((out[:4] == 7.0).all())
    assert pages_status(ws) == 4 and pages_status(ws) == 0
    c.check(out, before, skipped=(0, 1, 2, 3))


@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 2, False), (256, 4, 2, False), (512, 8, 1, True), (512, 4, 2, False)])
@pytest.mark.parametrize("split_rows", [0, 32])
def test_values_that_are_not_finite_stay_with_their_queries(D, hq, hkv, shared, split_rows):
    """A node's K and V of NaN or infinity reach that node and what hangs on it only; a value in the window's
    last row only those that see it."""
    T, G = 13, hq // hkv
    parent = random_parents(2, T, 4)
    c = Case(T, hq, hkv, D, [90, 40], 16, shared, window=32, parent=parent, split_rows=split_rows, seed=9)
    before, paths = c.full.clone(), c.paths
    clean = tree_decode(c.step, **c.args())
    for bad in (float("nan"), float("inf"), -float("inf")):
        kn, vn = c.kn.clone(), None if shared else c.vn.clone()
        (kn if shared else vn)[0, 4, 0] = bad
        kn[1, 2, 0, 5] = bad
        args = dict(c.args(), k_new=kn, v_new=vn)
        out = tree_decode(c.step, **args)
        for b, node in ((0, 4), (1, 2)):
            o, bound = c.exact(before, b)
            for i in range(T):
                if node not in paths[b][i]:
                    check(out[b, i, :G], o[0, i], bound[0, i], f"sequence {b} node {i}")
                elif b == 0:
                    assert not bool(torch.isfinite(out[b, i, :G]).any()), (b, i)
        assert torch.equal(out[:, :, G:], clean[:, :, G:])  # the other kv heads


def test_chosen_paths_equal_the_chain():
    """A tree's node sees what the last of a chain of its path sees."""
    D, hq, hkv, T = 128, 8, 2, 30
    parent = random_parents(1, T, 11)
    c = Case(T, hq, hkv, D, [100], 16, parent=parent, seed=10)
    out = c.run()
    for i in (T - 1, T // 2, 3):
        path = c.paths[0][i]
        d = Case(len(path), hq, hkv, D, [100], 16, seed=10)
        for plane in range(2):
            for k in range((100 + 15) // 16):
                d.pool[plane, int(d.table[0, k])] = c.pool[plane, int(c.table[0, k])]
        d.q, d.kn, d.vn = (x[:, path].contiguous() for x in (c.q, c.kn, c.vn))
        err = (d.run()[0, -1].float() - out[0, i].float()).abs()
        assert float(err.max()) <= 2e-2


def test_graph_replays():
    D, hq, hkv, T = 256, 4, 2, 6
    c = Case(T, hq, hkv, D, [100, 250], 16, parent=random_parents(2, T, 2), spare=4, split_rows=64, seed=12)
    args = c.args()
    call = TreeCall(c.step, **args)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for turn in range(3):
        c.q.copy_(_rows(c.q.shape, _gen(20 + turn), 2.5))
        args["parent"].copy_(random_parents(2, T, 30 + turn, 0.2 * turn))
        c.parent = args["parent"].cpu()
        c.paths = [paths_of(c.parent[b].tolist()) for b in range(2)]
        before = c.full.clone()
        call.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        c.check(call.out, before)


def test_two_streams():
    """Two steps at once, each with its workspace, on streams of their own."""
    a = Case(5, 8, 2, 128, [700, 30], 16, split_rows=64, seed=13)
    b = Case(7, 8, 1, 512, [900, 1], 32, True, split_rows=64, seed=14)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    before = [a.full.clone(), b.full.clone()]
    torch.cuda.synchronize()
    outs = [tree_decode(c.step, **c.args(), stream=st) for c, st in zip((a, b), s)]
    torch.cuda.synchronize()
    a.check(outs[0], before[0])
    b.check(outs[1], before[1])


@pytest.mark.parametrize("T", [1, 4, 20, 64])
@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 2, False), (256, 4, 2, False), (512, 8, 1, True)])
def test_padded_batches(D, hq, hkv, shared, T):
    """Sequences of no rows, no pages and no nodes beside real ones give zeros and are not counted."""
    parent = random_parents(5, T, T)
    parent[1::2] = -2
    c = Case(T, hq, hkv, D, [70, 0, 500, 0, 3], 16, shared, parent=parent, seed=T)
    c.table[1::2] = -1
    out = torch.full_like(c.q, float("nan"))
    workspace = new_tree_workspace(c.step, DEV)
    c.run(out=out, workspace=workspace)
    assert (out[1::2] == 0).all()
    assert pages_status(workspace) == 0


def test_pages_past_32_bit_offsets():
    """A pool of more than 2^32 elements; the sequence's pages lie at its end."""
    D, hq, hkv, R = 128, 8, 8, 1024
    N = (2 ** 32) // (hkv * R * D) + 4
    pool = torch.empty((1, N, hkv, R, D), dtype=BF, device=DEV)
    g = _gen(15)
    rows = _rows((hkv, 2 * R, D), g)
    pool[0, N - 1], pool[0, N - 3] = rows[:, :R], rows[:, R:]
    table = torch.tensor([[N - 1, N - 3]], dtype=torch.int32, device=DEV)
    length = torch.tensor([2 * R - 4], dtype=torch.int32, device=DEV)
    q, kn = _rows((1, 3, hq, D), g, 2.5), _rows((1, 3, hkv, D), g)
    step = TreeStep.for_pages(pool[0], table, hq, 3, kv_shared=True, scale=D ** -0.5)
    out = tree_decode(step, q, kn, None, pool[0], None, length, table)
    seen = torch.ones((3, 2 * R - 1), dtype=torch.bool, device=DEV).tril(2 * R - 4)
    for h in range(hkv):
        k = torch.cat([rows[h, :2 * R - 4], kn[0, :, h]])
        o, bound = attend64(q[0, :, h], k, k, seen, D ** -0.5)
        check(out[0, :, h], o, bound, f"head {h}")
    assert torch.equal(pool[0, N - 3, :, R - 4:R - 1], kn[0].transpose(0, 1))


@pytest.mark.parametrize("D,hq,hkv,shared,T,lengths", [
    (128, 32, 8, False, 1, [4000]), (128, 32, 8, False, 6, [4000, 900]), (128, 32, 8, False, 6, [300, 9]), (128, 16, 2, False, 64, [600] * 20),
    (128, 32, 8, False, 16, [8000, 5000]), (128, 32, 8, False, 40, [9000, 100]), (128, 16, 16, True, 64, [3000]),
    (256, 32, 16, False, 4, [5000, 11]), (256, 32, 16, False, 20, [6000, 3]), (256, 32, 16, False, 64, [9000, 4000]), (256, 16, 1, True, 64, [500, 2]),
    (512, 32, 4, True, 2, [6000, 70]), (512, 32, 4, True, 4, [6000, 70]), (512, 32, 4, True, 8, [6000, 70]), (512, 32, 4, True, 12, [9000, 70]),
    (512, 32, 4, True, 12, [20000, 13000]), (512, 32, 4, True, 64, [200] * 9), (512, 8, 8, False, 64, [3000, 17]), (512, 16, 2, False, 4, [9000]),
    (512, 16, 4, False, 64, [700, 4000]), (512, 32, 4, True, 30, [300])])
@pytest.mark.parametrize("window", [0, 1024])
def test_every_form(D, hq, hkv, shared, T, lengths, window):
    """The forms and splits that the rules choose between, with holes in the trees."""
    Case(T, hq, hkv, D, lengths, 32, shared, window, parent=random_parents(len(lengths), T, T, 0.1), seed=T + D).run()


@pytest.mark.parametrize("D,hq,hkv,shared,T,cap", [(128, 32, 8, False, 40, 20000), (256, 32, 16, False, 64, 9000), (256, 32, 16, False, 20, 9000),
                                                   (512, 32, 4, True, 8, 9000), (512, 32, 4, True, 64, 9000), (512, 8, 4, False, 64, 9000)])
def test_tiles_over_bad_pages_and_values(D, hq, hkv, shared, T, cap):
    """What the tiles do about pages that are none and values that are not finite."""
    parent = random_parents(2, T, 5)
    parent[:, T - 3:] = torch.tensor([-2, T, T - 2], dtype=torch.int32)  # no nodes: two that are told so, one on such
    c = Case(T, hq, hkv, D, [700, 90], 16, shared, parent=parent, spare=(cap - 700) // 16, seed=T)
    G, before = hq // hkv, c.full.clone()
    bad = 2
    clean, clean_bound = c.exact(before, 1)
    (c.kn if shared else c.vn)[0, bad, 1] = float("inf")
    c.kn[1, 1, 0, 3] = float("nan")
    held = c.table[0, 7].item()
    c.table[0, 7] = -7
    out = tree_decode(c.step, **c.args())
    c.table[0, 7] = held
    k = [torch.cat([p[c.table[0, :44].long()].transpose(0, 1).reshape(hkv, -1, D)[:, :700], n[0].transpose(0, 1)], 1)
         for p, n in ((before[0], c.kn), (before[-1], c.kn if shared else c.vn))]
    seen = torch.zeros((T, 700 + T), dtype=torch.bool, device=DEV)
    for i, path in enumerate(c.paths[0]):
        if path:
            seen[i, :700] = True
            seen[i, [700 + j for j in path]] = True
    seen[:, 112:128] = False
    for h in range(hkv):
        sees = torch.tensor([h == 1 and bad in path for path in c.paths[0]], device=DEV)
        kk, vv = k[0][h].clone(), k[1][h].clone()
        if h == 1:  # (clean where the others look)
            kk[700 + bad], vv[700 + bad] = 0.0, 0.0
        o, bound = attend64(c.q[0, :, h * G:(h + 1) * G].reshape(T * G, D), kk, vv, seen.repeat_interleave(G, 0), D ** -0.5)
        got = out[0, :, h * G:(h + 1) * G].reshape(T * G, D)
        rest = (~sees).repeat_interleave(G)
        check(got[rest], o[rest], bound[rest], f"kv head {h}")
        assert not bool(torch.isfinite(got[~rest]).any())
    for i, path in enumerate(c.paths[1]):
        for h in range(hkv):
            if 1 not in path or h != 0:
                check(out[1, i, h * G:(h + 1) * G], clean[h, i], clean_bound[h, i], f"node {i} kv head {h}")
