"""GPU parity of esda_prefix_decode against 64 bits (_attn64.py: the bound is derived there, per
element) and against esda_decode over one cache that holds prefix and own rows.

Rows of the own caches that are not visible are NaN.
"""
import pytest
import torch

from _attn64 import attend64, check
from apertura_amd.decode import DecodeStep, decode_status, decode_step
from apertura_amd.prefill import PrefillStep, prefill
from apertura_amd.prefix import PrefixCall, PrefixStep, new_prefix_workspace, prefix_decode
from apertura_amd.rope import rope, rope_frequencies

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


class Case:
    def __init__(self, B, hq, hkv, D, P, cap, own, shared=False, split_keys=0, split_rows=0, max_visible=0, seed=0):
        g = _gen(seed)
        self.B, self.hq, self.hkv, self.D, self.P, self.cap, self.own, self.shared = B, hq, hkv, D, P, cap, own, shared
        self.q, self.kn = _rows((B, hq, D), g, 2.5), _rows((B, hkv, D), g)
        self.pk, self.kc = _rows((hkv, P, D), g), _rows((B, hkv, cap, D), g)
        self.pv = self.pk if shared else _rows((hkv, P, D), g)
        self.vc = self.kc if shared else _rows((B, hkv, cap, D), g)
        self.vn = None if shared else _rows((B, hkv, D), g)
        for b, m in enumerate(own):  # own[b]: the new token's row
            if 0 <= m < cap:
                self.kc[b, :, m:] = float("nan")
                self.vc[b, :, m:] = float("nan")
        self.pos = torch.tensor([P + m for m in own], dtype=torch.int32, device=DEV)
        self.step = PrefixStep.for_caches(self.pk, self.kc, hq, split_keys, kv_shared=shared, scale=D ** -0.5,
                                          split_rows=split_rows, max_visible=max_visible)

    def args(self):
        return (self.q, self.kn, self.vn, self.pk, self.pv, self.kc, self.vc, self.pos)

    def run(self):
        print(f"\n[case] B={self.B} Hq={self.hq} Hkv={self.hkv} D={self.D} P={self.P} cap={self.cap} own={self.own[:6]}",
              flush=True)
        k0, v0 = self.kc.clone(), self.vc.clone()
        out = prefix_decode(self.step, *self.args())
        torch.cuda.synchronize()
        self.check(out, k0, v0)
        return out

    def check(self, out, k0, v0):
        G = self.hq // self.hkv
        kn, vn = self.kn, self.kn if self.shared else self.vn
        for b, m in enumerate(self.own):
            for h in range(self.hkv):
                k = torch.cat([self.pk[h], k0[b, h, :m], kn[b, h][None]])
                v = torch.cat([self.pv[h], v0[b, h, :m], vn[b, h][None]])
                o, bound = attend64(self.q[b, h * G:(h + 1) * G], k, v,
                                    torch.ones((G, len(k)), dtype=torch.bool, device=DEV), self.D ** -0.5)
                check(out[b, h * G:(h + 1) * G], o, bound, f"sequence {b} kv head {h}")
        for c, c0, new in ((self.kc, k0, kn), (self.vc, v0, vn)):
            for b, m in enumerate(self.own):
                c0[b, :, m] = new[b]
            assert torch.equal(c.view(torch.int16), c0.view(torch.int16)), "cache bytes"


HEADS = [(128, 8, 2, False), (128, 16, 1, True), (256, 4, 2, False), (256, 5, 5, True), (512, 8, 1, True),
         (512, 4, 2, False)]


def _own(B, cap, seed):
    g = torch.Generator().manual_seed(seed)
    own = torch.randint(0, cap, (B,), generator=g).tolist()
    own[0] = cap - 1
    if B > 1:
        own[1] = 0
    return own


@pytest.mark.parametrize("P", [1, 31, 32, 33, 500])
@pytest.mark.parametrize("B", [1, 2, 3, 9, 33])
@pytest.mark.parametrize("D,hq,hkv,shared", HEADS)
def test_prefix_lengths_and_batches(D, hq, hkv, shared, B, P):
    Case(B, hq, hkv, D, P, 70, _own(B, 70, B + P), shared, seed=P).run()


@pytest.mark.parametrize("split_keys,split_rows", [(32, 0), (64, 16), (1024, 0), (0, 32)])
@pytest.mark.parametrize("D,hq,hkv,shared", HEADS)
def test_splits(D, hq, hkv, shared, split_keys, split_rows):
    Case(5, hq, hkv, D, 401, 150, _own(5, 150, 1), shared, split_keys, split_rows, seed=1).run()
    Case(1, hq, hkv, D, 401, 150, [149], shared, split_keys, split_rows, seed=2).run()


@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 32, 8, False), (256, 32, 16, False), (512, 32, 4, True)])
def test_serving_shapes(D, hq, hkv, shared):
    Case(32, hq, hkv, D, 2100, 40, _own(32, 40, 3), shared, seed=3).run()
    Case(1, hq, hkv, D, 5000, 300, [123], shared, seed=4).run()


@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 8, False), (512, 8, 1, True)])
def test_the_largest_batch(D, hq, hkv, shared):
    Case(256, hq, hkv, D, 100, 9, _own(256, 9, 5), shared, seed=5).run()


@pytest.mark.parametrize("P", [20000])
@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 2, False), (256, 4, 2, False), (512, 8, 1, True)])
def test_long_prefix(D, hq, hkv, shared, P):
    """More than 64 partials a row."""
    Case(2, hq, hkv, D, P, 64, [3, 63], shared, seed=6).run()
    Case(2, hq, hkv, D, P, 64, [3, 63], shared, split_keys=128, split_rows=16, seed=6).run()


def test_a_low_estimate_of_own_rows():
    Case(1, 8, 2, 128, 64, 500, [480], max_visible=32, seed=7).run()
    Case(3, 8, 2, 128, 64, 500, [480, 2, 333], max_visible=32, seed=7).run()


@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 2, False), (256, 4, 2, False), (512, 8, 1, True)])
def test_one_cache_holding_both(D, hq, hkv, shared):
    """esda_decode over caches that hold prefix and own rows: each is within its bound of the exact
    values, so the two within both bounds of each other."""
    c = Case(4, hq, hkv, D, 300, 50, [10, 49, 0, 25], shared, seed=8)
    k = torch.cat([c.pk[None].expand(4, -1, -1, -1), c.kc], dim=2)
    v = k if shared else torch.cat([c.pv[None].expand(4, -1, -1, -1), c.vc], dim=2)
    step = DecodeStep.for_cache(k, hq, kv_shared=shared, scale=D ** -0.5)
    a = decode_step(step, c.q, c.kn, c.vn, k, v, c.pos)
    b = c.run()
    err = (a.float() - b.float()).abs()
    assert float(err.max()) <= 2e-2 and float(err.mean()) <= 2e-3


def test_sequences_outside_their_cache_are_skipped():
    c = Case(5, 8, 2, 128, 100, 32, [3, 32, -1, -200, 31], seed=9)
    ws, out, k0 = new_prefix_workspace(c.step, DEV), torch.full_like(c.q, 5.0), c.kc.clone()
    prefix_decode(c.step, *c.args(), out=out, workspace=ws)
    assert decode_status(c.step.own, ws) == 3
    assert bool((out[1:4] == 5.0).all()) and bool((out[[0, 4]] != 5.0).any())
    k0[0, :, 3], k0[4, :, 31] = c.kn[0], c.kn[4]
    assert torch.equal(c.kc.view(torch.int16), k0.view(torch.int16))
    for keep in (0, 4):
        o, bound = attend64(c.q[keep, :4], torch.cat([c.pk[0], c.kc[keep, 0, :c.own[keep] + 1]]),
                            torch.cat([c.pv[0], c.vc[keep, 0, :c.own[keep] + 1]]),
                            torch.ones((4, 100 + c.own[keep] + 1), dtype=torch.bool, device=DEV), 128 ** -0.5)
        check(out[keep, :4], o, bound)


def test_one_sequence_that_is_not_finite_leaves_the_others():
    """A NaN in one sequence's own rows or query: the others' outputs bit for bit as without it."""
    c, d = (Case(6, 8, 2, 128, 200, 40, [5, 39, 0, 17, 8, 30], seed=10) for _ in range(2))
    a = c.run()
    d.kc[3, :, 2], d.q[1, 2] = float("nan"), float("nan")
    b = prefix_decode(d.step, *d.args())
    assert bool(b[3].isnan().all()) and bool(b[1, 2].isnan().all())
    b[3], b[1, 2] = a[3], a[1, 2]
    assert torch.equal(a, b)


def test_strided_prefix_and_caches():
    """The prefix as a view into a longer buffer, own caches with gaps between heads."""
    g, B, hq, hkv, D, P, cap = _gen(11), 3, 4, 2, 256, 77, 24
    big = _rows((hkv, 200, D), g)
    pk = big[:, 50:50 + P]
    big[:, :50], big[:, 50 + P:] = float("nan"), float("nan")
    buf = torch.full((B, hkv, 40, D), float("nan"), dtype=BF, device=DEV)
    kc = buf[:, :, :cap]
    kc.copy_(_rows((B, hkv, cap, D), g))
    vc, pv = _rows((B, hkv, cap, D), g), _rows((hkv, 200, D), g)[:, :P]
    c = Case(B, hq, hkv, D, P, cap, [23, 4, 0], seed=12)
    c.pk, c.pv = pk, pv
    vbuf = torch.zeros_like(buf)
    c.kc, c.vc = kc, vbuf[:, :, :cap]
    c.vc.copy_(vc)
    c.step = PrefixStep.for_caches(pk, kc, hq, scale=D ** -0.5)
    c.run()
    assert bool(buf[:, :, cap:].isnan().all()) and bool((vbuf[:, :, cap:] == 0).all())


def test_prefix_past_32_bits():
    """The second kv head of the prefix 2^31 + 4096 elements behind the first."""
    D, P, hs, g = 128, 90, 2 ** 31 + 4096, _gen(13)
    buf = torch.empty(hs + P * D, dtype=BF, device=DEV)
    pk = torch.as_strided(buf, (2, P, D), (hs, D, 1))
    pk.copy_(_rows((2, P, D), g))
    c = Case(3, 8, 2, D, P, 20, [19, 0, 7], shared=True, seed=14)
    c.pk = c.pv = pk
    c.step = PrefixStep.for_caches(pk, c.kc, 8, kv_shared=True, scale=D ** -0.5)
    c.run()


def test_captured_and_on_another_stream():
    """A captured loop of steps, its replays checked on refilled inputs with eager steps of another
    workspace between them; and a second graph on the same workspace, replayed in turn."""
    c = Case(4, 8, 2, 256, 150, 64, [0, 10, 20, 30], seed=15)
    ws = new_prefix_workspace(c.step, DEV)
    call = PrefixCall(c.step, *c.args(), workspace=ws)
    other = Case(4, 8, 2, 256, 150, 64, [1, 11, 21, 31], seed=16)
    call2 = PrefixCall(other.step, *other.args(), workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    k0, v0 = c.kc.clone(), c.vc.clone()
    call(side)
    torch.cuda.current_stream().wait_stream(side)
    c.check(call.out, k0, v0)
    k0, v0 = other.kc.clone(), other.vc.clone()
    call2()  # its first token
    other.check(call2.out, k0, v0)
    graphs = []
    for f in (call, call2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            f()
        graphs.append(graph)
    g = _gen(17)
    for _ in range(4):
        for case, f, graph in ((c, call, graphs[0]), (other, call2, graphs[1])):
            case.pos += 1
            case.own = [m + 1 for m in case.own]
            for t, gain in ((case.q, 2.5), (case.kn, 1.0), (case.vn, 1.0)):
                t.copy_(_rows(t.shape, g, gain))
            k0, v0 = case.kc.clone(), case.vc.clone()
            graph.replay()
            torch.cuda.synchronize()
            case.check(f.out, k0, v0)


def test_two_samples_of_one_prompt():
    """A prompt through rope and prefill, then two sequences decoded behind it for three tokens: each
    as a decode over its own full cache."""
    hq, hkv, D, P, cap, g = 8, 2, 128, 90, 16, _gen(18)
    inv, _ = rope_frequencies(D, 10000.0, device=DEV)
    x_q, x_k, x_v = _rows((P, hq, D), g), _rows((P, hkv, D), g), _rows((P, hkv, D), g)
    pos = torch.arange(P, dtype=torch.int32, device=DEV)
    pk, pv = torch.empty((hkv, P, D), dtype=BF, device=DEV), x_v.transpose(0, 1).contiguous()
    q, _ = rope(x_q, x_k, pos, inv, k_out=pk.transpose(0, 1))
    prefill(PrefillStep.for_tensors(q.transpose(0, 1), pk, scale=D ** -0.5), q.transpose(0, 1), pk, pv)
    kc, vc = (torch.zeros((2, hkv, cap, D), dtype=BF, device=DEV) for _ in range(2))
    full_k, full_v = (torch.zeros((2, hkv, P + cap, D), dtype=BF, device=DEV) for _ in range(2))
    full_k[:, :, :P], full_v[:, :, :P] = pk, pv
    step, one = PrefixStep.for_caches(pk, kc, hq, scale=D ** -0.5), DecodeStep.for_cache(full_k, hq, scale=D ** -0.5)
    for t in range(3):
        at = torch.full((2,), P + t, dtype=torch.int32, device=DEV)
        qt, kt = rope(_rows((2, hq, D), g), _rows((2, hkv, D), g), at, inv)
        vt = _rows((2, hkv, D), g)
        a = prefix_decode(step, qt, kt, vt, pk, pv, kc, vc, at)
        b = decode_step(one, qt, kt, vt, full_k, full_v, at)
        err = (a.float() - b.float()).abs()
        assert float(err.max()) <= 2e-2 and float(err.mean()) <= 2e-3
    assert torch.equal(kc[:, :, :3], full_k[:, :, P:P + 3]) and torch.equal(vc[:, :, :3], full_v[:, :, P:P + 3])


@pytest.mark.parametrize("split", [0, 64])
@pytest.mark.parametrize("B,hq,hkv,D,P", [(3, 8, 2, 128, 45), (3, 8, 2, 128, 161), (30, 16, 2, 128, 161), (70, 8, 2, 128, 90),
                                          (5, 8, 4, 256, 45), (40, 8, 4, 256, 200), (90, 8, 2, 256, 173),
                                          (3, 8, 2, 512, 45), (3, 8, 2, 512, 201), (40, 8, 2, 512, 173)])
def test_value_that_is_infinite_reaches_its_queries_only(B, hq, hkv, D, P, split):
    """In the prefix's last row and in a sequence's last own row: infinite in its dim for the queries
    that see it (0 x inf from the rows that fill a stage would be NaN), the rest bit for bit."""
    G, own = hq // hkv, [(7 * i + 3) % 50 for i in range(B)]
    c = Case(B, hq, hkv, D, P, 50, own, split_keys=split, seed=20)
    a = c.run()
    c.pv[1, P - 1, 5], c.pv[0, 2, 6], c.vn[2, 0, 9] = float("inf"), float("inf"), -float("inf")
    b = prefix_decode(c.step, *c.args())
    assert bool((b[:, G:2 * G, 5] == float("inf")).all()) and bool((b[:, :G, 6] == float("inf")).all())
    assert bool((b[2, :G, 9] == -float("inf")).all())
    b[:, G:2 * G, 5], b[:, :G, 6], b[2, :G, 9] = a[:, G:2 * G, 5], a[:, :G, 6], a[2, :G, 9]
    assert torch.equal(a, b)


@pytest.mark.parametrize("D,hq", [(128, 8), (256, 4), (512, 8)])
def test_own_caches_past_32_bits(D, hq):
    """The second sequence's own cache 2^31 + 4096 elements behind the first's."""
    hkv, cap, gap, g = 2, 70, 2 ** 31 + 4096, _gen(21)
    buf = torch.empty(gap + hkv * cap * D, dtype=BF, device=DEV)
    kc = torch.as_strided(buf, (2, hkv, cap, D), (gap, cap * D, D, 1))
    c = Case(2, hq, hkv, D, 100, cap, [33, 69], shared=True, seed=22)
    kc.copy_(c.kc)
    c.kc = c.vc = kc
    c.step = PrefixStep.for_caches(c.pk, kc, hq, kv_shared=True, scale=D ** -0.5)
    c.run()


@pytest.mark.parametrize("B,D", [(2, 128), (40, 128), (3, 256), (2, 512), (12, 512)])
def test_two_steps_at_once(B, D):
    """Two layers' steps over one prefix on two streams, each in a workspace of its own, ten times: as one
    after the other."""
    cases = [Case(B, 8, 2, D, 500, 130, [(11 * i + 7 * s) % 130 for i in range(B)], shared=D == 512, seed=23 + s)
             for s in (0, 1)]
    cases[1].pk, cases[1].pv = cases[0].pk, cases[0].pv
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = [[prefix_decode(c.step, *c.args(), stream=s) for c, s in zip(cases, streams)] for _ in range(10)]
    torch.cuda.synchronize()
    for got in outs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("split_rows,split_keys", [(0, 0), (64, 384), (384, 416), (400, 352), (896, 1024), (16, 64)])
@pytest.mark.parametrize("shared,B", [(True, 2), (True, 14), (False, 3), (False, 20)])
def test_runs_of_every_length_at_head_dim_512(shared, B, split_rows, split_keys):
    """Own rows and prefix on both sides of the length up to which runs go in groups of stages, beside
    runs (few query rows), four-wave tiles and eight-wave ones."""
    own = [0, 899, 1, 15, 16, 17, 63, 64, 65, 127, 383, 384, 385, 400, 447, 448, 600, 31, 32, 33][:B]
    Case(B, 8, 1, 512, 1300, 900, own, shared, split_keys, split_rows, seed=25).run()


@pytest.mark.parametrize("D,hq,hkv,P,split_keys", [(128, 32, 8, 700, 64), (256, 32, 16, 500, 32), (512, 32, 4, 640, 64),
                                                   (128, 32, 8, 1200, 32)])
def test_merges_of_many_partials(D, hq, hkv, P, split_keys):
    """10 .. 41 partials a row, of few rows (groups in turn) and of many (a thread each)."""
    for B in (1, 64):
        Case(B, hq, hkv, D, P, 100, _own(B, 100, B), D == 512, split_keys, 48, seed=26 + B).run()


@pytest.mark.parametrize("D,hq,hkv,shared", [(128, 8, 2, False), (256, 4, 2, False), (512, 8, 1, True)])
def test_forced_splits_longer_than_any_row(D, hq, hkv, shared):
    """split_keys and split_rows up to the end of int32: one split of each, also where more own rows
    are visible than the estimate says."""
    for keys, rows in ((2 ** 31 - 32, 0), (0, 2 ** 31 - 16), (2 ** 31 - 32, 2 ** 31 - 16)):
        Case(4, hq, hkv, D, 100, 64, [63, 0, 17, 40], shared, keys, rows, seed=40).run()
        Case(2, hq, hkv, D, 300, 200, [199, 60], shared, keys, rows, max_visible=32, seed=41).run()


@pytest.mark.parametrize("keys", [[32], list(range(32)), list(range(64)), list(range(16, 33)), []])
@pytest.mark.parametrize("B", [1, 3, 9, 33])
@pytest.mark.parametrize("D,hq,hkv,shared", HEADS)
def test_keys_of_minus_infinity(D, hq, hkv, shared, B, keys):
    """Prefix keys whose scores are -inf, alone in a stage or a whole split of them, and a new token that
    is its sequence's one own row: weights of 0, whichever kind of workgroup meets them."""
    P = 33 if keys == [32] else 100
    for split in (0, 32, 64):
        c = Case(B, hq, hkv, D, P, 40, _own(B, 40, 5), shared, split_keys=split, seed=60)
        c.q[..., 3] = c.q[..., 3].abs() + 0.5
        c.pk[:, keys, 3] = -float("inf")
        c.kn[..., 3] = -float("inf")
        k0, v0 = c.kc.clone(), c.vc.clone()
        out = prefix_decode(c.step, *c.args())
        G, vn = hq // hkv, c.kn if shared else c.vn
        dims = torch.arange(D, device=DEV) != 3 if shared else torch.ones(D, dtype=torch.bool, device=DEV)
        for b, m in enumerate(c.own):
            seen = torch.ones((G, P + m + 1), dtype=torch.bool, device=DEV)
            seen[:, keys + [P + m]] = False
            for h in range(hkv):
                k = torch.cat([c.pk[h], k0[b, h, :m], c.kn[b, h][None]])
                v = torch.cat([c.pv[h], v0[b, h, :m], vn[b, h][None]])
                o, bound = attend64(c.q[b, h * G:(h + 1) * G], k, v, seen, D ** -0.5)
                check(out[b, h * G:(h + 1) * G][:, dims], o[:, dims], bound[:, dims], f"sequence {b} kv head {h}")
