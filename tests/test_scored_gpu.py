"""GPU parity of esda_scored_prefill and esda_scored_decode against 64 bits (_attn64.py: the
bound is derived there, per element).

q has a gain of 2.5, so a row's weight sits on a few keys and a key lost or let in shows; keys and
values that no query sees are NaN or infinite, so a masked one that is used shows at once.
"""
import pytest
import torch

from _attn64 import attend64, check
from apertura_amd.decode import DecodeStep, decode_status, decode_step, new_workspace
from apertura_amd.prefill import PrefillStep, prefill
from apertura_amd.rope import rope, rope_frequencies
from apertura_amd.scored import (Score, ScoredDecodeCall, scored_decode, scored_prefill,
                                 scored_prefill_workspace_bytes)

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


def _slopes(hq):
    return 2.0 ** (-6.0 * (torch.arange(hq, device=DEV, dtype=torch.float32) + 1) / hq)


def _seen(step, score, q_doc=None, k_doc=None):
    qa = (step.q_pos0 + torch.arange(step.seq_q, device=DEV))[:, None]
    ka = (step.k_pos0 + torch.arange(step.seq_k, device=DEV))[None]
    m = (ka <= qa) | (ka < score.prefix)
    if step.window:
        m &= ka > qa - step.window
    if q_doc is not None:
        m &= (q_doc[:, None] == k_doc[None]) & (k_doc >= 0)[None]
    return m, (qa - ka).abs().double()


def _check_prefill(step, score, q, k, v, out, q_doc=None, k_doc=None, what=""):
    """Every row of out [Sq, Hq, D]; q [Hq, Sq, D], k / v [Hkv, Sk, D] views."""
    seen, dist = _seen(step, score, q_doc, k_doc)
    G = step.num_q_heads // step.num_kv_heads
    for h in range(step.num_q_heads):
        bias = None if score.slopes is None else score.slopes[h].double() * dist
        o, b = attend64(q[h], k[h // G], v[h // G], seen, step.scale, score.softcap, bias)
        check(out[:, h], o, b, f"{what} head {h}")


def _poison(step, score, k, v, q_doc=None, k_doc=None):
    """NaN and infinities where no query looks."""
    seen, _ = _seen(step, score, q_doc, k_doc)
    dead = (~seen.any(0)).nonzero().flatten()
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=BF, device=DEV)
    k[:, dead] = bad[dead % 3][None, :, None]
    if v is not k:
        v[:, dead] = bad[(dead + 1) % 3][None, :, None]


HEADS = {128: (4, 2, False), 256: (4, 2, False), 512: (8, 1, True)}
SCORES = {"plain": dict(), "cap": dict(softcap=20.0), "bias": dict(biased=True), "both": dict(softcap=8.0, biased=True)}


def _run(D, Sq, past, seed=0, softcap=0.0, biased=False, prefix=0, window=0, docs=None, split=0, heads=None,
         k_first=0, more=0, poison=True):
    """One chunk against 64 bits.  docs: (q_doc, k_doc); k_first: position of the first key kept;
    more: keys past the last query."""
    hq, hkv, shared = heads or HEADS[D]
    g = _gen(seed)
    Sk = past + Sq - k_first + more
    q, k = _rows((hq, Sq, D), g, 2.5), _rows((hkv, Sk, D), g)
    v = k if shared else _rows((hkv, Sk, D), g)
    score = Score(softcap, _slopes(hq) if biased else None, prefix)
    step = PrefillStep(hq, hkv, D, Sq, Sk, past, k_first, window, D ** -0.5, split)
    qd, kd = docs if docs is not None else (None, None)
    if poison:
        _poison(step, score, k, v, qd, kd)
    print(f"\n[case] D={D} Sq={Sq} past={past} {score.softcap} {biased} prefix={prefix} window={window} "
          f"docs={docs is not None} split={split}", flush=True)
    out = torch.full((Sq, hq, D), 9.0, dtype=BF, device=DEV)
    scored_prefill(step, score, q, k, v, qd, kd, out=out)
    torch.cuda.synchronize()
    _check_prefill(step, score, q, k, v, out, qd, kd)
    return out


@pytest.mark.parametrize("name", SCORES)
@pytest.mark.parametrize("Sq,past", [(1, 0), (1, 100), (2, 31), (17, 0), (64, 37), (130, 0), (257, 700), (33, 2050)])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_scores(D, Sq, past, name):
    _run(D, Sq, past, **SCORES[name])


@pytest.mark.parametrize("split", [32, 96, 1024])
@pytest.mark.parametrize("D,heads", [(128, (8, 1, False)), (256, (8, 2, False)), (512, (16, 1, True)), (512, (4, 2, False))])
def test_split_keys(D, heads, split):
    _run(D, 70, 411, softcap=10.0, biased=True, split=split, heads=heads)


@pytest.mark.parametrize("Sq,heads", [(1100, (32, 16, False)), (300, (16, 8, False)), (40, (4, 4, False))])
def test_every_kernel_form_of_head_dim_256(Sq, heads):
    _run(256, Sq, 0, softcap=15.0, window=200, heads=heads)


@pytest.mark.parametrize("D,Sq,heads", [(512, 400, (32, 4, True)), (512, 20, (8, 4, True)), (512, 300, (32, 4, False)),
                                        (512, 12, (4, 4, False)), (128, 700, (32, 8, False))])
def test_every_kernel_form_of_the_other_head_dims(D, Sq, heads):
    _run(D, Sq, 50, softcap=15.0, biased=True, heads=heads)


@pytest.mark.parametrize("prefix", [1, 31, 64, 100, 5000])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_prefix(D, window, prefix):
    _run(D, 150, 0, prefix=prefix, window=window, softcap=30.0)
    _run(D, 20, 90, prefix=prefix, window=window, biased=True, more=13)


@pytest.mark.parametrize("window", [1, 17, 32, 500])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_window(D, window):
    _run(D, 90, 300, window=window, softcap=30.0, biased=True, k_first=max(0, 300 - window + 1))


def _ids(kind, n, g):
    if kind == "runs":       # documents of 1 .. 60 tokens, a padded end
        ids = torch.repeat_interleave(torch.arange(n, device=DEV), torch.randint(1, 61, (n,), device=DEV, generator=g))[:n]
        ids[n - n // 8:] = -1
    elif kind == "shuffled":  # any id at any token, some negative
        ids = torch.randint(-1, 4, (n,), device=DEV, generator=g)
    elif kind == "wide":      # ids to the end of int32, not in order
        ids = torch.randint(0, 3, (n,), device=DEV, generator=g) * (2 ** 30) + 2 ** 30 - 1
    elif kind == "one":
        ids = torch.zeros(n, dtype=torch.int64, device=DEV)
    else:                     # "none": padding only
        ids = torch.full((n,), -1, device=DEV)
    return ids.to(torch.int32)


@pytest.mark.parametrize("kind", ["runs", "shuffled", "wide", "one", "none"])
@pytest.mark.parametrize("n", [1, 50, 333])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_documents(D, n, kind):
    ids = _ids(kind, n, _gen(n))
    out = _run(D, n, 0, docs=(ids, ids), softcap=20.0, biased=True)
    assert bool((out[ids < 0] == 0).all())


@pytest.mark.parametrize("split", [0, 512])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_documents_far_behind(D, split):
    """40 queries whose documents lie in a few places of 6100 keys: most stages hold none of them, and
    more than 64 in a row."""
    k_doc = (torch.arange(6100, device=DEV) // 100).to(torch.int32)
    q_doc = torch.tensor([3] * 11 + [59] * 9 + [60] * 15 + [-1] * 4 + [70], dtype=torch.int32, device=DEV)
    k_doc[4000:4010] = 3
    k_doc[6000:6050] = -1
    _run(D, 40, 6100 - 40, docs=(q_doc, k_doc), split=split, biased=True)


def test_documents_over_more_keys_than_are_summed_up():
    """140,000 keys in one split: the stages past the first 131,072 keys are computed with their mask."""
    n = 140000
    k_doc = (torch.arange(n, device=DEV) // 5000).to(torch.int32)
    q_doc = torch.tensor([0, 26, 27, 27, -1, 13], dtype=torch.int32, device=DEV)
    _run(128, 6, n - 6, docs=(q_doc, k_doc), split=1 << 20, biased=True, heads=(2, 1, False))


@pytest.mark.parametrize("D", [128, 256, 512])
def test_documents_with_prefix_and_window(D):
    ids = _ids("runs", 200, _gen(3))
    _run(D, 200, 0, docs=(ids, ids), prefix=120, window=30)


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("split", [0, 32])
def test_rows_that_see_nothing(D, split):
    """Keys after every query, keys behind every window, and both with some rows that see."""
    hq, hkv, shared = HEADS[D]
    g = _gen(5)
    q, k = _rows((hq, 50, D), g), _rows((hkv, 70, D), g)
    v = k if shared else _rows((hkv, 70, D), g)
    for q0, k0, window in ((0, 50, 0), (0, 500, 0), (1000, 0, 100), (0, 20, 0), (60, 0, 25), (2 ** 31 - 51, 0, 7)):
        step = PrefillStep(hq, hkv, D, 50, 70, q0, k0, window, 1.0, split)
        out = torch.full((50, hq, D), 9.0, dtype=BF, device=DEV)
        scored_prefill(step, Score(), q, k, v, out=out)
        seen, _ = _seen(step, Score())
        assert bool((out[~seen.any(1)] == 0).all())
        _check_prefill(step, Score(), q, k, v, out)


@pytest.mark.parametrize("split", [0, 64])
@pytest.mark.parametrize("D,heads", [(128, None), (256, None), (256, (32, 16, False)), (512, None), (512, (4, 2, False))])
def test_values_that_are_not_finite_reach_only_their_rows(D, heads, split):
    """An infinite and a NaN value in one document: every other document's rows as without them, its
    own rows NaN or infinite in those dims as the formula gives."""
    hq, hkv, shared = heads or HEADS[D]
    n, g = 160, _gen(6)
    ids = (torch.arange(n, device=DEV) // 23).to(torch.int32)
    q, k, v = _rows((hq, n, D), g), _rows((hkv, n, D), g), _rows((hkv, n, D), g)
    if shared:
        v = k
    step = PrefillStep(hq, hkv, D, n, n, scale=D ** -0.5, split_keys=split)
    clean = scored_prefill(step, Score(softcap=9.0), q, k, v, ids, ids)
    v2 = v.clone()
    k2 = v2 if shared else k
    v2[:, 50, 7], v2[:, 51, 9], v2[0, 120, D - 1] = float("inf"), float("nan"), -float("inf")
    out = scored_prefill(step, Score(softcap=9.0), q, k2, v2, ids, ids)
    touched = ((ids == 2) & (torch.arange(n, device=DEV) >= 50)) | ((ids == 5) & (torch.arange(n, device=DEV) >= 120))
    for h in range(hq):
        seen, _ = _seen(step, Score(), ids, ids)
        o, b = attend64(q[h], k[h // (hq // hkv)], v[h // (hq // hkv)], seen, step.scale, 9.0)
        check(out[~touched, h], o[~touched], b[~touched], f"head {h}")
    if not shared:
        rows = out[touched].float()
        inf7 = torch.arange(n, device=DEV)[touched] < 115  # the rows of document 2
        assert bool((rows[inf7][..., 7] == float("inf")).all())
        assert bool(rows[inf7 & (torch.arange(n, device=DEV)[touched] >= 51)][..., 9].isnan().all())
        assert bool((rows[~inf7][:, :hq // hkv, D - 1] == -float("inf")).all())
        assert bool(rows[..., 20].isfinite().all())


def test_a_query_that_is_not_finite_is_its_own():
    D, n, g = 128, 40, _gen(7)
    q, k, v = _rows((4, n, D), g), _rows((2, n, D), g), _rows((2, n, D), g)
    step = PrefillStep(4, 2, D, n, n, scale=D ** -0.5)
    a = scored_prefill(step, Score(softcap=5.0), q, k, v)
    q[1, 13, 3] = float("nan")
    b = scored_prefill(step, Score(softcap=5.0), q, k, v)
    assert bool(b[13, 1].isnan().all())
    b[13, 1] = a[13, 1]
    assert torch.equal(a, b)


def test_large_scores_saturate():
    """Scores far past the cap: tanh is 1 to the last bit, equal weights where every score is."""
    D, n, g = 128, 64, _gen(8)
    q, k, v = _rows((4, n, D), g, 60.0), _rows((2, n, D), g, 60.0), _rows((2, n, D), g)
    step = PrefillStep(4, 2, D, n, n, scale=1.0)
    for cap in (0.5, 30.0, 1000.0):
        out = scored_prefill(step, Score(softcap=cap), q, k, v)
        seen, _ = _seen(step, Score())
        for h in range(4):
            o, b = attend64(q[h], k[h // 2], v[h // 2], seen, 1.0, cap)
            check(out[:, h], o, b, f"cap {cap} head {h}")


def test_far_positions():
    """Positions near 2^31, and distances past 2^24 (their bias is exact to 2^-24 of itself, inside
    the bound's 2^-20)."""
    D, g = 128, _gen(9)
    q, k, v = _rows((4, 30, D), g), _rows((2, 30, D), g), _rows((2, 30, D), g)
    for q0, k0 in ((2 ** 31 - 200, 2 ** 31 - 190), (2 ** 31 - 200, 5), (5, 2 ** 31 - 200)):
        step = PrefillStep(4, 2, D, 30, 30, q0, k0, 0, D ** -0.5)
        score = Score(slopes=torch.full((4,), 2.0 ** -24, device=DEV), prefix=2 ** 31 - 1)
        out = scored_prefill(step, score, q, k, v)
        _check_prefill(step, score, q, k, v, out)


@pytest.mark.parametrize("D", [128, 256, 512])
def test_plain_score_and_the_plain_call(D):
    """They add the keys in opposite orders; each is within the bound of the exact values."""
    hq, hkv, shared = HEADS[D]
    g = _gen(10)
    q, k = _rows((hq, 77, D), g), _rows((hkv, 277, D), g)
    v = k if shared else _rows((hkv, 277, D), g)
    step = PrefillStep(hq, hkv, D, 77, 277, 200, 0, 0, D ** -0.5)
    _check_prefill(step, Score(), q, k, v, scored_prefill(step, Score(), q, k, v))
    _check_prefill(step, Score(), q, k, v, prefill(step, q, k, v))


def test_strides_and_memory_around():
    """q as a [Sq, Hq, D] buffer's transpose, k and v inside a longer cache, out with gaps."""
    hq, hkv, D, n, cap, g = 4, 2, 256, 45, 200, _gen(11)
    qb, kc, vc = _rows((n, hq, D), g, 2.5), _rows((hkv, cap, D), g), _rows((hkv, cap, D), g)
    kc[:, 60 + n:], vc[:, 60 + n:] = float("nan"), float("nan")  # behind the last key
    kc[:, :20], vc[:, :20] = float("inf"), float("inf")          # before the first
    q, k, v = qb.transpose(0, 1), kc[:, 20:60 + n], vc[:, 20:60 + n]
    buf = torch.full((n, hq + 1, D + 8), 3.0, dtype=BF, device=DEV)
    out = buf[:, :hq, :D]
    step = PrefillStep.for_tensors(q, k, out, q_pos0=40, k_pos0=0, scale=D ** -0.5)
    score = Score(softcap=12.0, slopes=_slopes(hq))
    scored_prefill(step, score, q, k, v, out=out)
    _check_prefill(step, score, q, k, v, out)
    out.fill_(3.0)
    assert bool((buf == 3.0).all())


def test_keys_past_32_bits():
    """A second kv head 2^31 + 4096 elements behind the first."""
    D, n, hs, g = 128, 40, 2 ** 31 + 4096, _gen(12)
    buf = torch.empty(hs + n * D, dtype=BF, device=DEV)
    k = torch.as_strided(buf, (2, n, D), (hs, D, 1))
    k.copy_(_rows((2, n, D), g))
    q = _rows((4, n, D), g, 2.5)
    step = PrefillStep.for_tensors(q, k, scale=D ** -0.5)
    ids = _ids("runs", n, g)
    out = scored_prefill(step, Score(softcap=9.0), q, k, k, ids, ids)
    _check_prefill(step, Score(softcap=9.0), q, k, k, out, ids, ids)


def test_prefill_captured_and_on_another_stream():
    hq, hkv, D, Sq, Sk, g = 8, 1, 512, 40, 500, _gen(13)
    q, k = _rows((hq, Sq, D), g, 2.5), _rows((hkv, Sk, D), g)
    ids = _ids("runs", Sk, g)
    qd = ids[-Sq:].clone()
    score = Score(softcap=20.0, slopes=_slopes(hq))
    step = PrefillStep(hq, hkv, D, Sq, Sk, Sk - Sq, 0, 0, D ** -0.5, 96)
    ws = torch.empty(scored_prefill_workspace_bytes(step, score), dtype=torch.uint8, device=DEV)
    out = torch.empty((Sq, hq, D), dtype=BF, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    scored_prefill(step, score, q, k, k, qd, ids, out=out, workspace=ws, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    _check_prefill(step, score, q, k, k, out, qd, ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        scored_prefill(step, score, q, k, k, qd, ids, out=out, workspace=ws)
    for i in range(4):
        q.copy_(_rows((hq, Sq, D), g, 2.5))
        k.copy_(_rows((hkv, Sk, D), g))
        ids.copy_(_ids("runs", Sk, g))
        qd.copy_(ids[-Sq:])
        want = scored_prefill(step, score, q, k, k, qd, ids)  # its own workspace
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, want)
        _check_prefill(step, score, q, k, k, out, qd, ids)


# --------------------------------------------------------------------------------- decode

def _check_decode(step, score, q, kc, vc, kn, vn, pos, out, base=None):
    """Caches as they were before the step."""
    G = step.num_q_heads // step.num_kv_heads
    for b, p in enumerate(pos):
        lo = max(0, p - step.window + 1) if step.window else 0
        if base is not None:
            lo = max(lo, base[b])
        at = torch.arange(lo, p + 1, device=DEV)
        rows = at % step.cap if step.ring else at - (base[b] if base is not None else 0)
        for h in range(step.num_q_heads):
            k, v = kc[b, h // G, rows].clone(), vc[b, h // G, rows].clone()
            k[-1], v[-1] = kn[b, h // G], vn[b, h // G]
            bias = None if score.slopes is None else score.slopes[h].double() * (p - at)[None].double()
            o, bound = attend64(q[b, h][None], k, v, torch.ones((1, len(at)), dtype=torch.bool, device=DEV), step.scale,
                                score.softcap, bias)
            check(out[b, h][None], o, bound, f"sequence {b} head {h}")


def _decode(B, hq, hkv, D, cap, pos, shared=False, softcap=0.0, biased=False, window=0, ring=False, base=None, split=0,
            seed=0):
    g = _gen(seed)
    q, kc, kn = _rows((B, hq, D), g, 2.5), _rows((B, hkv, cap, D), g), _rows((B, hkv, D), g)
    vc, vn = (kc, kn) if shared else (_rows((B, hkv, cap, D), g), _rows((B, hkv, D), g))
    step = DecodeStep(B, hq, hkv, D, cap, window, ring, shared, D ** -0.5, split_rows=split)
    score = Score(softcap, _slopes(hq) if biased else None)
    k0, v0 = kc.clone(), vc.clone()
    print(f"\n[case] decode B={B} D={D} cap={cap} pos={pos} cap={softcap} biased={biased} ring={ring}", flush=True)
    pt = torch.tensor(pos, dtype=torch.int32, device=DEV)
    bt = None if base is None else torch.tensor(base, dtype=torch.int32, device=DEV)
    out = scored_decode(step, score, q, kn, None if shared else vn, kc, vc, pt, bt)
    torch.cuda.synchronize()
    _check_decode(step, score, q, k0, v0, kn, vn, pos, out, base)
    for c, c0, new in ((kc, k0, kn), (vc, v0, vn)):
        for b, p in enumerate(pos):
            c0[b, :, p % cap if ring else p - (base[b] if base else 0)] = new[b]
        assert torch.equal(c.view(torch.int16), c0.view(torch.int16))
    return out


SHAPES = {128: (8, 2, False), 256: (4, 2, False), 512: (8, 1, True)}


@pytest.mark.parametrize("name", SCORES)
@pytest.mark.parametrize("pos", [0, 1, 15, 16, 100, 700])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_decode_one_sequence(D, pos, name):
    hq, hkv, shared = SHAPES[D]
    _decode(1, hq, hkv, D, 701, [pos], shared, **SCORES[name])


@pytest.mark.parametrize("name", ["cap", "both"])
@pytest.mark.parametrize("D,heads", [(128, (32, 8, False)), (256, (32, 16, False)), (512, (32, 4, True)),
                                     (512, (16, 1, False)), (256, (5, 5, True)), (128, (16, 1, True))])
def test_decode_ragged_batch(D, heads, name):
    hq, hkv, shared = heads
    _decode(5, hq, hkv, D, 400, [0, 399, 17, 250, 31], shared, **SCORES[name])


@pytest.mark.parametrize("pos", [[63], [64], [1000, 63, 500]])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_decode_ring(D, pos):
    hq, hkv, shared = SHAPES[D]
    _decode(len(pos), hq, hkv, D, 64, pos, shared, 12.0, True, window=64, ring=True)
    _decode(len(pos), hq, hkv, D, 64, pos, shared, 0.0, True, window=40, ring=True)


def test_decode_window_and_row_base():
    _decode(3, 4, 2, 256, 128, [200, 130, 127], False, 7.0, True, window=50, base=[100, 10, 0])
    _decode(1, 4, 2, 128, 300, [260], False, 7.0, True, split=32)
    # packed kv heads (one split per pair of a large batch)
    _decode(64, 16, 16, 128, 40, [i % 40 for i in range(64)], False, 7.0, True, window=33, ring=False, split=64)
    _decode(160, 8, 8, 128, 16, [50 + i for i in range(160)], False, 7.0, True, window=16, ring=True)


def test_decode_skips_what_is_outside_its_cache():
    g = _gen(20)
    B, hq, hkv, D, cap = 4, 8, 2, 128, 32
    q, kc, vc = _rows((B, hq, D), g), _rows((B, hkv, cap, D), g), _rows((B, hkv, cap, D), g)
    kn, vn = _rows((B, hkv, D), g), _rows((B, hkv, D), g)
    step = DecodeStep(B, hq, hkv, D, cap, scale=0.1)
    pos = torch.tensor([3, 32, -1, 31], dtype=torch.int32, device=DEV)
    ws, out, k0 = new_workspace(step, DEV), torch.full((B, hq, D), 5.0, dtype=BF, device=DEV), kc.clone()
    scored_decode(step, Score(softcap=3.0), q, kn, vn, kc, vc, pos, out=out, workspace=ws)
    assert decode_status(step, ws) == 2
    assert bool((out[1:3] == 5.0).all()) and bool((out[0] != 5.0).any())
    k0[0, :, 3], k0[3, :, 31] = kn[0], kn[3]
    assert torch.equal(kc, k0)


@pytest.mark.parametrize("D", [128, 256, 512])
def test_plain_score_and_the_plain_step(D):
    """They may split and add the rows differently; each is within the bound of the exact values."""
    hq, hkv, shared = SHAPES[D]
    g = _gen(21)
    q, kc, kn = _rows((3, hq, D), g), _rows((3, hkv, 300, D), g), _rows((3, hkv, D), g)
    vc, vn = (kc, None) if shared else (_rows((3, hkv, 300, D), g), _rows((3, hkv, D), g))
    step = DecodeStep(3, hq, hkv, D, 300, kv_shared=shared, scale=D ** -0.5)
    where = [299, 5, 100]
    pos = torch.tensor(where, dtype=torch.int32, device=DEV)
    for f in (lambda: scored_decode(step, Score(), q, kn, vn, kc, vc, pos),
              lambda: decode_step(step, q, kn, vn, kc, vc, pos)):
        k0, v0 = kc.clone(), vc.clone()
        _check_decode(step, Score(), q, k0, v0, kn, kn if shared else vn, where, f())


def test_decode_captured_and_on_another_stream():
    g = _gen(22)
    B, hq, hkv, D, cap = 3, 8, 2, 256, 200
    q, kc, vc = _rows((B, hq, D), g, 2.5), _rows((B, hkv, cap, D), g), _rows((B, hkv, cap, D), g)
    kn, vn = _rows((B, hkv, D), g), _rows((B, hkv, D), g)
    pos = torch.tensor([5, 100, 60], dtype=torch.int32, device=DEV)
    score, step = Score(10.0, _slopes(hq)), DecodeStep(B, hq, hkv, D, cap, scale=D ** -0.5)
    call = ScoredDecodeCall(step, score, q, kn, vn, kc, vc, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call(side)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(5):
        pos += 1
        for t, gain in ((q, 2.5), (kn, 1.0), (vn, 1.0)):
            t.copy_(_rows(t.shape, g, gain))
        k0, v0 = kc.clone(), vc.clone()
        graph.replay()
        torch.cuda.synchronize()
        _check_decode(step, score, q, k0, v0, kn, vn, pos.tolist(), call.out)


# ----------------------------------------------------------------- a layer's run together

def test_rope_prefill_and_decode_of_a_capped_layer():
    """A prompt with a prefix mask through rope into a cache, attended with capped scores, then three
    tokens decoded: each as the last row of a chunk over the whole sequence."""
    hq, hkv, D, n, cap, g = 8, 2, 256, 70, 96, _gen(23)
    inv, _ = rope_frequencies(128, 10000.0, device=DEV)
    score = Score(softcap=15.0, prefix=20)
    kc, vc = (torch.zeros((1, hkv, cap, D), dtype=BF, device=DEV) for _ in range(2))
    x_q, x_k, x_v = _rows((n + 3, hq, D), g, 2.5), _rows((n + 3, hkv, D), g), _rows((n + 3, hkv, D), g)
    pos = torch.arange(n + 3, dtype=torch.int32, device=DEV)
    q, k_all = rope(x_q, x_k, pos, inv)
    rope(None, x_k[:n], pos[:n], inv, k_out=kc[0, :, :n].transpose(0, 1))
    assert torch.equal(kc[0, :, :n].transpose(0, 1), k_all[:n])
    vc[0, :, :n] = x_v[:n].transpose(0, 1)
    step = PrefillStep.for_tensors(q[:n].transpose(0, 1), kc[0, :, :n], scale=D ** -0.5)
    out = scored_prefill(step, score, q[:n].transpose(0, 1), kc[0, :, :n], vc[0, :, :n])
    _check_prefill(step, score, q[:n].transpose(0, 1), kc[0, :, :n], vc[0, :, :n], out)
    dstep = DecodeStep.for_cache(kc, hq, scale=D ** -0.5)
    for t in range(n, n + 3):
        p = pos[t:t + 1]
        qt, kt = rope(x_q[t:t + 1], x_k[t:t + 1], p, inv)
        k0, v0 = kc.clone(), vc.clone()
        got = scored_decode(dstep, score, qt, kt, x_v[t:t + 1], kc, vc, p)
        _check_decode(dstep, score, qt, k0, v0, kt, x_v[t:t + 1], [t], got)


@pytest.mark.parametrize("B,hq,hkv,D,cap,ring", [(3, 8, 2, 128, 150, False), (3, 8, 4, 256, 150, False),
                                                 (3, 4, 2, 512, 150, False), (1, 4, 2, 256, 700, False),
                                                 (2, 4, 2, 512, 64, True), (64, 32, 16, 256, 24, True)])
def test_decode_value_that_is_infinite_reaches_its_queries_only(B, hq, hkv, D, cap, ring):
    """An infinite value in the last visible row (a stage's rows past it must not add 0 x inf) and one
    before: infinite in its dim for the queries of its kv head, every other element bit for bit."""
    g, G = _gen(30), hq // hkv
    q, kc, vc = _rows((B, hq, D), g), _rows((B, hkv, cap, D), g), _rows((B, hkv, cap, D), g)
    kn, vn = _rows((B, hkv, D), g), _rows((B, hkv, D), g)
    pos = [(i * 37 + 20) % (5 * cap if ring else cap) for i in range(B)]
    step = DecodeStep(B, hq, hkv, D, cap, window=cap if ring else 0, ring=ring, scale=D ** -0.5)
    posd = torch.tensor(pos, dtype=torch.int32, device=DEV)
    score = Score(20.0, _slopes(hq) * 2.0 ** -6)
    a = scored_decode(step, score, q, kn, vn, kc, vc, posd)
    vn[0, 0, 7], vc[0, hkv - 1, 3, 11] = float("inf"), -float("inf")
    b = scored_decode(step, score, q, kn, vn, kc, vc, posd)
    assert bool(a.isfinite().all())
    assert bool((b[0, :G, 7] == float("inf")).all()) and bool((b[0, hq - G:, 11] == -float("inf")).all())
    b[0, :G, 7], b[0, hq - G:, 11] = a[0, :G, 7], a[0, hq - G:, 11]
    assert torch.equal(a, b)


@pytest.mark.parametrize("D", [128, 256, 512])
def test_decode_cache_past_32_bits(D):
    """The second sequence's cache 2^31 + 4096 elements behind the first's."""
    B, hq, hkv, cap, gap, g = 2, 8, 2, 300, 2 ** 31 + 4096, _gen(31)
    buf = torch.empty(gap + hkv * cap * D, dtype=BF, device=DEV)
    kc = torch.as_strided(buf, (B, hkv, cap, D), (gap, cap * D, D, 1))
    kc.copy_(_rows((B, hkv, cap, D), g))
    q, kn, pos = _rows((B, hq, D), g, 2.5), _rows((B, hkv, D), g), [260, 299]
    step = DecodeStep.for_cache(kc, hq, kv_shared=True, scale=D ** -0.5)
    score, k0 = Score(9.0, _slopes(hq)), kc.clone()
    out = scored_decode(step, score, q, kn, None, kc, kc, torch.tensor(pos, dtype=torch.int32, device=DEV))
    _check_decode(step, score, q, k0, k0, kn, kn, pos, out)
    k0[0, :, 260], k0[1, :, 299] = kn[0], kn[1]
    assert torch.equal(kc, k0)


def test_calls_at_once_on_two_streams():
    """A prefill chunk in splits and a decode step, each on a stream and in a workspace of its own, over
    one cache's rows: ten rounds of both at once give what they give one after the other."""
    hq, hkv, D, n, g = 8, 2, 256, 600, _gen(32)
    q, k, v = _rows((hq, 40, D), g, 2.5), _rows((hkv, n, D), g), _rows((hkv, n, D), g)
    step, score = PrefillStep(hq, hkv, D, 40, n, n - 40, 0, 0, D ** -0.5, 128), Score(20.0, _slopes(hq))
    kc, vc, qd, kn, vn = (_rows(s, g) for s in ((3, hkv, 500, D), (3, hkv, 500, D), (3, hq, D), (3, hkv, D), (3, hkv, D)))
    dstep = DecodeStep(3, hq, hkv, D, 500, scale=D ** -0.5)
    pos = torch.tensor([499, 120, 3], dtype=torch.int32, device=DEV)
    want = scored_prefill(step, score, q, k, v)
    dwant = scored_decode(dstep, score, qd, kn, vn, kc, vc, pos)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream())
    outs = [(scored_prefill(step, score, q, k, v, stream=a), scored_decode(dstep, score, qd, kn, vn, kc, vc, pos, stream=b))
            for _ in range(10)]
    torch.cuda.synchronize()
    for x, y in outs:
        assert torch.equal(x, want) and torch.equal(y, dwant)


@pytest.mark.parametrize("D", [128, 256, 512])
def test_a_forced_split_longer_than_any_tile_s_keys(D):
    """split_keys at the end of int32 under a window, whose later tiles begin past key 0: every row as
    unsplit."""
    hq, hkv, shared = HEADS[D]
    _run(D, 400, 300, softcap=20.0, biased=True, window=64, split=2 ** 31 - 32)
    _run(D, 200, 0, window=33, prefix=70, split=2 ** 31 - 64)
    g = _gen(33)
    q, k = _rows((hq, 400, D), g, 2.5), _rows((hkv, 700, D), g)
    v = k if shared else _rows((hkv, 700, D), g)
    step = PrefillStep(hq, hkv, D, 400, 700, 300, 0, 64, D ** -0.5, 2 ** 31 - 32)
    out = torch.full((400, hq, D), 9.0, dtype=BF, device=DEV)
    _check_prefill(step, Score(), q, k, v, prefill(step, q, k, v, out=out))


# Caps far above the scores, and around them.  Up to 256 the capped score may be off by 2^-21 of the cap
# (an exponential and a reciprocal of half a step or one each, 2^-22 of a tanh), past it by 2^-21 of
# itself (the bound's 2^-20 holds that).
CAPS = [60.0, 256.0, 256.5, 1e3, 1e4, 1e5, 1e6, 1e8, 1e20, 1e30]


def _score_err(cap):
    return 2.0 ** -21 * cap if cap <= 256 else 0.0


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("gain", [2.5, 400.0])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_caps_of_any_size(D, gain, cap):
    hq, hkv, shared = HEADS[D]
    for Sq, past, split, biased in ((70, 0, 0, False), (33, 300, 64, True)):
        g = _gen(50)
        q, k = _rows((hq, Sq, D), g, gain), _rows((hkv, past + Sq, D), g)
        v = k if shared else _rows((hkv, past + Sq, D), g)
        score = Score(cap, _slopes(hq) if biased else None)
        step = PrefillStep(hq, hkv, D, Sq, past + Sq, past, 0, 0, D ** -0.5, split)
        out = scored_prefill(step, score, q, k, v)
        seen, dist = _seen(step, score)
        for h in range(hq):
            bias = score.slopes[h].double() * dist if biased else None
            o, b = attend64(q[h], k[h // (hq // hkv)], v[h // (hq // hkv)], seen, step.scale, cap, bias, _score_err(cap))
            check(out[:, h], o, b, f"cap {cap} head {h}")


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("gain", [2.5, 400.0])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_decode_caps_of_any_size(D, gain, cap):
    hq, hkv, shared = SHAPES[D]
    g, n = _gen(51), 333
    for biased in (False, True):
        q, kc, kn = _rows((1, hq, D), g, gain), _rows((1, hkv, n, D), g), _rows((1, hkv, D), g)
        vc, vn = (kc, kn) if shared else (_rows((1, hkv, n, D), g), _rows((1, hkv, D), g))
        step = DecodeStep(1, hq, hkv, D, n, kv_shared=shared, scale=D ** -0.5)
        score = Score(cap, _slopes(hq) if biased else None)
        out = scored_decode(step, score, q, kn, None if shared else vn, kc, vc,
                            torch.tensor([n - 1], dtype=torch.int32, device=DEV))
        dist = torch.arange(n - 1, -1, -1, device=DEV).double()[None]  # (the new row is in the cache now)
        for h in range(hq):
            bias = score.slopes[h].double() * dist if biased else None
            seen = torch.ones((1, n), dtype=torch.bool, device=DEV)
            o, b = attend64(q[0, h][None], kc[0, h // (hq // hkv)], vc[0, h // (hq // hkv)], seen, step.scale, cap, bias,
                            _score_err(cap))
            check(out[0, h][None], o, b, f"cap {cap} head {h}")


@pytest.mark.parametrize("split", [0, 64])
@pytest.mark.parametrize("cap", [0.0, 20.0, 1e7])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_rows_that_see_an_infinite_value_keep_their_other_dims(D, cap, split):
    """An infinite value of one dim: that dim infinite from its key on, the others of those rows as
    without it."""
    hq, hkv, n, g = 4, 2, 150, _gen(52)
    q, k, v = _rows((hq, n, D), g, 2.5), _rows((hkv, n, D), g), _rows((hkv, n, D), g)
    v[:, 60, 5] = float("inf")
    score = Score(cap, _slopes(hq))
    step = PrefillStep(hq, hkv, D, n, n, scale=D ** -0.5, split_keys=split)
    out = scored_prefill(step, score, q, k, v)
    assert bool((out[60:, :, 5] == float("inf")).all()) and bool(out[:60].isfinite().all())
    seen, dist = _seen(step, score)
    v[:, 60, 5] = 0.0
    for h in range(hq):
        o, b = attend64(q[h], k[h // 2], v[h // 2], seen, step.scale, cap, score.slopes[h].double() * dist, _score_err(cap))
        rest = torch.arange(D, device=DEV) != 5
        check(out[:, h][:, rest], o[:, rest], b[:, rest], f"head {h}")


# ------------------------------------------------------------ keys whose score is -inf: a weight of 0

@pytest.mark.parametrize("rows,split", [([20], 16), ([16], 16), (list(range(16)), 0), (list(range(32)), 0), (list(range(4, 40)), 16),
                                        (list(range(150)), 16)])
@pytest.mark.parametrize("D,heads", [(128, (8, 2, False)), (256, (4, 2, False)), (512, (8, 1, True)), (512, (4, 2, False))])
@pytest.mark.parametrize("scored", [True, False])
def test_decode_keys_of_minus_infinity(D, heads, rows, split, scored):
    """Whole stages and splits of them, first, last or alone: the row over the other keys (one K = V
    buffer: 0 x inf in the infinite dim alone)."""
    hq, hkv, shared = heads
    g = _gen(60)
    for n in ((21, 160) if rows == [20] else (17, 160) if rows == [16] else (160,)):
        q, kc, kn = _rows((2, hq, D), g, 2.5), _rows((2, hkv, n, D), g), _rows((2, hkv, D), g)
        vc, vn = (kc, None) if shared else (_rows((2, hkv, n, D), g), _rows((2, hkv, D), g))
        q[..., 3] = q[..., 3].abs() + 0.5
        for r in rows:
            if r < n - 1:
                kc[:, :, r, 3] = -float("inf")
            else:
                kn[..., 3] = -float("inf")
        step = DecodeStep(2, hq, hkv, D, n, kv_shared=shared, scale=D ** -0.5, split_rows=split)
        pos = torch.tensor([n - 1, n - 1], dtype=torch.int32, device=DEV)
        if scored:
            out = scored_decode(step, Score(), q, kn, vn, kc, vc, pos)
        else:
            out = decode_step(step, q, kn, vn, kc, vc, pos)
        seen = torch.ones((1, n), dtype=torch.bool, device=DEV)
        seen[:, [r for r in rows if r < n]] = False
        dims = torch.arange(D, device=DEV) != 3 if shared else torch.ones(D, dtype=torch.bool, device=DEV)
        for b in range(2):
            for h in range(hq):
                o, bound = attend64(q[b, h][None], kc[b, h // (hq // hkv)], vc[b, h // (hq // hkv)], seen, step.scale)
                check(out[b, h][None][:, dims], o[:, dims], bound[:, dims], f"n {n} sequence {b} head {h}")


@pytest.mark.parametrize("D", [128, 256, 512])
def test_out_beside_its_inputs_in_one_buffer(D):
    """Packed rows that hold q and out side by side, and an out between the kv heads of one arena: memory
    shared, elements not."""
    hq, hkv, n, g = 4, 2, 50, _gen(70)
    rows = torch.zeros((n, 2 * hq, D), dtype=BF, device=DEV)
    rows[:, :hq] = _rows((n, hq, D), g, 2.5)
    k, v = _rows((hkv, n, D), g), _rows((hkv, n, D), g)
    q, out, score = rows[:, :hq].transpose(0, 1), rows[:, hq:], Score(20.0, _slopes(hq))
    step = PrefillStep.for_tensors(q, k, out, scale=D ** -0.5)
    scored_prefill(step, score, q, k, v, out=out)
    _check_prefill(step, score, q, k, v, out)
    arena = torch.zeros(3 * n * D + n * hq * D, dtype=BF, device=DEV)
    ka = torch.as_strided(arena, (hkv, n, D), ((1 + hq) * n * D, D, 1))
    ka.copy_(k)
    out = arena[n * D:n * D + n * hq * D].view(n, hq, D)
    step = PrefillStep.for_tensors(q, ka, out, scale=D ** -0.5)
    scored_prefill(step, score, q, ka, ka, out=out)
    _check_prefill(step, score, q, ka, ka, out)
    assert torch.equal(ka, k)
