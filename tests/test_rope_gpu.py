"""GPU parity of esda_rope against the rotation in 64 bits.

Tolerance: one rounding to bf16 (half a step, 2^-8 of the value) plus the fp32 arithmetic
before it: cos and sin within 2^-23 (their polynomials and the rounding of the reduced angle),
the two products and their sum within 2^-23 of |x0| + |x1| together, so 2^-21 f (|x0| + |x1|)
covers both.
"""
import pytest
import torch

from apertura_amd.rope import RopeCall, RopeScaling, rope, rope_frequencies

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _rows(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(BF).cuda()


def _pairs(r, interleaved):
    i = torch.arange(r // 2, device="cuda")
    return (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)


def _ref(x, pos, inv, interleaved=False, inverse=False, factor=1.0):
    """(rotated rows, tolerance), float64."""
    r = 2 * inv.numel()
    i, j = _pairs(r, interleaved)
    a = pos.double()[:, None, None] * inv.double()
    c, s = factor * a.cos(), factor * a.sin() * (-1.0 if inverse else 1.0)
    y = x.double()
    x0, x1 = y[..., i].clone(), y[..., j].clone()
    tol = torch.zeros_like(y)
    y[..., i], y[..., j] = x0 * c - x1 * s, x1 * c + x0 * s
    slack = 2.0 ** -21 * abs(factor) * (x0.abs() + x1.abs())
    tol[..., i] = tol[..., j] = slack
    tol += y.abs() * 2.0 ** -8
    tol[..., r:] = 0.0  # copied
    return y, tol


def _check(x, got, pos, inv, **kw):
    want, tol = _ref(x, pos, inv, **kw)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err - tol).max()):.3e} past its tolerance"


def _pos(T, seed, far=131072):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-far, far, (T,), generator=g, dtype=torch.int32).cuda()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (128, 40), (128, 2), (256, 256), (256, 64), (256, 6),
                                   (512, 512), (512, 128), (512, 510)])
@pytest.mark.parametrize("T", [1, 3, 130])
def test_rows_against_64_bits(T, D, rot, interleaved):
    q, k, pos = _rows((T, 8, D), 1), _rows((T, 2, D), 2), _pos(T, 3)
    inv, _ = rope_frequencies(rot, 10000.0, device="cuda")
    qo, ko = rope(q, k, pos, inv, interleaved=interleaved)
    _check(q, qo, pos, inv, interleaved=interleaved)
    _check(k, ko, pos, inv, interleaved=interleaved)


@pytest.mark.parametrize("hq,hk", [(1, 0), (0, 1), (32, 16), (5, 3), (64, 8)])
@pytest.mark.parametrize("T", [1, 17, 1031])
def test_head_counts(T, hq, hk):
    q = _rows((T, hq, 256), 4) if hq else None
    k = _rows((T, hk, 256), 5) if hk else None
    pos = _pos(T, 6)
    inv, f = rope_frequencies(128, 1e6, RopeScaling("yarn", 4.0, 4096, 1.0, 32.0), device="cuda")
    qo, ko = rope(q, k, pos, inv, attn_factor=f)
    for x, y in ((q, qo), (k, ko)):
        assert (x is None) == (y is None)
        if x is not None:
            _check(x, y, pos, inv, factor=f)


def test_far_positions():
    """Positions to both ends of int32: the angle's product is off by 2^-22 at most there, four
    times the slack's share for cos and sin."""
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, 2 ** 24 + 1, -(2 ** 24) - 1, 0], dtype=torch.int32).cuda()
    q = _rows((6, 4, 128), 7)
    inv, _ = rope_frequencies(128, 10000.0, device="cuda")
    qo, _ = rope(q, None, pos, inv)
    i, j = _pairs(128, False)
    want, tol = _ref(q, pos, inv)
    more = 2.0 ** -22 * (q.double()[..., i].abs() + q.double()[..., j].abs())
    tol[..., i] += more
    tol[..., j] += more
    assert bool(((qo.double() - want).abs() <= tol).all())


def test_zero_frequencies_leave_their_pairs():
    q, pos = _rows((9, 4, 512), 8), _pos(9, 9)
    inv = torch.zeros(256)
    inv[:64] = 10000.0 ** (-torch.arange(64) * 2.0 / 512)
    qo, _ = rope(q, None, pos, inv.cuda())
    keep = torch.cat([torch.arange(64, 256), torch.arange(320, 512)]).cuda()
    assert torch.equal(qo[..., keep], q[..., keep])
    _check(q, qo, pos, inv.cuda())


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(interleaved):
    """The gradient of <w, rope(x)> is the inverse rotation of w: the formula's, and differences
    of the 64-bit rotation (linear in x, so exact up to rounding)."""
    T, H, D, r = 5, 3, 128, 48
    x, w, pos = _rows((T, H, D), 10), _rows((T, H, D), 11), _pos(T, 12)
    inv, _ = rope_frequencies(r, 10000.0, device="cuda")
    got, _ = rope(w, None, pos, inv, interleaved=interleaved, inverse=True, attn_factor=1.25)
    _check(w, got, pos, inv, interleaved=interleaved, inverse=True, factor=1.25)
    f = lambda y: (w.double() * _ref(y, pos, inv, interleaved=interleaved, factor=1.25)[0]).sum()
    for t, h, d in ((0, 0, 0), (1, 2, 23), (2, 1, 24), (3, 0, 47), (4, 2, 100)):
        step = torch.zeros_like(x, dtype=torch.float64)
        step[t, h, d] = 0.5
        diff = float(f(x.double() + step) - f(x.double() - step))
        assert abs(diff - float(got[t, h, d])) <= 2.0 ** -8 * abs(diff) + 2.0 ** -19 * 8.0


def test_there_and_back():
    q, pos = _rows((64, 8, 256), 13), _pos(64, 14)
    inv, _ = rope_frequencies(256, 10000.0, device="cuda")
    there, _ = rope(q, None, pos, inv)
    back, _ = rope(there, None, pos, inv, inverse=True)
    # two roundings of values no larger than the pair's length
    i, j = _pairs(256, False)
    size = torch.sqrt(q.double()[..., i] ** 2 + q.double()[..., j] ** 2)
    err = (back.double() - q.double()).abs()
    assert bool((err <= 2.6 * 2.0 ** -8 * torch.cat([size, size], -1)).all())


def _guarded(n):
    return torch.full((n,), 7.0, dtype=BF, device="cuda")


@pytest.mark.parametrize("offset", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("layout", ["packed", "head_major", "odd"])
def test_strides_alignment_and_untouched_memory(layout, offset):
    """q and k views of one buffer, at element offsets that allow vectors of 8, 4, 2 and 1, in
    place; everything outside the rows keeps its bytes."""
    T, Hq, Hk, D = 19, 6, 2, 128
    if layout == "packed":      # [T, q | k | v]
        row = (Hq + 2 * Hk) * D
        buf = _guarded(T * row + 16)
        q = torch.as_strided(buf, (T, Hq, D), (row, D, 1), offset)
        k = torch.as_strided(buf, (T, Hk, D), (row, D, 1), offset + Hq * D)
    elif layout == "head_major":
        buf = _guarded((Hq + Hk) * T * D + 16)
        q = torch.as_strided(buf, (T, Hq, D), (D, T * D, 1), offset)
        k = torch.as_strided(buf, (T, Hk, D), (D, T * D, 1), offset + Hq * T * D)
    else:                       # rows and heads with odd gaps
        row = (Hq + Hk) * (D + 3) + 5
        buf = _guarded(T * row + 16)
        q = torch.as_strided(buf, (T, Hq, D), (row, D + 3, 1), offset)
        k = torch.as_strided(buf, (T, Hk, D), (row, D + 3, 1), offset + Hq * (D + 3))
    q.copy_(_rows((T, Hq, D), 15))
    k.copy_(_rows((T, Hk, D), 16))
    before, q0, k0, pos = buf.clone(), q.clone(), k.clone(), _pos(T, 17)
    inv, _ = rope_frequencies(64, 10000.0, device="cuda")
    qo, ko = rope(q, k, pos, inv, q_out=q, k_out=k)
    assert qo is q and ko is k
    _check(q0, q, pos, inv)
    _check(k0, k, pos, inv)
    q.copy_(q0)
    k.copy_(k0)
    assert torch.equal(buf.view(torch.int16), before.view(torch.int16))


def test_output_into_a_cache_view():
    """Rows written straight into a [Hkv, cap, D] cache at their positions; the rows around stay."""
    Hk, cap, D, T, at = 4, 64, 512, 10, 23
    cache, k = _guarded(Hk * cap * D).view(Hk, cap, D), _rows((T, Hk, D), 18)
    pos = torch.arange(at, at + T, dtype=torch.int32, device="cuda")
    inv, _ = rope_frequencies(512, 10000.0, device="cuda")
    rope(None, k, pos, inv, k_out=cache[:, at:at + T].transpose(0, 1))
    _check(k, cache[:, at:at + T].transpose(0, 1), pos, inv)
    assert bool((cache[:, :at] == 7).all()) and bool((cache[:, at + T:] == 7).all())


def test_no_tokens():
    q = torch.empty((0, 4, 128), dtype=BF, device="cuda")
    inv, _ = rope_frequencies(128, 10000.0, device="cuda")
    qo, _ = rope(q, None, torch.empty(0, dtype=torch.int32, device="cuda"), inv)
    assert qo.shape == q.shape


def test_infinities_stay_in_their_pair():
    q, pos = _rows((4, 2, 128), 19), torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    inv, _ = rope_frequencies(64, 10000.0, device="cuda")
    bad = q.clone()
    bad[1, 0, 5], bad[2, 1, 100] = float("nan"), float("inf")
    a, b = rope(q, None, pos, inv)[0], rope(bad, None, pos, inv)[0]
    assert bool(b[1, 0, [5, 37]].isnan().all()) and float(b[2, 1, 100]) == float("inf")
    a[1, 0, [5, 37]] = b[1, 0, [5, 37]] = 0.0
    a[2, 1, 100] = b[2, 1, 100] = 0.0
    assert torch.equal(a, b)


def test_elements_past_32_bits():
    """2^17 + 3 tokens of 36 heads x 512: 2.4e9 elements each way."""
    T, H, D = 2 ** 17 + 3, 36, 512
    q = torch.zeros((T, H, D), dtype=BF, device="cuda")
    tail = _rows((5, H, D), 20)
    q[-5:] = tail
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    inv, _ = rope_frequencies(D, 10000.0, device="cuda")
    rope(q, None, pos, inv, q_out=q)
    _check(tail, q[-5:], pos[-5:], inv)
    assert float(q[:-5].abs().max()) == 0.0


def test_captured_and_on_another_stream():
    """A captured call replayed on refilled inputs, with eager calls between the replays."""
    q, k, pos = _rows((3, 8, 256), 21), _rows((3, 4, 256), 22), _pos(3, 23)
    inv, _ = rope_frequencies(256, 10000.0, device="cuda")
    call = RopeCall(q, k, pos, inv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    _check(q, call.q_out, pos, inv)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        q.copy_(_rows((3, 8, 256), 30 + i))
        k.copy_(_rows((3, 4, 256), 40 + i))
        pos.copy_(_pos(3, 50 + i))
        want = rope(q, k, pos, inv)
        graph.replay()
        assert torch.equal(call.q_out, want[0]) and torch.equal(call.k_out, want[1])
        _check(q, call.q_out, pos, inv)
