"""Rotary positions on the host: the frequency scalings against their formulas, and the calls
esda_rope refuses before it touches the device."""
import ctypes
import math

import pytest
import torch

from apertura_amd import _lib
from apertura_amd.rope import RopeCall, RopeScaling, rope_frequencies

FAKE = 0x10000000  # never dereferenced: validation fails first


def _plain(r, base):
    return [base ** (-2.0 * i / r) for i in range(r // 2)]


@pytest.mark.parametrize("r,base", [(2, 10000.0), (40, 10000.0), (64, 1e6), (128, 500000.0), (512, 1e6)])
def test_frequencies_plain_linear_ntk(r, base):
    def close(kind, want, factor=8.0):
        inv, f = rope_frequencies(r, base, RopeScaling(kind, factor=factor))
        assert f == 1.0 and inv.dtype == torch.float32 and inv.shape == (r // 2,)
        # one rounding to fp32 of a 64-bit value
        assert torch.allclose(inv.double(), torch.tensor(want, dtype=torch.float64), rtol=2.0 ** -23, atol=0)

    close("none", _plain(r, base))
    close("linear", [f / 8.0 for f in _plain(r, base)])
    if r > 2:
        close("ntk", _plain(r, base * 8.0 ** (r / (r - 2))))


def test_ntk_stretches_the_slowest_pair_by_the_factor():
    r, s = 128, 4.0
    a, _ = rope_frequencies(r, 1e4)
    b, _ = rope_frequencies(r, 1e4, RopeScaling("ntk", factor=s))
    assert b[0] == a[0] and abs(float(a[-1] / b[-1]) - s) < 1e-5


def test_bands_keep_fast_pairs_and_stretch_slow_ones():
    r, base, L, s = 128, 500000.0, 8192, 8.0
    inv, f = rope_frequencies(r, base, RopeScaling("bands", s, L, 1.0, 4.0))
    assert f == 1.0
    for i, got in enumerate(inv.tolist()):
        plain = base ** (-2.0 * i / r)
        turns = L * plain / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / 3.0))
        assert got == pytest.approx(keep * plain + (1 - keep) * plain / s, rel=2.0 ** -22)
    assert inv[0] == 1.0


def test_yarn_ramps_over_pairs_and_scales_cos_and_sin():
    r, base, L, s = 64, 10000.0, 4096, 16.0
    inv, f = rope_frequencies(r, base, RopeScaling("yarn", s, L, 1.0, 32.0))
    assert f == pytest.approx(0.1 * math.log(s) + 1.0, rel=1e-6)
    pair = lambda turns: r * math.log(L / (turns * 2 * math.pi)) / (2 * math.log(base))
    a, b = math.floor(pair(32.0)), math.ceil(pair(1.0))
    for i, got in enumerate(inv.tolist()):
        plain = base ** (-2.0 * i / r)
        keep = 1.0 - min(1.0, max(0.0, (i - a) / (b - a)))
        assert got == pytest.approx(keep * plain + (1 - keep) * plain / s, rel=2.0 ** -22)


@pytest.mark.parametrize("kw", [
    dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=514), dict(base=1.0), dict(base=math.inf), dict(base=math.nan),
    dict(kind="linear", factor=0.5), dict(kind="linear", factor=math.nan), dict(kind="ntk", factor=2.0, rot_dim=2),
    dict(kind="bands", factor=2.0, trained_len=0), dict(kind="yarn", factor=2.0, trained_len=64, low=4.0, high=4.0),
    dict(kind="yarn", factor=2.0, trained_len=64, low=0.0, high=4.0),
])
def test_bad_scalings_are_refused(kw):
    rot, base = kw.pop("rot_dim", 64), kw.pop("base", 10000.0)
    with pytest.raises(_lib.EsdaError) as ei:
        rope_frequencies(rot, base, RopeScaling(**kw))
    assert ei.value.code == 1


def test_unknown_scaling_is_refused():
    with pytest.raises(ValueError):
        rope_frequencies(64, 1e4, RopeScaling("cubic"))


def _call(q=FAKE, k=FAKE + (1 << 24), q_out=FAKE + (2 << 24), k_out=FAKE + (3 << 24), pos=FAKE + (4 << 24),
          inv=FAKE + (5 << 24), **kw):
    d = dict(tokens=4, num_q_heads=8, num_k_heads=2, head_dim=128, rot_dim=128, interleaved=0, inverse=0,
             attn_factor=1.0, q_row_stride=1024, q_head_stride=128, k_row_stride=256, k_head_stride=128,
             q_out_row_stride=1024, q_out_head_stride=128, k_out_row_stride=256, k_out_head_stride=128)
    d.update(kw)
    desc, args = _lib.RopeDesc(**d), _lib.RopeArgs(q, k, q_out, k_out, pos, inv)
    return _lib.lib().esda_rope(ctypes.byref(desc), ctypes.byref(args), None)


@pytest.mark.parametrize("kw", [
    dict(head_dim=64), dict(head_dim=96), dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=130), dict(tokens=-1), dict(tokens=2 ** 30 + 1), dict(num_k_heads=65537),
    dict(num_q_heads=-1), dict(num_q_heads=0, num_k_heads=0), dict(interleaved=2), dict(inverse=-1),
    dict(attn_factor=math.nan), dict(attn_factor=math.inf), dict(q=None), dict(k=None), dict(q_out=None),
    dict(k_out=None), dict(pos=None), dict(inv=None), dict(q=FAKE + 1), dict(pos=FAKE + 2), dict(q_row_stride=-8),
    dict(q_out_row_stride=1000),            # the rows of an output overlap
    dict(k_out_head_stride=64),             # the heads of an output overlap
    dict(q_out_row_stride=0),
    dict(q_row_stride=1 << 62),             # past any address
    dict(q_out=FAKE, q_row_stride=2048),    # in place with other strides
    dict(q_out=FAKE + 256),                 # an output over part of its input
    dict(k_out=FAKE + (2 << 24) + 256),     # k_out inside q_out
    dict(k_out=FAKE),                       # k_out over q
])
def test_bad_calls_are_refused(kw):
    assert _call(**kw) == 1
    assert b"esda_rope" in _lib.lib().esda_last_error()


def test_null_description_is_refused():
    assert _lib.lib().esda_rope(None, None, None) == 1


@pytest.mark.parametrize("kw", [
    dict(),
    dict(q_out=FAKE, k_out=FAKE + (1 << 24)),  # in place
    # q and k side by side in one row of 1280 elements, in place
    dict(k=FAKE + 2048, q_out=FAKE, k_out=FAKE + 2048, q_row_stride=1280, k_row_stride=1280, q_out_row_stride=1280,
         k_out_row_stride=1280),
    dict(num_k_heads=0, k=None, k_out=None),
    dict(num_q_heads=0, q=None, q_out=None),
])
def test_good_calls_reach_the_device(kw):
    if torch.cuda.is_available():
        pytest.skip("host check: made-up addresses")
    assert _call(**kw) in (3, 5)  # no GPU here; nothing is launched


def test_side_by_side_rows_that_overlap_are_refused():
    kw = dict(k=FAKE + 2048, q_out=FAKE, q_row_stride=1280, k_row_stride=1280, q_out_row_stride=1280,
              k_out_row_stride=1280)
    assert _call(k_out=FAKE + 2046, **kw) == 1   # one element into q's heads
    assert _call(k_out=FAKE + 2050, **kw) == 1   # one element into the next token's q
    assert _call(tokens=0) == 0                  # nothing to do


def test_front_end_refuses_wrong_tensors():
    q, pos, inv = torch.zeros(4, 8, 128, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32), torch.zeros(64)
    for args in ((q, None, pos, inv), (q.float(), None, pos, inv), (q[..., ::2], None, pos, inv),
                 (q, None, pos.long(), inv), (q, None, pos[:3], inv), (q, None, pos, inv.double()), (None, None, pos, inv),
                 (q[0], None, pos, inv)):
        with pytest.raises(ValueError):
            RopeCall(*args)


def test_values_that_a_description_would_wrap_are_refused():
    with pytest.raises(ValueError):
        rope_frequencies(2 ** 32 + 64, 10000.0)
    with pytest.raises(ValueError):
        rope_frequencies(64, 10000.0, RopeScaling("yarn", 8.0, 2 ** 32 + 8192, 1.0, 32.0))
