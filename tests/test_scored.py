"""Attention with modified scores on the host: workspace plans and the calls that esda_scored_* refuse
before they touch the device."""
import ctypes
import math

import pytest
import torch

from apertura_amd import _lib
from apertura_amd.decode import DecodeStep, workspace_bytes
from apertura_amd.prefill import PrefillStep, prefill_workspace_bytes
from apertura_amd.scored import Score, ScoredDecodeCall, scored_prefill, scored_prefill_workspace_bytes

FAKE = 0x10000000  # never dereferenced: validation fails first


def _step(**kw):
    base = dict(num_q_heads=8, num_kv_heads=2, head_dim=128, seq_q=64, seq_k=64)
    base.update(kw)
    return PrefillStep(**base)


@pytest.mark.parametrize("kw", [dict(), dict(seq_q=512, seq_k=16384, q_pos0=15872, head_dim=512, num_q_heads=32),
                                dict(seq_q=100, seq_k=1123, q_pos0=1023, window=1024, head_dim=256)])
def test_a_plain_score_plans_like_the_plain_call(kw):
    assert scored_prefill_workspace_bytes(_step(**kw), Score()) == prefill_workspace_bytes(_step(**kw))


def test_a_prefix_opens_keys_ahead():
    """One split of 64 keys holds what 16 fresh queries see; with a prefix they see 1024."""
    step = _step(seq_q=16, seq_k=1024, split_keys=64)
    assert scored_prefill_workspace_bytes(step, Score()) == 0
    assert scored_prefill_workspace_bytes(step, Score(prefix=1024)) == 16 * 16 * 8 * (128 * 4 + 8) + 256


@pytest.mark.parametrize("kw", [dict(q_pos0=10, seq_k=5), dict(k_pos0=100), dict(q_pos0=5000, window=16),
                                dict(k_pos0=2 ** 31 - 64 - 65)])
def test_keys_need_not_hold_the_queries(kw):
    assert scored_prefill_workspace_bytes(_step(**kw), Score()) == 0


@pytest.mark.parametrize("score", [Score(softcap=-1.0), Score(softcap=math.nan), Score(softcap=math.inf),
                                   Score(prefix=-1), Score(softcap=1e-44)])
def test_bad_scores_are_refused(score):
    with pytest.raises(_lib.EsdaError) as ei:
        scored_prefill_workspace_bytes(_step(), score)
    assert ei.value.code == 1
    assert _decode(softcap=score.softcap, prefix=score.prefix) == 1


@pytest.mark.parametrize("kw", [dict(head_dim=64), dict(num_q_heads=7), dict(seq_q=0), dict(seq_k=0), dict(window=-1),
                                dict(split_keys=40), dict(scale=0.0), dict(scale=math.nan), dict(q_pos0=-1),
                                dict(k_pos0=2 ** 31 - 64 - 63), dict(kv_head_stride=64), dict(q_row_stride=132)])
def test_bad_chunks_are_refused(kw):
    with pytest.raises(_lib.EsdaError) as ei:
        scored_prefill_workspace_bytes(_step(**kw), Score())
    assert ei.value.code == 1


def _prefill(q=FAKE, k=FAKE, v=FAKE, out=FAKE + (1 << 24), ws=None, nbytes=0, q_doc=None, k_doc=None, slopes=None, step=None):
    d = (step or _step()).desc()
    s = _lib.ScoreDesc(0.0, 0, slopes)
    a = _lib.ScoredPrefillArgs(q, k, v, out, ws, nbytes, q_doc, k_doc)
    return _lib.lib().esda_scored_prefill(ctypes.byref(d), ctypes.byref(s), ctypes.byref(a), None)


@pytest.mark.parametrize("kw", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=FAKE + 8), dict(out=FAKE),
                                dict(out=FAKE + 2), dict(q_doc=FAKE), dict(k_doc=FAKE), dict(q_doc=FAKE, k_doc=FAKE + 1),
                                dict(q_doc=FAKE + 2, k_doc=FAKE), dict(slopes=FAKE + 2)])
def test_bad_prefill_arguments_are_refused(kw):
    assert _prefill(**kw) == 1


def test_prefill_needs_its_workspace():
    step = _step(seq_q=16, seq_k=1024, q_pos0=1008, split_keys=64)
    need = scored_prefill_workspace_bytes(step, Score())
    assert need > 0
    assert _prefill(step=step) == 4
    assert _prefill(step=step, ws=FAKE, nbytes=need - 1) == 4
    assert _prefill(step=step, ws=FAKE + 4, nbytes=need) == 4


def test_null_structures_are_refused():
    d, s = _step().desc(), _lib.ScoreDesc()
    L = _lib.lib()
    assert L.esda_scored_prefill(None, ctypes.byref(s), None, None) == 1
    assert L.esda_scored_prefill(ctypes.byref(d), None, None, None) == 1
    assert L.esda_scored_prefill(ctypes.byref(d), ctypes.byref(s), None, None) == 1
    assert L.esda_scored_prefill_workspace_size(ctypes.byref(d), ctypes.byref(s), None) == 1
    assert L.esda_scored_decode(None, ctypes.byref(s), None, None) == 1


def _decode(softcap=0.0, prefix=0, slopes=None, ws=FAKE, nbytes=None, k_new=FAKE, v_cache=FAKE + (1 << 24), score=True,
            **kw):
    base = dict(batch=2, num_q_heads=8, num_kv_heads=2, head_dim=128, cap=64)
    base.update(kw)
    step = DecodeStep(**base)
    d, s = step.desc(), _lib.ScoreDesc(softcap, prefix, slopes)
    if nbytes is None:
        try:
            nbytes = workspace_bytes(step)
        except _lib.EsdaError:
            nbytes = 0
    a = _lib.DecodeArgs(FAKE, k_new, FAKE, FAKE, v_cache, FAKE, None, FAKE, ws, nbytes)
    return _lib.lib().esda_scored_decode(ctypes.byref(d), ctypes.byref(s) if score else None, ctypes.byref(a), None)


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(num_q_heads=68), dict(batch=257), dict(ring=True, window=0),
                                dict(slopes=FAKE + 1), dict(k_new=None), dict(v_cache=FAKE), dict(score=False),
                                dict(scale=0.0), dict(scale=math.inf)])
def test_bad_decode_calls_are_refused(kw):
    assert _decode(**kw) == 1


def test_decode_needs_its_workspace():
    assert _decode(ws=None) == 4
    assert _decode(nbytes=16) == 4
    assert _decode(ws=FAKE + 8) == 4


def test_front_end_refuses_wrong_tensors():
    bf = torch.bfloat16
    q, k = torch.zeros(8, 64, 128, dtype=bf), torch.zeros(2, 64, 128, dtype=bf)
    ids = torch.zeros(64, dtype=torch.int32)
    for kw in (dict(), dict(q_doc=ids), dict(q_doc=ids.long(), k_doc=ids), dict(q_doc=ids, k_doc=ids[:60])):
        with pytest.raises(ValueError):  # CPU tensors, or ids that do not fit
            scored_prefill(_step(), Score(), q, k, k.clone(), **kw)
    with pytest.raises(ValueError):
        scored_prefill(_step(), Score(slopes=torch.zeros(2)), q, k, k)
    with pytest.raises(ValueError):
        scored_prefill(_step(seq_k=65), Score(), q, k, k)
    step = DecodeStep(batch=2, num_q_heads=8, num_kv_heads=2, head_dim=128, cap=64)
    with pytest.raises(ValueError):
        ScoredDecodeCall(step, Score(), torch.zeros(2, 8, 128, dtype=bf), torch.zeros(2, 2, 128, dtype=bf), None,
                         torch.zeros(2, 2, 64, 128, dtype=bf), torch.zeros(2, 2, 64, 128, dtype=bf),
                         torch.zeros(2, dtype=torch.int32))


def test_an_output_that_overlaps_an_input_is_refused():
    """By any element: a view further into q, k or v, one that ends inside them, heads or rows between
    theirs.  (Calls that pass would be launched: those have real memory, in the GPU tests.)"""
    q_bytes, kv_bytes = 8 * 64 * 128 * 2, 2 * 64 * 128 * 2
    k, v = FAKE + (1 << 20), FAKE + (2 << 20)
    for out in (FAKE, FAKE + 16, FAKE + q_bytes - 16, FAKE - q_bytes + 16, k + 256, k + kv_bytes - 16, v - 16, v + kv_bytes - 16):
        assert _prefill(k=k, v=v, out=out) == 1, hex(out - FAKE)
    assert "overlap" in _lib.lib().esda_last_error().decode()
    # rows of one buffer whose out columns reach into k's, and heads that reach into the next
    rows = _step(q_row_stride=12 * 128, q_head_stride=128, out_row_stride=12 * 128, out_head_stride=128)
    assert _prefill(step=rows, k=k, v=v, out=FAKE + 2 * 128 * 7) == 1
    assert _prefill(step=_step(out_row_stride=2 ** 60, out_head_stride=128), k=k, v=v) == 1


@pytest.mark.parametrize("make", [
    lambda: Score(prefix=2 ** 32).desc(8), lambda: Score(prefix=2 ** 31).desc(8), lambda: Score(softcap=1e-46).desc(8),
    lambda: _step(q_pos0=2 ** 32 + 5).desc(), lambda: _step(k_pos0=-2 ** 32).desc(), lambda: _step(window=2 ** 32 + 8).desc(),
    lambda: _step(split_keys=2 ** 32 + 32).desc(),
    lambda: DecodeStep(batch=2, num_q_heads=8, num_kv_heads=2, head_dim=128, cap=64, window=2 ** 32 + 8).desc(),
    lambda: DecodeStep(batch=2, num_q_heads=8, num_kv_heads=2, head_dim=128, cap=64, max_visible=2 ** 32 + 8).desc(),
])
def test_values_that_a_description_would_change_are_refused(make):
    """A 32-bit field wraps what it cannot hold (a prefix of 2^32 would be none), and a cap below
    float32's smallest number is 0, which is no cap."""
    with pytest.raises(ValueError):
        make()
