"""The decode step over a shared prefix on the host: its workspace and the calls esda_prefix_decode
refuses before it touches the device."""
import ctypes
import math
import time

import pytest
import torch

from apertura_amd import _lib
from apertura_amd.decode import DecodeStep
from apertura_amd.prefix import PrefixCall, PrefixStep, prefix_workspace_bytes

FAKE = 0x10000000  # never dereferenced: validation fails first


def _step(prefix_len=100, prefix_head_stride=None, split_keys=0, **kw):
    base = dict(batch=4, num_q_heads=8, num_kv_heads=2, head_dim=128, cap=64)
    base.update(kw)
    return PrefixStep(DecodeStep(**base), prefix_len, prefix_head_stride, split_keys)


def test_workspace_holds_every_partial():
    """The status word, then (m, l) and O of every prefix split and own split of the 32 query rows."""
    up = lambda n: (n + 255) // 256 * 256
    for keys, splits in ((32, 4), (64, 2), (128, 1)):
        for rows, own in ((16, 4), (32, 2), (0, 1)):
            want = 256 + up(splits * 32 * 8) + up(own * 32 * 8) + (splits + own) * 32 * 128 * 4
            assert prefix_workspace_bytes(_step(split_keys=keys, split_rows=rows)) == want


def test_a_bound_on_own_rows_sizes_their_splits():
    big, small = _step(cap=100000, split_rows=512), _step(cap=100000, split_rows=512, max_visible=1000)
    assert prefix_workspace_bytes(small) < prefix_workspace_bytes(big)


@pytest.mark.parametrize("kw", [
    dict(prefix_len=0), dict(prefix_len=-1), dict(prefix_len=2 ** 30 + 1), dict(prefix_head_stride=99 * 128), dict(prefix_head_stride=100 * 128 + 4),
    dict(split_keys=16), dict(split_keys=-32), dict(window=16), dict(ring=True, window=64), dict(head_dim=64),
    dict(num_q_heads=9), dict(num_q_heads=34), dict(batch=0), dict(batch=257), dict(cap=0), dict(scale=0.0),
    dict(scale=math.nan), dict(split_rows=8), dict(batch=128, num_q_heads=16 * 16384, num_kv_heads=16384),
    dict(prefix_len=2 ** 30, cap=2 ** 30),
])
def test_bad_descriptions_are_refused(kw):
    with pytest.raises(_lib.EsdaError) as ei:
        prefix_workspace_bytes(_step(**kw))
    assert ei.value.code == 1


def _call(step=None, prefix_k=FAKE, prefix_v=FAKE + (1 << 24), row_base=None, ws=FAKE, nbytes=None, q=FAKE,
          k_new=FAKE, v_new=FAKE, k_cache=FAKE, v_cache=FAKE + (2 << 24), pos=FAKE, out=FAKE):
    step = step or _step()
    d = step.desc()
    a = _lib.PrefixArgs(_lib.DecodeArgs(q, k_new, v_new, k_cache, v_cache, pos, row_base, out, ws,
                                        prefix_workspace_bytes(step) if nbytes is None else nbytes), prefix_k, prefix_v)
    return _lib.lib().esda_prefix_decode(ctypes.byref(d), ctypes.byref(a), None)


@pytest.mark.parametrize("kw", [
    dict(prefix_k=None), dict(prefix_v=None), dict(prefix_k=FAKE + 8), dict(prefix_v=FAKE), dict(row_base=FAKE),
    dict(q=None), dict(k_new=None), dict(v_new=None), dict(k_cache=None), dict(v_cache=FAKE), dict(pos=None),
    dict(out=FAKE + 4), dict(step=_step(kv_shared=True)), dict(step=_step(kv_shared=True), v_cache=FAKE),
])
def test_bad_arguments_are_refused(kw):
    assert _call(**kw) == 1


def test_the_workspace_is_needed():
    assert _call(ws=None) == 4
    assert _call(ws=FAKE + 8) == 4
    assert _call(nbytes=prefix_workspace_bytes(_step()) - 1) == 4
    assert _lib.lib().esda_prefix_decode(None, None, None) == 1
    assert _lib.lib().esda_prefix_decode(ctypes.byref(_step().desc()), None, None) == 1


def test_front_end_refuses_wrong_tensors():
    bf = torch.bfloat16
    pk, c = torch.zeros(2, 100, 128, dtype=bf), torch.zeros(4, 2, 64, 128, dtype=bf)
    q, n, pos = torch.zeros(4, 8, 128, dtype=bf), torch.zeros(4, 2, 128, dtype=bf), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        PrefixStep.for_caches(pk[:, :, ::2], c, 8)
    with pytest.raises(ValueError):
        PrefixStep.for_caches(pk[:1], c, 8)
    step = PrefixStep.for_caches(pk, c, 8)
    assert step.prefix_len == 100 and step.desc().prefix_head_stride == 100 * 128
    for args in ((q, n, n, pk, pk.clone(), c, c.clone(), pos),             # not on a GPU
                 (q[:3], n, n, pk, pk.clone(), c, c.clone(), pos),
                 (q, n[:, :1], n, pk, pk.clone(), c, c.clone(), pos),
                 (q, n, n, pk[:, :99], pk.clone(), c, c.clone(), pos),
                 (q, n, n, pk, pk.clone(), c, c.clone(), pos.long())):
        with pytest.raises(ValueError):
            PrefixCall(step, *args)


@pytest.mark.parametrize("kw", [
    dict(prefix_len=2 ** 30, batch=256, cap=2 ** 22), dict(prefix_len=2 ** 30, batch=1, cap=1), dict(prefix_len=1, cap=2 ** 30),
    dict(prefix_len=2 ** 29, cap=2 ** 30, batch=7, head_dim=512, num_q_heads=32), dict(prefix_len=1, batch=1, cap=1, head_dim=256),
    dict(prefix_len=2 ** 30, batch=200, cap=16, num_q_heads=1024, num_kv_heads=64), dict(prefix_len=2 ** 30, cap=2 ** 30 - 1, split_rows=16),
    dict(prefix_len=3, batch=256, cap=2 ** 20, num_q_heads=16, num_kv_heads=1, head_dim=512, kv_shared=True),
])
def test_extreme_descriptions_plan_quickly(kw):
    """Every size of the documented range has a plan, found in milliseconds, of at most 64 own splits and
    at most 512 prefix splits and a workspace for them."""
    step = _step(**kw)
    t = time.perf_counter()
    n = prefix_workspace_bytes(step)
    assert time.perf_counter() - t < 0.25
    o = step.own
    row = o.batch * o.num_q_heads * (4 * o.head_dim + 8)
    assert 2 * row <= n <= (512 + 64) * row + 4096


def test_splits_longer_than_the_rows_are_one_split():
    """Forced splits up to the end of int32, alone and together, plan as one split of the prefix and
    one of the own rows; so does every length in between."""
    one = prefix_workspace_bytes(_step(split_keys=128, split_rows=64))
    top_keys, top_rows = 2 ** 31 - 32, 2 ** 31 - 16
    for keys, rows in ((top_keys, 64), (128, top_rows), (top_keys, top_rows), (2 ** 30, 2 ** 30), (2 ** 31 - 96, 2 ** 31 - 64)):
        assert prefix_workspace_bytes(_step(split_keys=keys, split_rows=rows)) == one
    for kw in (dict(cap=2 ** 30, max_visible=40), dict(cap=2 ** 30), dict(prefix_len=2 ** 30), dict(cap=2 ** 31 - 102)):
        n = prefix_workspace_bytes(_step(split_keys=top_keys, split_rows=top_rows, **kw))
        assert n == one
    # own rows take at most 64 splits, 100 keys of a prefix at most four
    assert prefix_workspace_bytes(_step(cap=2 ** 31 - 102, split_rows=16)) <= 68 * 32 * (4 * 128 + 8) + 4096
    assert prefix_workspace_bytes(_step(cap=2 ** 31 - 102)) <= 68 * 32 * (4 * 128 + 8) + 4096


@pytest.mark.parametrize("kw", [dict(prefix_len=2 ** 32 + 100), dict(split_keys=2 ** 32 + 32), dict(split_rows=2 ** 32 + 16)])
def test_values_that_a_description_would_wrap_are_refused(kw):
    with pytest.raises(ValueError):
        _step(**kw).desc()
