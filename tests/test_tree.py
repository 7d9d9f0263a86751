"""The step of drafted tokens on the host: its workspace and the calls esda_tree_decode refuses before it
touches the device."""
import ctypes
import math
import time

import pytest
import torch

from apertura_amd import _lib
from apertura_amd.tree import TreeCall, TreeStep, tree_workspace_bytes

FAKE = 0x10000000  # never dereferenced: validation fails first


def _step(**kw):
    base = dict(batch=4, nodes=5, num_q_heads=8, num_kv_heads=2, head_dim=128, num_pages=40, page_rows=16, max_pages=10)
    base.update(kw)
    return TreeStep(**base)


def _linear(**kw):
    return _step(**dict(dict(num_pages=4, page_rows=100, max_pages=0), **kw))


def test_workspace_holds_every_partial():
    """The status word, the sequences' pieces, then (m, l) and O of every piece of the query rows (a sequence
    has 165 keys at most; pieces of all heads in eights)."""
    up = lambda n, of=256: (n + of - 1) // of * of
    for rows, splits in ((32, 6), (64, 3), (96, 2)):
        parts = up(splits * 4 * 2, 8) * 5 * 4
        assert tree_workspace_bytes(_step(split_rows=rows)) == 256 + up(32) + up(parts * 8) + parts * 128 * 4
    for rows in (192, 320, 2 ** 31 - 32):  # one split: no partials
        assert tree_workspace_bytes(_step(split_rows=rows)) == 512


def test_bounds_on_rows_size_the_splits():
    """A window, of which a sequence sees no more; automatic splits of long caches do not go by the room for rows."""
    long = dict(max_pages=4000, split_rows=64)
    assert tree_workspace_bytes(_step(window=200, **long)) < tree_workspace_bytes(_step(**long))
    assert tree_workspace_bytes(_step(nodes=4, max_pages=8000)) == tree_workspace_bytes(_step(nodes=4, max_pages=4000))
    assert tree_workspace_bytes(_linear(split_rows=32)) > tree_workspace_bytes(_linear(split_rows=64))


@pytest.mark.parametrize("kw", [
    dict(batch=0), dict(batch=257), dict(nodes=0), dict(nodes=65), dict(num_q_heads=9), dict(num_q_heads=34), dict(num_kv_heads=0),
    dict(head_dim=64), dict(window=-1), dict(window=4), dict(num_pages=0), dict(num_pages=2 ** 22 + 1), dict(page_rows=8),
    dict(page_rows=24), dict(page_rows=8192), dict(max_pages=-1), dict(max_pages=2 ** 19, page_rows=4096),
    dict(max_pages=2 ** 19 - 1, page_rows=4096, split_rows=32), dict(max_pages=2 ** 20 + 1), dict(table_stride=9),
    dict(page_stride=2 * 16 * 128 - 8), dict(head_stride=16 * 128 + 4), dict(head_stride=8), dict(page_stride=-8),
    dict(page_stride=2 ** 60), dict(split_rows=16), dict(split_rows=-32), dict(scale=0.0),
    dict(scale=math.nan), dict(scale=math.inf), dict(batch=256, nodes=64, num_q_heads=16 * 64, num_kv_heads=64),
])
def test_bad_descriptions_are_refused(kw):
    with pytest.raises(_lib.EsdaError) as ei:
        tree_workspace_bytes(_step(**kw))
    assert ei.value.code == 1


@pytest.mark.parametrize("kw", [dict(num_pages=5), dict(page_rows=0), dict(page_rows=2 ** 30 + 1), dict(page_stride=2 * 100 * 128 - 8)])
def test_bad_linear_caches_are_refused(kw):
    with pytest.raises(_lib.EsdaError) as ei:
        tree_workspace_bytes(_linear(**kw))
    assert ei.value.code == 1


def _call(step=None, nbytes=None, **kw):
    step = step or _step()
    d = step.desc()
    a = dict(q=FAKE, k_new=FAKE + (1 << 22), v_new=FAKE + (2 << 22), k_pages=FAKE + (1 << 24), v_pages=FAKE + (2 << 24),
             table=FAKE, length=FAKE, parent=None, out=FAKE + (3 << 22), workspace=FAKE, workspace_bytes=tree_workspace_bytes(step) if nbytes is None else nbytes)
    a.update(kw)
    return _lib.lib().esda_tree_decode(ctypes.byref(d), ctypes.byref(_lib.TreeArgs(**a)), None)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(k_new=None), dict(v_new=None), dict(k_pages=None), dict(v_pages=None), dict(out=None), dict(length=None),
    dict(table=None), dict(v_pages=FAKE + (1 << 24)), dict(q=FAKE + 8), dict(out=FAKE + 4),
    dict(out=FAKE), dict(out=FAKE + 4 * 5 * 8 * 128 * 2 - 16), dict(out=FAKE + (1 << 22)), dict(out=FAKE + (2 << 22)),
    dict(out=FAKE + (1 << 24) + 4096), dict(out=FAKE + (2 << 24) + 40 * 2 * 16 * 128 * 2 - 16), dict(k_new=FAKE + (1 << 24)),
    dict(v_new=FAKE + (2 << 24) - 16), dict(v_new=FAKE + (1 << 24)), dict(v_new=FAKE + 2), dict(k_pages=FAKE + (1 << 24) + 8),
    dict(length=FAKE + 2), dict(table=FAKE + 2), dict(parent=FAKE + 1), dict(step=_linear()),
    dict(step=_step(kv_shared=True)),
])
def test_bad_arguments_are_refused(kw):
    assert _call(**kw) == 1


def test_the_workspace_is_needed():
    assert _call(out=FAKE + 4 * 5 * 8 * 128 * 2, workspace=None) == 4  # right behind q
    assert _call(workspace=None) == 4
    assert _call(workspace=FAKE + 8) == 4
    assert _call(nbytes=tree_workspace_bytes(_step()) - 1) == 4
    assert _lib.lib().esda_tree_decode(None, None, None) == 1
    assert _lib.lib().esda_tree_decode(ctypes.byref(_step().desc()), None, None) == 1
    assert _lib.lib().esda_tree_workspace_size(ctypes.byref(_step().desc()), None) == 1


def test_front_end_refuses_wrong_tensors():
    bf = torch.bfloat16
    pages, table = torch.zeros(9, 2, 16, 128, dtype=bf), torch.zeros(4, 3, dtype=torch.int32)
    q, n = torch.zeros(4, 5, 8, 128, dtype=bf), torch.zeros(4, 5, 2, 128, dtype=bf)
    length, parent = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 5, dtype=torch.int32)
    for args in ((pages[..., ::2], table, 8, 5), (pages[0], table, 8, 5), (pages, table.long(), 8, 5), (pages, table[:, ::2], 8, 5)):
        with pytest.raises(ValueError):
            TreeStep.for_pages(*args)
    with pytest.raises(ValueError):
        TreeStep.for_cache(pages[:, :, :, :64], 8, 5)
    step = TreeStep.for_pages(pages, table, 8, 5)
    good = dict(q=q, k_new=n, v_new=n, k_pages=pages, v_pages=pages.clone(), length=length, table=table, parent=parent)
    for kw in (dict(), dict(q=q[:3]), dict(q=q.transpose(1, 2)), dict(k_new=n[:, :4]), dict(v_new=None), dict(v_new=n[:, :, :1]),
               dict(k_pages=pages[:8]), dict(v_pages=pages[:, :, :8]), dict(length=length.long()), dict(length=length[:2]),
               dict(table=None), dict(table=table[:, :2]), dict(parent=parent.long()), dict(parent=parent[:, :4]), dict(out=q[:2])):
        with pytest.raises(ValueError):  # (the first: not on a GPU)
            TreeCall(step, **dict(good, **kw))
    linear = TreeStep.for_cache(torch.zeros(4, 2, 30, 128, dtype=bf), 8, 5)
    with pytest.raises(ValueError):
        TreeCall(linear, **good)


@pytest.mark.parametrize("kw", [dict(page_rows=2 ** 32 + 16), dict(max_pages=2 ** 32), dict(window=2 ** 32 + 64), dict(split_rows=2 ** 32)])
def test_values_that_a_description_would_wrap_are_refused(kw):
    with pytest.raises(ValueError):
        _step(**kw).desc()


@pytest.mark.parametrize("kw", [
    dict(batch=256, nodes=64, num_q_heads=32, num_kv_heads=4, head_dim=512, max_pages=2 ** 18, num_pages=2 ** 22, page_rows=4096),
    dict(max_pages=2 ** 19 - 1, page_rows=4096, split_rows=2 ** 23),
    dict(batch=1, nodes=1, num_q_heads=1, num_kv_heads=1, max_pages=1), dict(max_pages=2 ** 20, page_rows=1024),
    dict(batch=256, num_q_heads=512, num_kv_heads=32, max_pages=2 ** 16), dict(batch=1, nodes=64, max_pages=2 ** 20, window=2 ** 30),
    dict(batch=1, num_pages=1, page_rows=2 ** 30, max_pages=0),
])
def test_extreme_descriptions_plan_quickly(kw):
    step = _step(**kw)
    t = time.perf_counter()
    n = tree_workspace_bytes(step)
    assert time.perf_counter() - t < 0.25
    assert 512 <= n <= 4096 + step.batch * 4 + 600 * step.batch * step.nodes * step.num_q_heads * (4 * step.head_dim + 8)


def test_the_pieces_of_random_batches(tmp_path):
    """esda_tree_plan.h: every key in one piece, and no more pieces than the host makes room for."""
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = tmp_path / "tree_plan_check"
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                        os.path.join(root, "apertura_amd", "csrc"), os.path.join(root, "tests", "tree_plan_check.cpp"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
