"""Memory that a call of esda_pages.h or esda_tree.h would write to twice: pools, planes and workspaces that
overlap are refused before the device is touched, those that lie between one another are not."""
import ctypes
import os
import subprocess

import pytest

from apertura_amd import _lib
from apertura_amd.tree import TreeStep, tree_workspace_bytes

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AT = 0x10000000  # never dereferenced
N, R, D = 20, 16, 128
ROWS = R * D  # elements of a page of one head


def _error():
    return _lib.lib().esda_last_error().decode()


def _pool(at, planes=2, heads=3, dim=D, plane=None, page=None, head=None):
    """at: elements from AT."""
    head = R * dim if head is None else head
    page = heads * head if page is None else page
    return _lib.Pool(AT + 2 * at, planes, heads, dim, 0, N * page if plane is None else plane, page, head)


def _calls(pools, **kw):
    """(code, message) of every call on a cache of these pools."""
    c = _lib.Pages(num_pages=N, page_rows=R, slots=6, max_pages=5, table_stride=7, table=AT - (1 << 20), refs=AT - (1 << 19),
                   length=AT - (1 << 18), num_pools=len(pools), workspace=AT - (1 << 24), workspace_bytes=0)
    for i, p in enumerate(pools):
        c.pools[i] = p
    for k, v in kw.items():
        setattr(c, k, v)
    L, a, found = _lib.lib(), AT - (1 << 21), {}
    for name, call in {"reserve": lambda: L.esda_pages_reserve(ctypes.byref(c), a, a, 3, None),
                       "free": lambda: L.esda_pages_free(ctypes.byref(c), a, 3, None),
                       "fork": lambda: L.esda_pages_fork(ctypes.byref(c), a, a, None, 3, None),
                       "compact": lambda: L.esda_pages_compact(ctypes.byref(c), None),
                       "commit": lambda: L.esda_tree_commit(ctypes.byref(c), a, 5, 5, a, None)}.items():
        found[name] = call(), _error()
    return found


ONE = 2 * N * 3 * ROWS  # elements of a pool of 2 planes and 3 heads
OVER = [
    [_pool(0), _pool(0)], [_pool(0), _pool(8)], [_pool(8), _pool(0)], [_pool(0), _pool(ONE - 8)], [_pool(0), _pool(N * 3 * ROWS)],
    [_pool(0), _pool(5 * ONE), _pool(ONE // 2)],
    # heads of 128 and 256 dims over one another; a small pool within a large one
    [_pool(0), _pool(ROWS, 1, 1, 256)], [_pool(0), _pool(7 * ROWS, 1, 1)],
    # pages side by side, with the second's some elements too early
    [_pool(0, page=5 * ROWS), _pool(3 * ROWS - 8, heads=2, page=5 * ROWS)],
]
APART = [
    [_pool(0), _pool(ONE)], [_pool(ONE), _pool(0)], [_pool(0), _pool(ONE, 3, 1, 512), _pool(-3 * ONE)],
    # two pools' planes in turn; their pages in turn; heads in turn; pages of two head shapes in turn
    [_pool(0, plane=2 * N * 3 * ROWS), _pool(N * 3 * ROWS, plane=2 * N * 3 * ROWS)],
    [_pool(0, page=5 * ROWS), _pool(3 * ROWS, heads=2, page=5 * ROWS)],
    [_pool(0, head=2 * ROWS), _pool(ROWS, head=2 * ROWS)],
    [_pool(0, page=9 * ROWS, plane=3 * ROWS), _pool(6 * ROWS, 1, 1, 256, page=9 * ROWS)],
]


@pytest.mark.parametrize("pools", OVER)
def test_pools_that_overlap_are_refused(pools):
    for name, (code, why) in _calls(pools).items():
        assert code == 1 and "two pools overlap" in why, name


@pytest.mark.parametrize("pools", APART)
def test_pools_beside_and_between_one_another_are_taken(pools):
    for name, (code, why) in _calls(pools).items():
        assert code == 4 and "workspace" in why, name  # past the pools' checks


@pytest.mark.parametrize("at", [0, 8 * 1000, 2 * ONE - 16, -16])
def test_workspaces_over_a_pool_are_refused(at):
    for name, (code, why) in _calls([_pool(4 * ONE), _pool(0)], workspace=AT + at, workspace_bytes=1 << 30).items():
        assert code == 1 and "overlap a pool" in why, name


@pytest.mark.parametrize("what", ["table", "refs", "length"])
def test_workspaces_over_the_lists_are_refused(what):
    for name, (code, why) in _calls([_pool(0)], workspace_bytes=1 << 30, **{what: AT - (1 << 24) + 16}).items():
        if name != "commit" or what != "refs":
            assert code == 1 and "overlap table, refs or length" in why, name


def _tree(k, v, step, **kw):
    d = step.desc()
    ws = tree_workspace_bytes(step)
    base = 1 << 28
    a = dict(q=AT, k_new=AT + base, v_new=AT + 2 * base, k_pages=AT + 3 * base + 2 * k, v_pages=AT + 3 * base + 2 * v, table=AT + 5 * base,
             length=AT + 6 * base, parent=None, out=AT + 7 * base, workspace=None, workspace_bytes=ws)
    if step.max_pages == 0:
        a.update(table=None)
    a.update(kw)
    code = _lib.lib().esda_tree_decode(ctypes.byref(d), ctypes.byref(_lib.TreeArgs(**a)), None)
    return code, _error(), base, ws


def _step(**kw):
    return TreeStep(**dict(dict(batch=4, nodes=5, num_q_heads=8, num_kv_heads=2, head_dim=D, num_pages=N, page_rows=R, max_pages=10), **kw))


@pytest.mark.parametrize("k,v,kw", [(0, 8, {}), (0, ROWS, {}), (8, 0, {}), (0, 2 * N * ROWS - 8, {}), (0, ROWS, dict(page_stride=3 * ROWS)),
                                    (0, 2 * ROWS - 8, dict(page_stride=4 * ROWS)), (0, 50 * D, dict(num_pages=4, page_rows=100, max_pages=0))])
def test_planes_that_overlap_are_refused(k, v, kw):
    code, why, *_ = _tree(k, v, _step(**kw))
    assert code == 1 and "k_pages and v_pages" in why


@pytest.mark.parametrize("k,v,kw", [(0, 2 * N * ROWS, {}), (2 * N * ROWS, 0, {}), (0, 2 * ROWS, dict(page_stride=4 * ROWS)),
                                    (0, ROWS, dict(page_stride=4 * ROWS, head_stride=2 * ROWS)),
                                    (0, 200 * D, dict(num_pages=4, page_rows=100, max_pages=0, page_stride=400 * D))])
def test_planes_beside_and_between_one_another_are_taken(k, v, kw):
    code, why, *_ = _tree(k, v, _step(**kw))
    assert code == 4 and "workspace" in why


@pytest.mark.parametrize("what", ["q", "k_new", "v_new", "k_pages", "v_pages", "table", "length", "parent", "out"])
def test_step_workspaces_over_a_tensor_are_refused(what):
    step, base = _step(split_rows=32), 1 << 28
    ws = tree_workspace_bytes(step)
    at = dict(q=0, k_new=1, v_new=2, k_pages=3, v_pages=4, table=5, length=6, out=7, parent=8)
    for place in (16 - ws, 0):
        code, why, *_ = _tree(0, base // 2, step, parent=AT + 8 * base, workspace=AT + at[what] * base + place, workspace_bytes=ws)
        assert code == 1 and "the workspace must not overlap" in why, place


def test_apart_against_the_elements(tmp_path):
    """esda_page_view.h on random blocks."""
    exe = tmp_path / "page_view_check"
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "include"),
                        "-I", os.path.join(ROOT, "apertura_amd", "csrc"), os.path.join(ROOT, "tests", "page_view_check.cpp"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
