"""Caches in pages on the host: workspaces, and the calls that esda_pages.h and esda_tree_commit refuse
before they touch the device."""
import ctypes
import itertools

import pytest
import torch

from apertura_amd import _lib
from apertura_amd.pages import PagedCache, pages_read, pages_write

FAKE = 0x10000000  # never dereferenced: validation fails first


def _cache(pool=None, **kw):
    c = _lib.Pages(num_pages=20, page_rows=16, slots=6, max_pages=5, table_stride=5, table=FAKE, refs=FAKE, length=FAKE,
                   num_pools=1, workspace=FAKE, workspace_bytes=1 << 30)
    d = dict(data=FAKE, planes=2, num_kv_heads=3, head_dim=128, pad=0, plane_stride=20 * 3 * 16 * 128,
             page_stride=3 * 16 * 128, head_stride=16 * 128)
    d.update(pool or {})
    for i in range(_lib.MAX_POOLS):
        c.pools[i] = _lib.Pool(**d)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _calls():
    """Every call on a cache, as a function of it."""
    L = _lib.lib()
    return {
        "reserve": lambda c: L.esda_pages_reserve(ctypes.byref(c), FAKE, FAKE, 3, None),
        "free": lambda c: L.esda_pages_free(ctypes.byref(c), FAKE, 3, None),
        "fork": lambda c: L.esda_pages_fork(ctypes.byref(c), FAKE, FAKE, None, 3, None),
        "compact": lambda c: L.esda_pages_compact(ctypes.byref(c), None),
        "commit": lambda c: L.esda_tree_commit(ctypes.byref(c), FAKE, 5, 5, FAKE, None),
    }


BAD = [dict(num_pages=0), dict(num_pages=2 ** 22 + 1), dict(page_rows=8), dict(page_rows=48), dict(page_rows=8192), dict(slots=0),
       dict(slots=2 ** 20 + 1), dict(max_pages=0), dict(max_pages=2 ** 20 + 1), dict(max_pages=2 ** 19, page_rows=4096),
       dict(table_stride=4), dict(table_stride=-5), dict(length=None), dict(length=FAKE + 2), dict(table=FAKE + 1),
       dict(num_pools=-1), dict(num_pools=9), dict(num_pools=2),  # (the second pool is the first's memory)
       dict(pool=dict(data=None)), dict(pool=dict(data=FAKE + 8)), dict(pool=dict(planes=0)), dict(pool=dict(planes=4097)),
       dict(pool=dict(num_kv_heads=0)), dict(pool=dict(head_dim=64)), dict(pool=dict(head_stride=16 * 128 - 8)),
       dict(pool=dict(head_stride=16 * 128 + 4)), dict(pool=dict(page_stride=2 * 16 * 128)), dict(pool=dict(page_stride=-8)),
       dict(pool=dict(plane_stride=0)), dict(pool=dict(plane_stride=19 * 3 * 16 * 128)), dict(pool=dict(plane_stride=2 ** 62))]


@pytest.mark.parametrize("kw", BAD)
@pytest.mark.parametrize("name", ["reserve", "free", "fork", "compact", "commit"])
def test_bad_caches_are_refused(name, kw):
    assert _calls()[name](_cache(**kw)) == 1
    assert _lib.lib().esda_last_error().decode().startswith(("esda_pages_" if name != "commit" else "esda_tree_") + name)


@pytest.mark.parametrize("name", ["reserve", "free", "fork", "compact"])
def test_bad_tables_and_references_are_refused(name):
    for kw in (dict(table=None), dict(refs=None), dict(refs=FAKE + 2)):
        assert _calls()[name](_cache(**kw)) == 1


@pytest.mark.parametrize("name", ["reserve", "free", "fork", "compact", "commit"])
def test_the_workspace_is_needed(name):
    assert _calls()[name](_cache(workspace=None)) == 4
    assert _calls()[name](_cache(workspace=FAKE + 8)) == 4
    assert _calls()[name](_cache(workspace_bytes=128)) == 4


def test_bad_lists_are_refused():
    L, c = _lib.lib(), ctypes.byref(_cache())
    for n in (-1, 1025):
        assert L.esda_pages_reserve(c, FAKE, FAKE, n, None) == 1
        assert L.esda_pages_free(c, FAKE, n, None) == 1
        assert L.esda_pages_fork(c, FAKE, FAKE, FAKE, n, None) == 1
    assert L.esda_pages_fork(c, FAKE, FAKE, FAKE, 7, None) == 1  # more than there are slots
    for a, b in ((None, FAKE), (FAKE, None), (FAKE + 2, FAKE)):
        assert L.esda_pages_reserve(c, a, b, 2, None) == 1
        assert L.esda_pages_fork(c, a, b, None, 2, None) == 1
    assert L.esda_pages_fork(c, FAKE, FAKE, FAKE + 1, 2, None) == 1
    assert L.esda_pages_free(c, None, 2, None) == 1
    for args in ((FAKE, 5, 0, FAKE), (FAKE, 65, 65, FAKE), (FAKE, 4, 5, FAKE), (None, 5, 5, FAKE), (FAKE, 5, 5, None),
                 (FAKE + 2, 5, 5, FAKE)):
        assert L.esda_tree_commit(c, *args, None) == 1
    assert L.esda_pages_reserve(None, FAKE, FAKE, 1, None) == 1
    assert L.esda_tree_commit(None, FAKE, 5, 5, FAKE, None) == 1
    assert L.esda_pages_status(None, None, None) == 1


def test_linear_caches_of_a_commit():
    """Without a table: one page of any number of rows a slot."""
    pool = dict(plane_stride=6 * 3 * 50 * 128, page_stride=3 * 50 * 128, head_stride=50 * 128)
    for kw in (dict(max_pages=2), dict(num_pages=7), dict(page_rows=0), dict(page_rows=2 ** 30 + 1), dict(page_rows=51)):
        c = _cache(pool, **dict(dict(table=None, num_pages=6, page_rows=50, max_pages=1), **kw))
        assert _calls()["commit"](c) == 1, kw


def test_workspaces_grow_with_the_cache():
    def size(**kw):
        n, c = ctypes.c_size_t(0), _cache(**kw)
        _lib.check(_lib.lib().esda_pages_workspace_size(ctypes.byref(c), ctypes.byref(n)))
        return n.value

    base = size()
    assert base >= 256 + 6 * 4 + 1024 * (16 + 16) + 20 * 4 + 6 * 5 * 4
    assert size(num_pages=2 ** 22) >= 2 ** 22 * 4 + 2 ** 21 * 16
    assert size(slots=2000, max_pages=100) >= 1024 * 100 * 4 + base - 6 * 5 * 4
    n = ctypes.c_size_t(0)
    for kw in (dict(num_pages=0), dict(slots=-1), dict(max_pages=0)):
        assert _lib.lib().esda_pages_workspace_size(ctypes.byref(_cache(**kw)), ctypes.byref(n)) == 1
    assert _lib.lib().esda_pages_workspace_size(None, ctypes.byref(n)) == 1


def _rows(pool=None, **kw):
    c = _cache(pool)
    d = dict(num_pages=20, page_rows=16, batch=6, max_pages=5, table_stride=5, rows=40, pad=0,
             linear_plane_stride=6 * 3 * 40 * 128, linear_seq_stride=3 * 40 * 128, linear_head_stride=40 * 128)
    d.update(kw)
    return _lib.PageRowsDesc(pool=c.pools[0], **d)


@pytest.mark.parametrize("kw", [
    dict(num_pages=0), dict(page_rows=17), dict(batch=0), dict(max_pages=0), dict(table_stride=3), dict(rows=-1),
    dict(rows=2 ** 30 + 1), dict(linear_plane_stride=-8), dict(linear_seq_stride=4), dict(linear_head_stride=12),
    dict(pool=dict(planes=0)), dict(pool=dict(head_dim=100)), dict(pool=dict(page_stride=128)),
])
def test_bad_row_copies_are_refused(kw):
    L, d = _lib.lib(), _rows(**kw)
    assert L.esda_pages_write(ctypes.byref(d), FAKE, FAKE, FAKE, None) == 1
    assert L.esda_pages_read(ctypes.byref(d), FAKE, FAKE, FAKE, None) == 1


def test_bad_row_copy_arguments_are_refused():
    L, d = _lib.lib(), ctypes.byref(_rows())
    for f in (L.esda_pages_write, L.esda_pages_read):
        for args in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None), (FAKE + 2, FAKE, FAKE), (FAKE, FAKE, FAKE + 8)):
            assert f(d, *args, None) == 1
        assert f(None, FAKE, FAKE, FAKE, None) == 1
    # linear rows that meet the pool's, at either end
    reach, pool = 2 * (2 * 6 * 3 * 40 * 128), 2 * (2 * 20 * 3 * 16 * 128)
    for f in (L.esda_pages_write, L.esda_pages_read):
        for at in (0, pool - 16, 16 - reach):
            assert f(d, FAKE, FAKE, FAKE + at, None) == 1 and b"overlap the pool" in L.esda_last_error()
    # linear rows that overlap may be read from, not written to
    assert L.esda_pages_read(ctypes.byref(_rows(linear_head_stride=39 * 128)), FAKE, FAKE, FAKE, None) == 1


def test_strides_in_any_order():
    """The blocks of a pool may not overlap, whichever of planes, pages and heads is the widest apart."""
    sizes = dict(plane_stride=2, page_stride=20, head_stride=3)
    for order in itertools.permutations(sizes):
        width, strides = 16 * 128, {}
        for name in order:
            strides[name] = width
            width *= sizes[name]
        assert _calls()["compact"](_cache(strides, workspace_bytes=16)) == 4  # past the checks of the pool
        for name in order:
            assert _calls()["compact"](_cache(dict(strides, **{name: strides[name] - 8}))) == 1


def test_front_end_refuses_wrong_tensors():
    bf = torch.bfloat16
    pool, table, length = torch.zeros(2, 10, 3, 16, 128, dtype=bf), torch.zeros(4, 5, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for args in (([], table, length), ([pool[0]], table, length), ([pool, pool[:, :9]], table, length), ([pool.half()], table, length),
                 ([pool[..., ::2]], table, length), ([pool], table.long(), length), ([pool], table[:, ::2], length),
                 ([pool], table[0], length), ([pool], table, length[:3]), ([pool], table, length.long()),
                 ([pool], table, length, torch.zeros(9, dtype=torch.int32)), ([pool] * 9, table, length),
                 ([pool], table, length)):  # not on a GPU
        with pytest.raises(ValueError):
            PagedCache(*args)
    rows, row0 = torch.zeros(2, 4, 3, 7, 128, dtype=bf), torch.zeros(4, dtype=torch.int32)
    for args in ((pool[0], table, row0, rows), (pool, table, row0[:2], rows), (pool, table.long(), row0, rows),
                 (pool, table, row0, rows[0]), (pool, table, row0, rows[:1]), (pool, table, row0, rows.float()),
                 (pool, table, row0, rows[..., :64]), (pool, table, row0, rows)):
        with pytest.raises(ValueError):
            pages_write(*args)
    for args in ((pool, table, row0, -1), (pool, table, row0, 7), (pool, table, row0, 7, rows[:, :, :, :6]), (pool, table, row0.long(), 7)):
        with pytest.raises(ValueError):
            pages_read(*args)
