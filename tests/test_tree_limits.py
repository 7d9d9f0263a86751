"""The sizes that esda_tree.h names as the largest, on the host: the next ones are refused, by name."""
import pytest

from apertura_amd import _lib
from apertura_amd.tree import tree_workspace_bytes
from test_overlaps import AT, N, _calls, _pool, _step


@pytest.mark.parametrize("batch,nodes,hq,hkv,D", [(256, 64, 512, 32, 128), (256, 64, 256, 16, 256), (128, 64, 256, 16, 512), (256, 32, 512, 32, 256)])
def test_query_rows_of_a_step(batch, nodes, hq, hkv, D):
    """batch * nodes * num_q_heads * head_dim is 2^30, then less."""
    kw = dict(num_q_heads=hq, num_kv_heads=hkv, head_dim=D, num_pages=256 * N)
    assert batch * nodes * hq * D == 2 ** 30
    with pytest.raises(_lib.EsdaError) as ei:
        tree_workspace_bytes(_step(batch=batch, nodes=nodes, **kw))
    assert ei.value.code == 1 and "query rows" in str(ei.value)
    assert tree_workspace_bytes(_step(batch=batch - 1, nodes=nodes, **kw)) > 0
    assert tree_workspace_bytes(_step(batch=batch, nodes=nodes - 1, **kw)) > 0


def test_splits_of_a_step():
    """A room of 4,096 splits of 32 rows (the nodes' rows are the last five), then of one more."""
    for rows, taken in ((4096 * 32 - 16, True), (4096 * 32, False)):
        step = _step(max_pages=rows // 16, split_rows=32)
        if taken:
            assert tree_workspace_bytes(step) > 0
        else:
            with pytest.raises(_lib.EsdaError) as ei:
                tree_workspace_bytes(step)
            assert ei.value.code == 1 and "splits" in str(ei.value)


@pytest.mark.parametrize("planes,heads,D,slots", [(4096, 64, 512, 256), (1024, 8, 256, 2 ** 14), (33, 8, 128, 2 ** 19)])
def test_workgroups_of_a_commit(planes, heads, D, slots):
    """slots * groups is 2^23 or below, then above."""
    groups = (planes * heads * D + 4095) // 4096
    assert groups * slots <= 2 ** 23
    lists = dict(table=AT + (1 << 50), length=AT + (1 << 51))

    def commit(slots, pools=1):  # (refused for its workspace where the sizes are taken)
        return _calls([_pool(x << 42, planes, heads, D) for x in range(pools)], slots=slots, **lists)["commit"]

    assert commit(slots)[0] == 4
    for code, why in (commit(slots + 1) if groups * slots == 2 ** 23 else commit(2 ** 23 // groups, 2),
                      commit(slots, 1 + 2 ** 23 // (groups * slots))):
        assert code == 1 and "too many slots" in why
