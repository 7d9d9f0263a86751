"""esda_tree_decode: values that no query may see, whatever they are, and queries that are no node's.  Where
such a value only may not be seen, the outputs are compared bit by bit with those beside ordinary values."""
import pytest
import torch

from _attn64 import check
from apertura_amd.tree import tree_decode
from test_tree_gpu import Case, random_parents

pytestmark = pytest.mark.gpu
DEV = "cuda"

# D, query heads, kv heads, K = V, nodes, room in rows: runs of 16 and 32 query rows, runs of 512 dims (short ones in
# groups of stages), and each form of the tiles
FORMS = [(128, 8, 2, False, 4, 800), (128, 8, 2, False, 12, 800), (128, 32, 8, False, 6, 20000), (256, 4, 2, False, 5, 800),
         (512, 8, 1, True, 2, 800), (512, 4, 2, False, 5, 800), (128, 32, 8, False, 40, 20000), (256, 32, 16, False, 64, 9000),
         (256, 32, 16, False, 20, 9000), (512, 32, 4, True, 8, 9000), (512, 32, 4, True, 64, 9000), (512, 8, 4, False, 64, 9000)]


def _case(D, hq, hkv, shared, T, room, lengths=(700, 90, 0), **kw):
    parent = random_parents(len(lengths), T, 5)
    parent[:, T - 1] = -2
    parent[1, T // 2:] = T  # the second half no nodes
    return Case(T, hq, hkv, D, list(lengths), 16, shared, parent=parent, spare=(room - max(lengths)) // 16, seed=T, **kw)


def _none(c):
    return torch.tensor([[not path for path in paths] for paths in c.paths], device=DEV)


@pytest.mark.parametrize("split_rows", [0, 32, 2 ** 31 - 32])
@pytest.mark.parametrize("form", FORMS)
def test_queries_of_no_node(form, split_rows):
    """Whatever q holds where there is no node: zeros there, and the others' outputs as they are."""
    c = _case(*form, split_rows=split_rows)
    none = _none(c)
    want = tree_decode(c.step, **c.args())
    assert not bool(want[none].any())
    inf = float("inf")
    for bad in (inf, -inf, float("nan"), 3e38, [inf], [-inf]):
        q = c.q.clone()
        if isinstance(bad, list):  # in one dim: scores of either infinity
            q[..., 5][none] = bad[0]
        else:
            q[none] = bad
        out = tree_decode(c.step, **dict(c.args(), q=q))
        assert not bool(out[none].any() | out[none].isnan().any()), bad
        assert torch.equal(out, want), bad
