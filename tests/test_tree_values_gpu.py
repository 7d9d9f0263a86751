"""esda_tree_decode: values that no query may see, whatever they are, and queries that are no node's.  Where
such a value only may not be seen, the outputs are compared bit by bit with those beside ordinary values."""
import pytest
import torch

from _attn64 import check
from apertura_amd.tree import TreeCall, tree_decode
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


@pytest.mark.parametrize("split_rows", [0, 32])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("window", [0, 64])
def test_rows_that_nobody_sees(form, window, split_rows):
    """Rows of nodes that are none, rows before every window and rows of a page that is none enter with a weight
    of 0 and nothing of theirs: NaN and infinities there cost no bit of a row that does not see them."""
    c = _case(*form, split_rows=split_rows, window=max(window, form[4]) if window else 0)
    none = _none(c)
    # (an entry of the table that is no page; page 0 is nobody's)
    used = set(c.table[c.table >= 0].tolist())
    if 0 in used:
        free = next(i for i in range(c.pool.shape[1]) if i not in used)
        c.pool[:, free] = c.pool[:, 0]
        c.table[c.table == 0] = free
    c.table[0, 42] = -1  # rows 672 .. 687 of 700
    c.pool[:, 0] = 0.0
    clean = c.full.nan_to_num(nan=0.5)
    want = None
    for bad in (1.0, float("nan"), float("inf"), -float("inf")):
        c.full.copy_(clean)
        if bad != 1.0:  # before the windows, behind the last rows, pages of nobody
            c.pool[:, 0] = bad
            for b, n in enumerate(c.lengths):
                for r in range(max(0, n - c.window + 1) if c.window else 0):
                    if int(c.table[b, r // 16]) >= 0:
                        c.pool[:, int(c.table[b, r // 16]), :, r % 16] = bad
        kn, vn = c.kn.clone(), None if c.shared else c.vn.clone()
        for x in (kn, vn):
            if x is not None:
                x[none] = bad
        out = tree_decode(c.step, **dict(c.args(), k_new=kn, v_new=vn))
        assert bool(torch.isfinite(out).all())
        want = out if want is None else want
        assert torch.equal(out, want), bad


@pytest.mark.parametrize("form", FORMS)
def test_steps_repeat_themselves(form):
    """Whichever workgroup ends first, the sums are taken in the same order."""
    c = _case(*form)
    want = tree_decode(c.step, **c.args())
    for _ in range(5):
        assert torch.equal(tree_decode(c.step, **c.args()), want)


def test_calls_with_another_current_device_are_refused(monkeypatch):
    """A launch goes to the current device's stream, where the tensors are not."""
    c = _case(*FORMS[0])
    call = TreeCall(c.step, **c.args())
    want = call().clone()
    call.out.fill_(7.0)
    with monkeypatch.context() as m:
        m.setattr(torch._C, "_cuda_getDevice", lambda: 1)
        with pytest.raises(ValueError):
            call()
    assert bool((call.out == 7.0).all())
    assert torch.equal(call(), want)
