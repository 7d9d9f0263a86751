"""GPU parity of every kernel of esda_tree_decode, with K and V apart and one, with a merge and without."""
import pytest

from _tree_forms import STEPS
from test_tree_gpu import Case, random_parents

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("step,shared,form", STEPS)
def test_every_kernel(step, shared, form, window):
    """Trees with holes over sequences of several lengths, all room of the table theirs (a window of 70 rows may
    take another kernel; its keys are few)."""
    D, hq, hkv, T, lengths, room, split = step
    parent = random_parents(len(lengths), T, D + T, 0.1)
    c = Case(T, hq, hkv, D, lengths, 16, shared, window, parent=parent, split_rows=split, spare=room // 16 - (max(lengths) + T + 15) // 16, seed=T)
    assert c.step.max_pages * c.step.page_rows == room
    c.run()
