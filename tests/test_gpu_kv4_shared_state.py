"""Steps of a shared cache whose arguments are the cache's own state."""

import pytest

from kv4_shared_ref import SharedPlan
from test_gpu_kv4_shared import check_state, check_step, make

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("seqs", [6, 1100])   # one workgroup, launches
def test_lengths_as_they_are_on_the_gpu(seqs):
    """keep=c.lens: what the step reads of it is what it was before the step."""
    c = make(max_seqs=seqs, n_pages=200)
    plan = SharedPlan(seqs, 32, 16, 200)
    rest = [0] * (seqs - 6)
    check_step(c, plan, [40, 40, 40, 7, 0, 0] + rest)
    for grow, parent in (([1, 2, 3, 4, 0, 5], [0, 1, 2, 3, 4, 5]), ([30, 0, 1, 64, 33, 2], [0, 1, 2, 3, 4, 5])):
        s = c.step(grow=grow + rest, keep=c.lens, parent=parent + list(range(6, seqs)))
        (starts, slots, pos), _, err = plan.step(grow + rest, list(plan.lens), parent + list(range(6, seqs)), sum(grow))
        assert err == 0 and c.errors() == 0
        check_state(c, plan)
        assert s.starts.tolist() == starts and s.slots.tolist() == slots and s.positions.tolist() == pos
    # as rows to grow by, too: every sequence doubles, from its neighbour
    keep = [plan.lens[s ^ 1] if s < 6 else 0 for s in range(seqs)]
    parent = [s ^ 1 if s < 6 else s for s in range(seqs)]
    grow, n = list(plan.lens), sum(plan.lens)
    s = c.step(grow=c.lens, keep=torch.tensor(keep, dtype=torch.int32, device="cuda"), parent=parent, max_rows=n)
    (starts, slots, pos), _, err = plan.step(grow, keep, parent, n)
    assert err == 0 and c.errors() == 0
    check_state(c, plan)
    assert s.starts.tolist() == starts and s.slots.tolist() == slots and s.positions.tolist() == pos
