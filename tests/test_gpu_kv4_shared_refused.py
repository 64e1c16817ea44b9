"""Steps of sequences that share pages which cannot be done: nothing changes, the number of free pages and
what the pool holds among it, in one workgroup and in several launches."""

import pytest

from kv4_shared_ref import SharedPlan
from test_gpu_kv4_shared import check_step, make, state

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

PAGES = 60


def filled(seqs):
    """A cache whose sequences 0 and 1 hold rows that others can go on from inside of a page, with bytes
    in all of its pages."""
    c = make(max_seqs=seqs, n_pages=PAGES, max_len=512, n_layers=2)
    plan = SharedPlan(seqs, 32, 16, PAGES)
    check_step(c, plan, [100, 40] + [0] * (seqs - 2))
    c.pool.copy_(torch.randint(256, c.pool.shape, generator=torch.Generator().manual_seed(1), dtype=torch.uint8))
    return c, plan


def asked(seqs):
    """Three that go on, each inside a page that others hold: copies in both layers."""
    idle = seqs - 3
    return [7] * 3 + [0] * idle, [90, 33, 90] + [0] * idle, [0, 1, 0] + list(range(3, seqs))


def check_refused(c, before, pool, n_rows, seqs, step, err):
    assert c.errors() == err
    after = state(c)
    assert len(before) == 4
    for x, y in zip(before, after):
        assert torch.equal(x, y)
    assert torch.equal(c.pool, pool)
    assert step.starts.tolist() == [0] * (seqs + 1)
    assert step.slots.tolist() == step.positions.tolist() == [-1] * n_rows


@pytest.mark.parametrize("seqs", [6, 1100])   # one workgroup, launches
@pytest.mark.parametrize("what,err", [("keep", 8), ("negative", 8), ("grow", 8), ("parent", 8), ("pool", 16),
                                      ("one_page", 16), ("rows", 32), ("page", 128), ("edge", 128), ("given_up", 128)])
def test_nothing_changes(what, err, seqs):
    c, plan = filled(seqs)
    grow, keep, parent = asked(seqs)
    n_rows = sum(grow)
    if what == "keep":
        keep[1] = 41
    elif what == "negative":
        grow[2] = -1
    elif what == "grow":
        grow[seqs - 1] = 513
    elif what == "parent":
        parent[2] = seqs
    elif what == "pool":
        grow[0], grow[1], grow[2] = 400, 470, 422
        grow[3:6] = [512, 512, 512]
        n_rows = sum(grow)
    elif what == "one_page":      # 54 pages are free; the copies (of 0's third page, of none of 1's) decide
        grow[3:6] = [512, 512, 512]
        grow[0], grow[1], grow[2] = 7 + 31, 33, 7
        n_rows = sum(grow)
        held = SharedPlan(seqs, 32, 16, PAGES)
        held.table, held.lens = [list(t) for t in plan.table], list(plan.lens)
        while held.step(grow, keep, parent, 10**6)[2] == 0:     # the smallest step that one page is short for
            held.table, held.lens = [list(t) for t in plan.table], list(plan.lens)
            grow[1] += 1
            n_rows += 1
    elif what == "rows":
        n_rows -= 1
    elif what == "page":
        c.table[0, 1] = PAGES
    elif what == "edge":
        c.table[0, 2] = -1
    elif what == "given_up":
        parent[1], keep[1] = 0, 33                              # 1 gives up its pages for 0's
        c.table[1, 1] = 2**31 - 1
    before, pool = state(c), c.pool.clone()
    step = c.step(grow=grow, keep=keep, parent=parent, max_rows=n_rows)
    check_refused(c, before, pool, n_rows, seqs, step, err)
    # the same again, then one that can be done
    step = c.step(grow=grow, keep=keep, parent=parent, max_rows=n_rows)
    check_refused(c, before, pool, n_rows, seqs, step, err)
    if err != 128:
        before = list(plan.table)
        _, copies = check_step(c, plan, *asked(seqs))
        assert copies and before != plan.table
        for src, dst, kept in copies:
            blocks = -(-kept // 32)
            assert torch.equal(c.pool[:, dst, :, :blocks], pool[:, src, :, :blocks])


@pytest.mark.parametrize("seqs", [6, 1100])
def test_captured_steps_that_are_refused_in_turn(seqs):
    """A graph of a step whose lengths fit every second time: no copies are left over from the one before."""
    c, plan = filled(seqs)
    ints = dict(dtype=torch.int32, device="cuda")
    grow, keep, parent = (torch.tensor(x, **ints) for x in asked(seqs))
    start = [t.clone() for t in (c.lens, c.table, c.refs, c.n_free, c.pool)]
    n_rows = 30

    def again():
        for t, was in zip((c.lens, c.table, c.refs, c.n_free, c.pool), start):
            t.copy_(was)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.step(grow=grow, keep=keep, parent=parent, max_rows=n_rows)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = c.step(grow=grow, keep=keep, parent=parent, max_rows=n_rows)
    again()
    for i in range(6):
        if i % 2 == 0:            # done
            graph.replay()
            assert c.errors() == 0 and s.slots[0].item() >= 0
            again()
        else:
            keep[1] = 41
            before, pool = state(c), c.pool.clone()
            graph.replay()
            check_refused(c, before, pool, n_rows, seqs, s, 8)
            keep[1] = 33
