"""Sequences that share pages of the 4-bit cache: the step's pages, counts, slots and copies against a
plain implementation, what the sequences then hold row by row, attention over shared pages."""

import random

import numpy as np
import pytest

from kv4_shared_ref import SharedPlan

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def make(**kw):
    from mirror_sd_amd.kv4 import KV4Cache
    args = dict(n_kv_heads=2, n_pages=60, max_seqs=6, max_len=512, page=32, shared=True)
    args.update(kw)
    return KV4Cache(**args)


def state(c):
    torch.cuda.synchronize()
    return [x.cpu().clone() for x in (c.lens, c.table, c.refs, c.n_free)]


def check_state(c, plan):
    lens, table, refs, n_free = state(c)
    want = torch.full_like(table, -1)
    for s, t in enumerate(plan.table):
        want[s, :len(t)] = torch.tensor(t, dtype=torch.int32)
    assert lens.tolist() == plan.lens
    assert torch.equal(table, want)
    assert refs.tolist() == plan.refs()
    assert n_free.item() == plan.refs().count(0)


def check_step(c, plan, grow, keep=None, parent=None, max_rows=None):
    """The step on both sides; its new slots."""
    max_rows = sum(grow) if max_rows is None else max_rows
    before = state(c)
    step = c.step(grow=grow, keep=keep, max_rows=max_rows, parent=parent)
    (starts, slots, pos), copies, err = plan.step(grow, keep, parent, max_rows)
    assert c.errors() == err
    if err:
        after = state(c)
        for x, y in zip(before[:3], after[:3]):
            assert torch.equal(x, y)
    else:
        check_state(c, plan)
    assert step.starts.tolist() == starts
    assert step.slots.tolist() == slots
    assert step.positions.tolist() == pos
    return step, copies


def random_step(rng, plan, page, cap, most):
    n = len(plan.lens)
    parent = [rng.randrange(n) if rng.random() < 0.4 else s for s in range(n)]
    keep = [rng.choice([plan.lens[p], plan.lens[p], rng.randint(0, plan.lens[p]), 0,
                        plan.lens[p] // page * page]) for p in parent]
    grow = [min(cap - k, rng.choice([0, 0, 1, rng.randint(0, most)])) for k in keep]
    return parent, keep, grow


@pytest.mark.parametrize("page,seqs,seed", [(32, 6, 0), (64, 6, 1), (128, 3, 2), (256, 2, 3), (32, 1, 4),
                                            (32, 70, 5), (32, 300, 6)])
def test_random_steps(page, seqs, seed):
    rng = random.Random(seed)
    cap = 16 * page
    pool = 9 * seqs + 5
    c = make(page=page, n_pages=pool, max_seqs=seqs, max_len=cap)
    plan = SharedPlan(seqs, page, 16, pool)
    done = 0
    for i in range(40):
        parent, keep, grow = random_step(rng, plan, page, cap, 3 * page)
        if i % 7 == 3:
            parent = None
            keep = [rng.randint(0, x) for x in plan.lens]
            grow = [min(cap - k, g) for k, g in zip(keep, grow)]
        if i % 11 == 5:
            keep = None
            grow = [min(cap - plan.lens[p], g) for p, g in zip(parent or range(seqs), grow)]
        before = plan.lens
        check_step(c, plan, grow, keep, parent, sum(grow) + rng.choice([0, 0, 5]))
        done += plan.lens != before
    assert done > 5


def values(x):
    import kv4_ref as R
    return R.values(x)


@pytest.mark.parametrize("layers,kv,page", [(1, 1, 32), (3, 2, 64), (2, 5, 128)])
def test_sequences_hold_their_rows(layers, kv, page):
    """Every sequence's rows, in every layer, after every step of a random run: those of its parent,
    then its own, whatever others write."""
    rng, g = random.Random(page), torch.Generator().manual_seed(page)
    seqs, cap = 7, 8 * page
    c = make(n_kv_heads=kv, n_pages=60, max_seqs=seqs, max_len=cap, page=page, n_layers=layers)
    plan = SharedPlan(seqs, page, 8, 60)
    held = [np.zeros((0, layers, 2, kv, 128)) for _ in range(seqs)]
    for _ in range(14):
        parent, keep, grow = random_step(rng, plan, page, cap, page + 9)
        lens = plan.lens
        step, copies = check_step(c, plan, grow, keep, parent)
        if plan.lens == lens and not sum(grow):
            continue
        if plan.lens != [k + n for k, n in zip(keep, grow)]:
            continue
        x = torch.randn((sum(grow), layers, 2, kv, 128), generator=g).half().cuda()
        for l in range(layers):
            c.append(x[:, l, 0], x[:, l, 1], step.slots, l)
        new, at = values(x.double().cpu().numpy()), 0
        old = held
        held = []
        for s in range(seqs):
            held.append(np.concatenate((old[parent[s]][:keep[s]], new[at:at + grow[s]])))
            at += grow[s]
        for s in range(seqs):
            rows = [plan.table[s][r // page] * page + r % page for r in range(plan.lens[s])]
            for l in range(layers):
                k, v = c.read(rows, l, dtype=torch.float32)
                np.testing.assert_array_equal(k.double().cpu().numpy(), held[s][:, l, 0])
                np.testing.assert_array_equal(v.double().cpu().numpy(), held[s][:, l, 1])
    assert c.errors() == 0


def test_all_candidates_write_the_first_stays():
    c = make(max_seqs=5)
    plan = SharedPlan(5, 32, 16, 60)
    check_step(c, plan, [40, 0, 0, 0, 0])
    _, copies = check_step(c, plan, [3] * 5, [40] * 5, [0] * 5)
    assert len(copies) == 4 and plan.table[0][1] == 1          # sequence 0 goes on in its own page
    # a holder that does not write: the one that does copies
    check_step(c, plan, [0] * 5, [40, 40, 40, 0, 0], [0, 0, 0, 3, 4])
    _, copies = check_step(c, plan, [1, 0, 0, 0, 0])
    assert len(copies) == 1
    # rows that end with a page: nothing to copy
    check_step(c, plan, [0] * 5, [32] * 5, [1] * 5)
    _, copies = check_step(c, plan, [2] * 5)
    assert not copies
    # a kept row less than what others hold
    check_step(c, plan, [0] * 5, [34] * 5, [2] * 5)
    _, copies = check_step(c, plan, [4, 4, 4, 0, 0], [33, 34, 1, 34, 0])
    assert [n for _, _, n in copies] == [1, 2, 1]   # sequences 0, 1, 2: what they hold others hold too


def test_sequences_change_places():
    c = make(max_seqs=4)
    plan = SharedPlan(4, 32, 16, 60)
    check_step(c, plan, [50, 70, 1, 0])
    check_step(c, plan, [0] * 4, None, [1, 0, 3, 2])
    check_step(c, plan, [1] * 4, None, [3, 2, 1, 0])
    check_step(c, plan, [0] * 4, [0] * 4, [3, 2, 1, 0])
    assert plan.refs() == [0] * 60


@pytest.mark.parametrize("what,bit", [("keep", 8), ("grow", 8), ("parent", 8), ("low", 8), ("pool", 16),
                                      ("rows", 32)])
@pytest.mark.parametrize("seqs", [6, 1100])
def test_steps_that_cannot_be_done_change_nothing(what, bit, seqs):
    c = make(max_seqs=seqs, n_pages=60, max_len=512)
    plan = SharedPlan(seqs, 32, 16, 60)
    check_step(c, plan, [100, 40] + [0] * (seqs - 2))
    grow, keep, parent = [7] * 3 + [0] * (seqs - 3), [90, 33, 90] + [0] * (seqs - 3), [0, 1, 0] + list(range(3, seqs))
    if what == "keep":
        keep[1] = 41
    elif what == "grow":
        grow[seqs - 1] = 513
    elif what == "parent":
        parent[2] = seqs
    elif what == "low":
        parent[2], keep[2] = -1, 0
    elif what == "pool":
        grow[0], grow[1], grow[2] = 400, 470, 422
        grow[3:6] = [512, 512, 512]
    check_step(c, plan, grow, keep, parent, sum(grow) - (what == "rows"))
    check_step(c, plan, [1] * 3 + [0] * (seqs - 3), [90, 33, 90] + [0] * (seqs - 3), [0, 1, 0] + list(range(3, seqs)))


@pytest.mark.parametrize("seqs", [4, 1100])
def test_page_ids_outside_the_pool_refuse_the_step(seqs):
    c = make(max_seqs=seqs)
    plan = SharedPlan(seqs, 32, 16, 60)
    check_step(c, plan, [100, 40] + [0] * (seqs - 2))
    idle = [0] * (seqs - 2)
    for row, col, page in ((0, 1, 60), (0, 0, -1), (1, 1, 2**31 - 1)):
        was = c.table[row, col].item()
        c.table[row, col] = page
        before = state(c)
        s = c.step(grow=[1, 1] + idle, keep=[32, 33] + idle, parent=[1, 0] + list(range(2, seqs)), max_rows=4)
        assert c.errors() == 128 and s.starts.tolist() == [0] * (seqs + 1) and s.slots.tolist() == [-1] * 4
        for x, y in zip(before[:3], state(c)[:3]):
            assert torch.equal(x, y)
        c.table[row, col] = was
    check_step(c, plan, [1, 1] + idle, [32, 33] + idle, [1, 0] + list(range(2, seqs)))


@pytest.mark.parametrize("seqs,page,rows", [(1100, 32, 3), (40, 32, 400), (20, 256, 700)])
def test_steps_in_several_launches(seqs, page, rows):
    rng = random.Random(rows)
    width = 2048 // page
    pool = 70000 if seqs == 20 else 8 * seqs * max(1, rows // page + 2)
    c = make(n_kv_heads=1, max_seqs=seqs, page=page, max_len=2048, n_pages=pool)
    plan = SharedPlan(seqs, page, width, pool)
    check_step(c, plan, [rng.randint(1, rows) for _ in range(seqs)])
    for _ in range(4):
        parent = [rng.randrange(seqs) if rng.random() < 0.5 else s for s in range(seqs)]
        keep = [rng.choice([plan.lens[p], rng.randint(0, plan.lens[p])]) for p in parent]
        grow = [min(2048 - k, rng.randint(0, rows)) for k in keep]
        check_step(c, plan, grow, keep, parent, sum(grow) + 9000 * (rows > 3))


def test_a_captured_step_is_replayed():
    """A graph of a step and its copies, with eager steps between its replays."""
    c = make(max_seqs=6, n_layers=2, n_pages=100)
    plan = SharedPlan(6, 32, 16, 100)
    check_step(c, plan, [45, 60, 0, 0, 0, 0])
    grow, keep, parent = (torch.zeros(6, dtype=torch.int32, device="cuda") for _ in range(3))
    parent.copy_(torch.arange(6))
    keep.copy_(c.lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.step(grow=grow, keep=keep, parent=parent, max_rows=40)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = c.step(grow=grow, keep=keep, parent=parent, max_rows=40)
    rng = random.Random(4)
    for i in range(6):
        p, k, g = random_step(rng, plan, 32, 512, 6)
        for dst, src in ((parent, p), (keep, k), (grow, g)):
            dst.copy_(torch.tensor(src))
        graph.replay()
        (starts, slots, pos), _, err = plan.step(g, k, p, 40)
        assert not err and c.errors() == 0
        check_state(c, plan)
        assert s.starts.tolist() == starts and s.slots.tolist() == slots and s.positions.tolist() == pos
        check_step(c, plan, [2, 0, 1, 0, 0, 0], None, [0, 0, 2, 3, 4, 5])


def test_two_caches_on_two_streams():
    rng = random.Random(9)
    plans = [SharedPlan(5, 32, 16, 60) for _ in range(2)]
    caches = [make(max_seqs=5) for _ in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(12):
        for c, plan, st in zip(caches, plans, streams):
            parent, keep, grow = random_step(rng, plan, 32, 512, 20)
            with torch.cuda.stream(st):
                c.step(grow=grow, keep=keep, parent=parent)
            plan.step(grow, keep, parent, sum(grow))
    torch.cuda.synchronize()
    for c, plan in zip(caches, plans):
        check_state(c, plan)


def test_refusals():
    from mirror_sd_amd.kv4 import KV4Cache
    c = KV4Cache(n_kv_heads=1, n_pages=4, max_seqs=2, max_len=64)
    assert c.refs is None and c.free is not None
    with pytest.raises(ValueError, match="shared"):
        c.step(parent=[0, 0])
    c = make()
    assert c.free is None
    with pytest.raises(ValueError):
        c.step(parent=[0] * 5)
    with pytest.raises(ValueError):
        c.step(parent=[0.5] * 6)
    with pytest.raises(ValueError):
        KV4Cache(n_kv_heads=1, n_pages=4, max_seqs=65536, max_len=2**19, page=32, shared=True)
