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


# ------------------------------------------------------------------ attention over shared pages

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def rows(n, kv, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, 2, kv, 128), generator=g)
    x[:, 0, :, ::41] *= 6
    return x.to(dtype).cuda()


def family(kv, page, sizes, prefix, own, dtype, seed=0, spare=3, room=0):
    """A cache in which the sequences of group g go on from one text of prefix[g] rows, each by own[s]
    of its own: (cache, what every sequence holds in 64 bits, group boundaries)."""
    n = sum(sizes)
    first = [sum(sizes[:g]) for g in range(len(sizes) + 1)]
    of = [g for g, m in enumerate(sizes) for _ in range(m)]
    lens = [prefix[g] + o for g, o in zip(of, own)]
    pool = sum(-(-p // page) for p in prefix) + sum(-(-x // page) + 1 for x in lens) + spare
    c = make(n_kv_heads=kv, max_seqs=n, max_len=max(max(lens), 1) + room, page=page, n_pages=pool)
    heads = [rows(p, kv, 10 * seed + g, dtype) for g, p in enumerate(prefix)]
    mine = [rows(o, kv, 1000 + 10 * seed + s, dtype) for s, o in enumerate(own)]
    step = c.step(grow=[prefix[g] if s == first[g] else 0 for s, g in enumerate(of)])
    x = torch.cat(heads)
    c.append(x[:, 0], x[:, 1], step.slots)
    step = c.step(grow=own, keep=[prefix[g] for g in of], parent=[first[g] for g in of])
    x = torch.cat(mine)
    c.append(x[:, 0], x[:, 1], step.slots)
    assert c.errors() == 0
    import kv4_ref as R
    held = [R.values(torch.cat((heads[g], mine[s])).double().cpu().numpy()) for s, g in enumerate(of)]
    return c, held, first


def queries(n, heads, seed, dtype):
    g = torch.Generator().manual_seed(seed + 77)
    return (1.5 * torch.randn((n, heads, 128), generator=g)).to(dtype).cuda()


def check_rows(q, starts, held, causal, out, lse=None, scale=128 ** -0.5):
    """Within the bound of one attention; the join adds two powers and products to a state, 24 fp32
    roundings at most where both parts weigh more than 2^-20 (as 768 more keys would)."""
    import kv4_ref as R
    half = torch.finfo(q.dtype).eps / 2
    for s, kv in enumerate(held):
        a, b = starts[s], starts[s + 1]
        if a == b:
            continue
        o, l, mass, size = R.attend(q[a:b].double().cpu().numpy(), kv[:, 0], kv[:, 1], causal, scale)
        tol, ltol = R.attend_tolerance(o, l, mass, size, len(kv) + 768, half)
        off = np.abs(out[a:b].double().cpu().numpy() - o)
        assert (off <= tol).all(), (s, float((off / tol).max()))
        if lse is not None:
            got = lse[a:b].double().cpu().numpy()
            empty = np.isneginf(l)
            assert (np.isneginf(got) == empty).all()
            assert (np.abs(got[~empty] - l[~empty]) <= ltol[~empty]).all(), s


def ends(x):
    return np.concatenate(([0], np.cumsum(x))).astype(int).tolist()


FAMILIES = [  # heads, kv, page, sizes, prefix, own rows, q rows
    (4, 2, 32, [2], [64], [1, 1], [1, 1]),
    (8, 2, 32, [3, 2], [100, 700], [1, 40, 33, 64, 5], [1, 1, 1, 1, 1]),
    (32, 8, 64, [9], [513], [1, 2, 3, 4, 5, 64, 65, 63, 128], [1] * 9),
    (5, 5, 64, [4, 1, 3], [31, 0, 64], [3, 90, 4, 1, 1, 2, 3, 4], [1] * 8),
    (16, 2, 32, [4], [333], [8, 9, 40, 8], [8, 8, 8, 8]),
    (6, 2, 128, [3, 3], [257, 1000], [20, 30, 40, 50, 60, 20], [20, 7, 0, 33, 1, 20]),
    (64, 1, 32, [5, 1], [160, 5], [1, 1, 1, 1, 1, 1], [1] * 6),
    (2, 1, 256, [40], [300], [1 + i % 7 for i in range(40)], [1] * 40),
    (4, 1, 32, [2, 2], [96, 96], [150, 131, 0, 0], [130, 131, 0, 0]),
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv,page,sizes,prefix,own,q_lens", FAMILIES)
def test_attend_shared(heads, kv, page, sizes, prefix, own, q_lens, causal, dtype):
    c, held, groups = family(kv, page, sizes, prefix, own, DT[dtype], seed=heads)
    starts = ends(q_lens)
    q = queries(starts[-1], heads, page, DT[dtype])
    out, lse = c.attend(q, starts, causal=causal, return_lse=True, groups=groups)
    assert c.errors() == 0
    check_rows(q, starts, held, causal, out, lse)
    assert torch.equal(c.attend(q, starts, causal=causal, groups=groups), out)
    # each sequence a group of its own: nothing is shared
    alone = list(range(len(q_lens) + 1))
    check_rows(q, starts, held, causal, c.attend(q, starts, causal=causal, groups=alone))
    # a boundary in the middle of a family, and sequences that no group names
    check_rows(q, starts, held, causal, c.attend(q, starts, causal=causal, groups=[1, len(q_lens)]))


def test_long_shared_text():
    """20 thousand shared rows: partials of the shared part in many workers."""
    c, held, groups = family(2, 64, [7, 3], [20001, 5000], [30 + s for s in range(10)], torch.float16)
    for m in (1, 5):
        starts = ends([m] * 10)
        q = queries(10 * m, 8, m, torch.float16)
        out, lse = c.attend(q, starts, causal=True, return_lse=True, groups=groups)
        check_rows(q, starts, held, True, out, lse)


def test_sequences_that_no_longer_agree():
    """Pages are shared as far as the tables agree from the first on, and no further."""
    c, held, groups = family(2, 32, [4], [320], [5, 6, 7, 8], torch.float16)
    q = queries(4, 4, 3, torch.float16)
    starts = [0, 1, 2, 3, 4]
    for s, page in ((2, 6), (3, 3), (1, 9), (0, 0)):
        # sequence s gets a page of its own for these rows, with other rows in it
        spare = (c.refs == 0).nonzero()[0].item()
        x = rows(32, 2, 50 + s, torch.float16)
        c.append(x[:, 0], x[:, 1], torch.arange(32 * spare, 32 * spare + 32).to(torch.int32))
        c.refs[spare] += 1
        c.table[s, page] = spare
        held[s][32 * page:32 * page + 32] = values(x.double().cpu().numpy())
        check_rows(q, starts, held, False, c.attend(q, starts, groups=groups))
    assert c.errors() == 0


@pytest.mark.parametrize("m", [1, 31, 33, 100])
def test_new_rows_inside_shared_pages(m):
    """Sequences that share all of their pages, the new rows' too: with causal, keys that some row
    does not see are not taken for all."""
    c, held, groups = family(2, 32, [3], [130], [0, 0, 0], torch.float16)
    starts = ends([m, m, m])
    q = queries(3 * m, 4, 5, torch.float16)
    for causal in (True, False):
        out, lse = c.attend(q, starts, causal=causal, return_lse=True, groups=groups)
        check_rows(q, starts, held, causal, out, lse)
    c.lens.zero_()
    out, lse = c.attend(q, starts, causal=True, return_lse=True, groups=groups)
    assert not out.any() and torch.isneginf(lse).all() and c.errors() == 0


def test_idle_sequences_do_not_count():
    c, held, groups = family(1, 32, [5], [200], [4, 4, 4, 4, 4], torch.bfloat16)
    c.step(keep=[204, 0, 204, 30, 204])                       # 1 is finished, 3 cut short
    starts = [0, 2, 2, 4, 4, 6]
    q = queries(6, 8, 6, torch.bfloat16)
    check_rows(q, starts, held, False, c.attend(q, starts, groups=groups))
    check_rows(q, starts, held, True, c.attend(q, starts, causal=True, groups=groups))


def test_groups_and_pages_that_do_not_fit():
    from mirror_sd_amd import kv4
    c, held, groups = family(2, 32, [3, 2], [100, 70], [4, 5, 6, 7, 8], torch.float16)
    starts = [0, 1, 2, 3, 4, 5]
    q = queries(5, 4, 7, torch.float16)
    for bad in ([0, 4, 3, 5], [-1, 3, 5], [0, 3, 6], [3, 0], [0, 2**31 - 1]):
        out = c.attend(q, starts, groups=bad)
        assert c.errors() == kv4.ERR_PAGE, bad
        check_rows(q, starts, held, False, out)
    # a page outside the pool in the shared text: its keys are absent for all
    table = c.table.clone()
    for page in (-1, c.n_pages, 2**31 - 1):
        c.table[:3, 1] = page
        out = c.attend(q, starts, groups=groups)
        assert c.errors() == kv4.ERR_PAGE
        want = [np.concatenate((h[:32], h[64:])) for h in held[:3]] + held[3:]
        check_rows(q, starts, want, False, out)
        c.table.copy_(table)
    # a length or a row range that does not fit: that sequence has no rows, the others theirs
    lens = c.lens.clone()
    for value in (-1, 2**31 - 1):
        c.lens[1] = value
        out = torch.full_like(q, 7.0)
        c.attend(q, starts, out=out, groups=groups)
        assert c.errors() == kv4.ERR_PAGE and (out[1] == 7.0).all()
        check_rows(q, [0, 1, 1, 1, 1, 1], held, False, out)
        check_rows(q[2:], [0, 0, 0, 1, 2, 3], held, False, out[2:])
        c.lens.copy_(lens)
    out = torch.full_like(q, 7.0)
    c.attend(q, [0, 1, 2, 3, 9, 5], out=out, groups=groups)
    assert c.errors() == kv4.ERR_PAGE and (out[3:] == 7.0).all()
    check_rows(q, [0, 1, 2, 3, 3, 3], held, False, out)


def test_rows_of_no_sequence_stay_and_queries_in_place():
    c, held, groups = family(2, 32, [3], [100], [4, 5, 6], torch.float16)
    q = queries(8, 4, 8, torch.float16)
    starts = [2, 3, 5, 6]
    want = c.attend(q, starts, groups=groups)
    out = torch.full_like(q, 3.0)
    c.attend(q, starts, out=out, groups=groups)
    assert (out[:2] == 3.0).all() and (out[6:] == 3.0).all() and torch.equal(out[2:6], want[2:6])
    wide = torch.randn((8, 10, 128), device="cuda").half()     # a part of a projection's row
    wide[:, 3:7] = q
    assert torch.equal(c.attend(wide[:, 3:7], starts, groups=groups)[2:6], want[2:6])
    c.attend(q, starts, out=q, groups=groups)
    assert torch.equal(q[2:6], want[2:6])


def test_what_a_row_does_not_see_of_shared_pages():
    """NaN and infinite rows past a sequence's end, in a page that it shares with one that sees them."""
    c, held, groups = family(2, 64, [3], [100], [0, 0, 0], torch.float16)
    x = rows(100, 2, 0, torch.float16)
    bad = x.clone()
    bad[96:] = float("nan")
    bad[90, 1] = float("inf")
    slots = [c.table[0, r // 64].item() * 64 + r % 64 for r in range(100)]
    c.append(bad[:, 0], bad[:, 1], slots)
    c.step(keep=[90, 100, 80])
    starts = [0, 1, 2, 3]
    q = queries(3, 4, 9, torch.float16)
    out = c.attend(q, starts, groups=groups)
    assert torch.isnan(out[1]).all()
    check_rows(q, starts, [held[0][:90], [], held[2][:80]][:1], False, out)
    check_rows(q[2:], [0, 1], [held[2][:80]], False, out[2:])


@pytest.mark.parametrize("m,heads", [(1, 8), (12, 8)])
def test_captured_steps_of_candidates(m, heads):
    """A graph of a forking step, its rows in and attention over what is shared, replayed with other
    parents, lengths, rows and groups, and eager work between."""
    c, held, _ = family(2, 32, [4, 4], [150, 90], [m] * 8, torch.float16, spare=40, room=80)
    ints = dict(dtype=torch.int32, device="cuda")
    keep, parent, grow = c.lens.clone(), torch.arange(8, **ints), torch.full((8,), m, **ints)
    groups = torch.tensor([0, 4, 8], **ints)
    x, q = rows(8 * m, 2, 1, torch.float16), queries(8 * m, heads, 1, torch.float16)
    side = torch.cuda.Stream()
    lens, table, refs, free = (t.clone() for t in (c.lens, c.table, c.refs, c.n_free))

    def step():
        s = c.step(grow=grow, keep=keep, parent=parent, max_rows=8 * m)
        c.append(x[:, 0], x[:, 1], s.slots)
        return c.attend(q, s.starts, causal=True, groups=groups)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t, was in ((c.lens, lens), (c.table, table), (c.refs, refs), (c.n_free, free)):
        t.copy_(was)
    rng = random.Random(m)
    import kv4_ref as R
    for i in range(5):
        now = c.lens.tolist()
        p = [4 * (s // 4) + rng.randrange(4) for s in range(8)]
        k = [now[j] - rng.choice([0, 0, 3]) for j in p]
        parent.copy_(torch.tensor(p))
        keep.copy_(torch.tensor(k))
        groups.copy_(torch.tensor([[0, 4, 8], [0, 8, 8], [2, 4, 7]][i % 3]))
        x.copy_(rows(8 * m, 2, 60 + i, torch.float16))
        q.copy_(queries(8 * m, heads, 60 + i, torch.float16))
        graph.replay()
        assert c.errors() == 0
        new = R.values(x.double().cpu().numpy())
        held = [np.concatenate((held[p[s]][:k[s]], new[s * m:s * m + m])) for s in range(8)]
        check_rows(q, ends([m] * 8), held, True, out)
        check_rows(q, ends([m] * 8), held, True, c.attend(q, ends([m] * 8), causal=True))
    assert c.errors() == 0


def test_two_shared_calls_at_once():
    a = family(2, 32, [6], [3000], [3] * 6, torch.float16)
    b = family(1, 64, [3, 2], [900, 2000], [20] * 5, torch.bfloat16, seed=3)
    qa, qb = queries(6, 8, 1, torch.float16), queries(100, 6, 2, torch.bfloat16)
    sa, sb = ends([1] * 6), ends([20] * 5)
    want = [a[0].attend(qa, sa, groups=a[2]), b[0].attend(qb, sb, causal=True, groups=b[2])]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        with torch.cuda.stream(streams[0]):
            got[0].append(a[0].attend(qa, sa, groups=a[2]))
        with torch.cuda.stream(streams[1]):
            got[1].append(b[0].attend(qb, sb, causal=True, groups=b[2]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_many_groups():
    """More groups than 64, of which some are empty; tiles of every size in the shared part."""
    sizes = [1 + i % 3 for i in range(90)]
    prefix = [(37 * i) % 200 if sizes[i] > 1 else 0 for i in range(90)]
    c, held, groups = family(1, 32, sizes, prefix, [1 + s % 40 for s in range(sum(sizes))], torch.float16)
    n = sum(sizes)
    for heads in (1, 8, 40):
        q = queries(n, heads, heads, torch.float16)
        check_rows(q, list(range(n + 1)), held, True,
                   c.attend(q, list(range(n + 1)), causal=True, groups=groups))
    wide = sorted(groups + groups)[:n + 1]                    # every other group is empty
    check_rows(q, list(range(n + 1)), held, True, c.attend(q, list(range(n + 1)), causal=True, groups=wide))


def test_thousands_of_sequences():
    """3000 sequences, every second one going on from the one before it; a sample of them checked."""
    n = 3000
    c = make(n_kv_heads=1, max_seqs=n, max_len=96, n_pages=2 * n)
    x = rows(33 * n // 2, 1, 1, torch.float16)
    step = c.step(grow=[33, 0] * (n // 2))
    c.append(x[:, 0], x[:, 1], step.slots)
    y = rows(2 * n, 1, 2, torch.float16)
    step = c.step(grow=[2] * n, keep=[33] * n, parent=[s - s % 2 for s in range(n)])
    c.append(y[:, 0], y[:, 1], step.slots)
    q = queries(2 * n, 4, 3, torch.float16)
    out = c.attend(q, step.starts, causal=True, groups=list(range(0, n + 1, 2)))
    assert c.errors() == 0
    x, y = values(x.double().cpu().numpy()), values(y.double().cpu().numpy())
    for s in list(range(0, n, 97)) + [n - 2, n - 1]:
        held = np.concatenate((x[33 * (s // 2):33 * (s // 2) + 33], y[2 * s:2 * s + 2]))
        check_rows(q[2 * s:2 * s + 2], [0, 2], [held], True, out[2 * s:2 * s + 2])


def test_refusals_of_groups():
    c, _, _ = family(2, 32, [3], [40], [1, 1, 1], torch.float16)
    q = queries(3, 4, 1, torch.float16)
    for groups in ([0], [], [0, 1, 2, 3, 3], [[0, 3]], [0.0, 3.0]):
        with pytest.raises(ValueError):
            c.attend(q, [0, 1, 2, 3], groups=groups)
    assert c.attend(q[:0], [0, 0, 0, 0], groups=[0, 3]).shape == (0, 4, 128)


def test_candidates_are_drafted_verified_and_the_best_goes_on():
    """What the operators are for: of each request's candidate blocks the one with the most accepted
    tokens goes on, the next candidates fork from it.  Every step against plain arithmetic."""
    import verify_ref as V
    from mirror_sd_amd import verify_draft
    requests, size, block, kv, heads, vocab = 3, 4, 6, 2, 8, 500
    n = requests * size
    g = torch.Generator().manual_seed(2)
    c, held, groups = family(kv, 32, [size] * requests, [70, 33, 200], [0] * n, torch.float16, spare=60, room=50)
    import kv4_ref as R
    parent, keep = list(range(n)), c.lens.tolist()
    for i in range(4):
        step = c.step(grow=[block] * n, keep=keep, parent=parent)
        held = [held[p][:k] for p, k in zip(parent, keep)]
        x = rows(n * block, kv, 200 + i, torch.float16)
        c.append(x[:, 0], x[:, 1], step.slots)
        new = R.values(x.double().cpu().numpy())
        held = [np.concatenate((h, new[s * block:s * block + block])) for s, h in enumerate(held)]
        q = queries(n * block, heads, 300 + i, torch.float16)
        out = c.attend(q, step.starts, causal=True, groups=groups)
        check_rows(q, step.starts.tolist(), held, True, out)
        logits = 2 * torch.randn((n * block, vocab), generator=g)
        ids = torch.randint(vocab, (n * block,), generator=g).int()
        likely = torch.rand(n * block, generator=g) < 0.7
        logits[:-1].scatter_add_(1, ids[1:, None].long(), 9.0 * likely[1:, None].float())
        u = torch.rand(n * block, generator=g)
        v = verify_draft(logits.cuda().bfloat16(), ids.cuda(), step.starts, u.cuda(), temperature=0.8)
        want = V.verify(logits.bfloat16().double().numpy(), ids.numpy(), step.starts.tolist(), u.numpy(),
                        [float(np.float32(0.8))] * n)
        accepted = v.accepted.tolist()
        assert accepted == want[0].tolist() and v.next_ids.tolist() == want[1].tolist()
        best = [max(range(r * size, r * size + size), key=lambda s: accepted[s]) for r in range(requests)]
        parent = [best[s // size] for s in range(n)]
        keep = [len(held[p]) - block + accepted[p] + 1 for p in parent]
    assert c.errors() == 0


def test_pool_past_32_bits():
    """A pool of 5.6 GB whose last pages alone are free: copies and attention past 2^32 bytes."""
    pages = 20000
    if torch.cuda.mem_get_info()[0] < 9 << 30:
        pytest.skip("needs 9 GB")
    c = make(n_kv_heads=8, page=256, n_pages=pages, max_seqs=3, max_len=1024)
    c.refs[:pages - 12] = 1                  # (held by tables that are not this cache's)
    x = rows(300, 8, 1, torch.float16)
    step = c.step(grow=[300, 0, 0])
    assert step.slots.min().item() == 256 * (pages - 12)
    c.append(x[:, 0], x[:, 1], step.slots)
    y = rows(6, 8, 2, torch.float16)
    step = c.step(grow=[1, 2, 3], keep=[300, 300, 280], parent=[0, 0, 0])
    assert len({s // 256 for s in step.slots.tolist()}) == 3
    c.append(y[:, 0], y[:, 1], step.slots)
    x, y = values(x.double().cpu().numpy()), values(y.double().cpu().numpy())
    held = [np.concatenate((x, y[:1])), np.concatenate((x, y[1:3])), np.concatenate((x[:280], y[3:]))]
    for s in range(3):
        got = c.read([c.table[s, r // 256].item() * 256 + r % 256 for r in range(len(held[s]))], dtype=torch.float32)
        for i in range(2):
            np.testing.assert_array_equal(got[i].double().cpu().numpy(), held[s][:, i])
    q = queries(3, 16, 4, torch.float16)
    check_rows(q, [0, 1, 2, 3], held, True, c.attend(q, [0, 1, 2, 3], causal=True, groups=[0, 3]))
    assert c.errors() == 0


def test_steps_that_free_everything_and_begin_again():
    """A pool to its last page, given back in every order, by the parent, by its continuations."""
    rng = random.Random(3)
    c = make(max_seqs=5, n_pages=20)
    plan = SharedPlan(5, 32, 16, 20)
    for _ in range(8):
        check_step(c, plan, [200, 0, 0, 0, 0], [0] * 5)
        check_step(c, plan, [9] * 5, [200] * 5, [0] * 5)      # 7 pages and 4 copies, 2 rows into an eighth
        order = list(range(5))
        rng.shuffle(order)
        for s in order:
            keep = list(plan.lens)
            keep[s] = 0
            check_step(c, plan, [0] * 5, keep)
        assert plan.refs() == [0] * 20 and c.n_free.item() == 20
