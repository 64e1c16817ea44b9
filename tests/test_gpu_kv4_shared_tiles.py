"""Attention over shared keys where groups have many rows: tiles of 32 for groups and rests in one
launch, tiles of 128 for the groups in a launch of their own.  Every result against 64 bits."""

import random

import numpy as np
import pytest

import kv4_ref as R
from kv4_shared_shapes import TILES_32, TILES_128
from test_gpu_kv4_shared import DT, ends, family, queries, rows

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SHAPES = [(tile, name) for tile, s in ((32, TILES_32), (128, TILES_128)) for name in s]


def shape(tile, name):
    return (TILES_32 if tile == 32 else TILES_128)[name]


def check(tile, q, starts, held, causal, out, lse=None, some=None):
    """Rows of the sequences `some` (default: all) within the bound of one attention; the join adds two
    powers and products to a state, 24 fp32 roundings at most where both parts weigh more than
    2^-20 (as 768 more keys would).  Only tiles of 128 take the queries in parts."""
    half = torch.finfo(q.dtype).eps / 2
    for s in range(len(held)) if some is None else some:
        a, b = starts[s], starts[s + 1]
        if a == b:
            continue
        kv = held[s]
        o, l, mass, size = R.attend(q[a:b].double().cpu().numpy(), kv[:, 0], kv[:, 1], causal, 128 ** -0.5)
        tol, ltol = R.attend_tolerance(o, l, mass, size, len(kv) + 768, half, split=tile == 128)
        off = np.abs(out[a:b].double().cpu().numpy() - o)
        assert (off <= tol).all(), (s, float((off / tol).max()))
        if lse is not None:
            got = lse[a:b].double().cpu().numpy()
            empty = np.isneginf(l)
            assert (np.isneginf(got) == empty).all()
            assert (np.abs(got[~empty] - l[~empty]) <= ltol[~empty]).all(), s


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("tile,name", SHAPES)
def test_attend(tile, name, causal, dtype):
    heads, kv, page, sizes, prefix, own, q_lens = shape(tile, name)
    c, held, groups = family(kv, page, sizes, prefix, own, DT[dtype], seed=tile + heads)
    starts = ends(q_lens)
    q = queries(starts[-1], heads, page, DT[dtype])
    out, lse = c.attend(q, starts, causal=causal, return_lse=True, groups=groups)
    assert c.errors() == 0
    check(tile, q, starts, held, causal, out, lse, range(0, len(held), 4) if name == "long" else None)
    for _ in range(3):
        assert torch.equal(c.attend(q, starts, causal=causal, groups=groups), out)
    c.attend(q, starts, causal=causal, groups=groups, out=q)   # in the queries' place
    assert torch.equal(q, out) and c.errors() == 0


FEW = [(32, 40), (128, 72)]   # tiles, sequences of one row of 8 heads


@pytest.mark.parametrize("tile,n", FEW)
def test_groups_that_cut_through_families(tile, n):
    """Boundaries inside a family, sequences of no group, sequences that no longer agree."""
    c, held, _ = family(1, 32, [n // 2, n - n // 2], [200, 330], [1 + s % 5 for s in range(n)], torch.float16)
    starts = ends([1] * n)
    q = queries(n, 8, tile, torch.float16)
    for groups in ([1, n], [n // 4, n - 3], [0, n // 2]):
        check(tile, q, starts, held, True, c.attend(q, starts, causal=True, groups=groups))
    for s, page in ((3, 4), (n // 2 + 1, 7), (0, 2), (n - 1, 0)):
        # sequence s gets a page of its own for these rows, with other rows in it
        spare = (c.refs == 0).nonzero()[0].item()
        x = rows(32, 1, 50 + s, torch.float16)
        c.append(x[:, 0], x[:, 1], torch.arange(32 * spare, 32 * spare + 32).to(torch.int32))
        c.refs[spare] += 1
        c.table[s, page] = spare
        held[s][32 * page:32 * page + 32] = R.values(x.double().cpu().numpy())
        check(tile, q, starts, held, False, c.attend(q, starts, groups=[0, n // 2]))
        check(tile, q, starts, held, True, c.attend(q, starts, causal=True, groups=[n // 2, n]))
    assert c.errors() == 0


@pytest.mark.parametrize("tile,n", FEW)
def test_what_does_not_fit(tile, n):
    """Pages outside the pool are absent for all, lengths and ranges that do not fit leave their
    sequence without rows, boundaries out of order share nothing; each is reported."""
    from mirror_sd_amd import kv4
    c, held, groups = family(1, 32, [n], [140], [1 + s % 7 for s in range(n)], torch.bfloat16)
    starts = ends([1] * n)
    q = queries(n, 8, 3, torch.bfloat16)
    table = c.table.clone()
    for page in (-1, c.n_pages, 2**31 - 1):
        c.table[:, 1] = page
        out = c.attend(q, starts, groups=groups)
        assert c.errors() == kv4.ERR_PAGE
        check(tile, q, starts, [np.concatenate((h[:32], h[64:])) for h in held], False, out)
        c.table.copy_(table)
    lens = c.lens.clone()
    for value in (-1, 2**31 - 1):
        c.lens[5] = value
        out = torch.full_like(q, 7.0)
        c.attend(q, starts, out=out, groups=groups)
        assert c.errors() == kv4.ERR_PAGE and (out[5] == 7.0).all()
        check(tile, q, starts, held, False, out, some=[s for s in range(n) if s != 5])
        c.lens.copy_(lens)
    for bad in ([n, 0], [-1, n], [0, n + 1]):
        out = c.attend(q, starts, groups=bad)
        assert c.errors() == kv4.ERR_PAGE, bad
        check(tile, q, starts, held, False, out)
    c.attend(q, starts, groups=groups)
    assert c.errors() == 0


@pytest.mark.parametrize("tile,n", FEW)
def test_rows_of_no_sequence_stay_and_strided_queries(tile, n):
    c, held, groups = family(1, 64, [n], [200], [2] * n, torch.float16)
    starts = [x + 3 for x in ends([1] * n)]
    q = queries(n + 5, 8, 8, torch.float16)
    want = c.attend(q, starts, groups=groups)
    check(tile, q, starts, held, False, want)
    out = torch.full_like(q, 3.0)
    c.attend(q, starts, out=out, groups=groups)
    assert (out[:3] == 3.0).all() and (out[n + 3:] == 3.0).all() and torch.equal(out[3:n + 3], want[3:n + 3])
    wide = torch.full((n + 5, 24, 128), float("nan"), device="cuda").half()   # a part of a projection's row
    wide[:, 8:16] = q
    assert torch.equal(c.attend(wide[:, 8:16], starts, groups=groups)[3:n + 3], want[3:n + 3])


@pytest.mark.parametrize("tile,n", FEW)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_what_a_row_does_not_see_of_shared_pages(tile, n, dtype):
    """NaN and infinite rows past most sequences' ends, in a page that all share."""
    c, held, groups = family(1, 64, [n], [100], [0] * n, DT[dtype])
    x = rows(100, 1, 0, DT[dtype])
    bad = x.clone()
    bad[96:] = float("nan")
    bad[90, 1] = float("inf")
    c.append(bad[:, 0], bad[:, 1], [c.table[0, r // 64].item() * 64 + r % 64 for r in range(100)])
    lens = [100 if s == 7 else 65 + s % 26 for s in range(n)]
    c.step(keep=lens)
    starts = ends([1] * n)
    q = queries(n, 8, 9, DT[dtype])
    out = c.attend(q, starts, groups=groups)
    assert torch.isnan(out[7]).all()
    check(tile, q, starts, [h[:m] for h, m in zip(held, lens)], False, out, some=[s for s in range(n) if s != 7])


@pytest.mark.parametrize("tile,n", FEW)
def test_keys_past_the_queries_range(tile, n):
    """Keys of 10^5 in a shared page and in a rest, under fp16 queries that are as small there."""
    c, held, groups = family(1, 32, [n], [130], [20] * n, torch.float16)
    q = queries(n, 8, 11, torch.float16)
    q[:, :, 32:64] *= 1e-4
    for page in (1, 3):
        x = rows(32, 1, 90 + page, torch.float16).float()
        x[:, 0, :, 32:64] *= 2e5
        c.append(x[:, 0], x[:, 1], torch.arange(32).to(torch.int32) + 32 * c.table[0, page].item())
        for s in range(n):
            if c.table[s, page] == c.table[0, page]:
                held[s][32 * page:32 * page + 32] = R.values(x.double().cpu().numpy())
    starts = ends([1] * n)
    out, lse = c.attend(q, starts, return_lse=True, groups=groups)
    check(tile, q, starts, held, False, out, lse)
    assert c.errors() == 0


@pytest.mark.parametrize("tile,n,size", [(32, 40, 20), (128, 136, 68)])
def test_captured_steps_of_candidates(tile, n, size):
    """A graph of a forking step, its rows in and attention over what is shared, replayed with other
    parents, lengths, rows and groups, and eager work between."""
    c, held, _ = family(1, 32, [size] * 2, [150, 90], [1] * n, torch.float16, spare=3 * n, room=60)
    ints = dict(dtype=torch.int32, device="cuda")
    keep, parent, grow = c.lens.clone(), torch.arange(n, **ints), torch.ones(n, **ints)
    groups = torch.tensor([0, size, n], **ints)
    x, q = rows(n, 1, 1, torch.float16), queries(n, 8, 1, torch.float16)
    state = [t.clone() for t in (c.lens, c.table, c.refs, c.n_free)]

    def step():
        s = c.step(grow=grow, keep=keep, parent=parent, max_rows=n)
        c.append(x[:, 0], x[:, 1], s.slots)
        return c.attend(q, s.starts, causal=True, return_lse=True, groups=groups)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for t, was in zip((c.lens, c.table, c.refs, c.n_free), state):
        t.copy_(was)
    rng = random.Random(n)
    starts = ends([1] * n)
    for i in range(5):
        now = c.lens.tolist()
        p = [size * (s // size) + rng.randrange(size) for s in range(n)]
        k = [now[j] - rng.choice([0, 0, 1]) for j in p]
        parent.copy_(torch.tensor(p))
        keep.copy_(torch.tensor(k))
        groups.copy_(torch.tensor([[0, size, n], [0, n, n], [2, size, n - 1]][i % 3]))
        x.copy_(rows(n, 1, 60 + i, torch.float16))
        q.copy_(queries(n, 8, 60 + i, torch.float16))
        graph.replay()
        assert c.errors() == 0
        new = R.values(x.double().cpu().numpy())
        held = [np.concatenate((held[p[s]][:k[s]], new[s:s + 1])) for s in range(n)]
        check(tile, q, starts, held, True, out, lse)
        eager = c.attend(q, starts, causal=True, groups=groups)
        assert torch.equal(eager, out)
    assert c.errors() == 0


def test_calls_at_once():
    """Tiles of 32 and of 128 on two streams, and two graphs in one pool."""
    a = family(1, 32, [40], [700], [3] * 40, torch.float16)
    b = family(2, 64, [72, 60], [900, 300], [2 + s % 9 for s in range(132)], torch.bfloat16, seed=3)
    qa, qb = queries(40, 8, 1, torch.float16), queries(132, 16, 2, torch.bfloat16)
    sa, sb = (torch.tensor(ends([1] * n), dtype=torch.int32, device="cuda") for n in (40, 132))
    ga, gb = (torch.tensor(x[2], dtype=torch.int32, device="cuda") for x in (a, b))
    calls = [lambda: a[0].attend(qa, sa, groups=ga), lambda: b[0].attend(qb, sb, causal=True, groups=gb)]
    want = [f() for f in calls]
    check(32, qa, ends([1] * 40), a[1], False, want[0])
    check(128, qb, ends([1] * 132), b[1], True, want[1])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    graphs, out = [], []
    for f in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            out.append(f())
        graphs.append(graph)
    for i in (0, 1, 1, 0, 1, 0):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(out[i], want[i])
