"""The paged 4-bit cache against plain 64-bit arithmetic: rows in and out bit for bit, the step's
pages and slots, attention over ragged sequences within a bound derived from its roundings."""

import numpy as np
import pytest

import kv4_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def make(**kw):
    from mirror_sd_amd.kv4 import KV4Cache
    args = dict(n_kv_heads=2, n_pages=40, max_seqs=4, max_len=1024, page=32)
    args.update(kw)
    return KV4Cache(**args)


def rows(n, kv, seed, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, 2, kv, 128), generator=g)
    x[:, 0, :, ::41] *= 6
    x[:, 1] *= torch.exp(torch.randn((n, 1, 1), generator=g))
    return x.to(dtype).cuda()


def special_rows(dtype):
    """Rows whose groups meet every rule of the format."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn((40, 2, 2, 128), generator=g)
    x[0] = 0
    x[1] = -0.0
    x[2, :, :, 32:] = 0                                     # groups of zeros beside others
    for i, top in enumerate((1.0, 1.75, 1.7500001, 1.7509766, 1.9990234, 6.0, 7.0, 7.0078125)):
        ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]) * top / 7
        x[3 + i] = torch.cat((ties, -ties, torch.tensor([top, -top]))).repeat(8)
    unit = torch.tensor([7.0] + [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5] * 3 + [-0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0])
    for i, e in enumerate((0, -3, 5, -12)):
        x[12 + i] = (unit * 2.0 ** e).repeat(4)
    x[16] *= 2.0 ** -20                                     # fp16 subnormals
    x[17] *= 1e4
    x[18, 0, 0, 5] = float("inf")
    x[19, 1, 1, 127] = float("nan")
    x[20, :, :, 64] = -float("inf")
    if dtype != torch.float16:
        x[21] *= 2.0 ** -130
        x[22] *= 2.0 ** 120
        x[23] *= 2.0 ** -126
        x[24, :, :, 0] = 2.0 ** -133
        x[25, :, :, :32] = 3.3e38
    return x.to(dtype).cuda()


def same(got, want):
    """Equal bit for bit (but for zeros' signs and NaNs' bits) to want in got's type: every value of
    the format is one of fp32's, fp16's and bf16's unless it lies past their range."""
    want = torch.from_numpy(np.asarray(want, np.float64)).to(got.dtype)
    np.testing.assert_array_equal(got.double().cpu().numpy(), want.double().numpy())


# ------------------------------------------------------------------ rows


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("page", [32, 256])
def test_rows_are_the_format(dtype, page):
    c = make(page=page, n_pages=7)
    x = special_rows(DT[dtype])
    slots = torch.randperm(7 * page)[:40].to(torch.int32).cuda()
    c.append(x[:, 0], x[:, 1], slots)
    want = R.values(x.double().cpu().numpy())
    k, v = c.read(slots, dtype=torch.float32)
    same(k, want[:, 0])
    same(v, want[:, 1])
    k, v = c.read(slots, dtype=DT[dtype])
    same(k, want[:, 0])
    same(v, want[:, 1])
    assert c.errors() == 0


def test_every_fp16_value_as_the_largest_of_its_group():
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    top = bits.view(torch.float16)
    g = torch.Generator().manual_seed(1)
    x = (torch.rand((65536, 32), generator=g) * 2 - 1).to(torch.float16) * top[:, None]
    x[:, 17] = top
    x = x.reshape(-1, 2, 2, 128).cuda()
    c = make(page=64, n_pages=128)
    slots = torch.arange(x.shape[0], dtype=torch.int32).cuda()
    c.append(x[:, 0], x[:, 1], slots)
    k, v = c.read(slots, dtype=torch.float32)
    want = R.values(x.double().cpu().numpy())
    same(k, want[:, 0])
    same(v, want[:, 1])


@pytest.mark.parametrize("n,kv,layers", [(1, 1, 1), (33, 3, 2), (257, 5, 1)])
def test_rows_strides_layers_and_neighbours(n, kv, layers):
    c = make(n_kv_heads=kv, n_pages=20, n_layers=layers)
    before = torch.randint(0, 256, c.pool.shape, dtype=torch.uint8, device="cuda")
    c.pool.copy_(before)
    wide = torch.randn((n, 2 * kv * 128 + 64), device="cuda").half()      # rows of a fused projection
    k = wide[:, :kv * 128].unflatten(1, (kv, 128))
    v = torch.randn((kv, n, 128), device="cuda").half().transpose(0, 1)   # head-major rows
    slots = torch.randperm(20 * 32)[:n].to(torch.int32).cuda()
    c.append(k, v, slots, layer=layers - 1)
    gk, gv = c.read(slots, layer=layers - 1, dtype=torch.float32)
    same(gk, R.values(k.double().cpu().numpy()))
    same(gv, R.values(v.double().cpu().numpy()))
    # an offset that is not 16-byte aligned, and a row stride that is not a multiple of 8
    odd = torch.randn((n, kv * 128 + 3), device="cuda").half()[:, 1:1 + kv * 128].unflatten(1, (kv, 128))
    c.append(odd, odd, slots, layer=layers - 1)
    same(c.read(slots, layer=layers - 1, dtype=torch.float32)[1], R.values(odd.double().cpu().numpy()))
    # nothing else moved: other slots' rows, other layers
    rest = torch.ones(20 * 32, dtype=torch.bool)
    rest[slots.cpu().long()] = False
    rest = rest.nonzero()[:, 0].to(torch.int32).cuda()
    got = [t.clone() for t in c.read(rest, layer=layers - 1, dtype=torch.float32)]
    after = c.pool.clone()
    c.pool.copy_(before)
    for a, b in zip(got, c.read(rest, layer=layers - 1, dtype=torch.float32)):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    assert layers == 1 or torch.equal(after[0], before[0])


def test_slots_outside_the_pool():
    from mirror_sd_amd import kv4
    c = make(n_pages=3)
    x = rows(6, 2, 0)
    slots = torch.tensor([0, -1, 95, 96, -2, 2**31 - 1], dtype=torch.int32).cuda()
    c.append(x[:2, 0], x[:2, 1], slots[:2])
    assert c.errors() == 0                                   # -1 is no error
    c.append(x[:, 0], x[:, 1], slots)
    assert c.errors() == kv4.ERR_SLOT and c.errors() == 0
    k, v = c.read(slots, dtype=torch.float32)
    assert c.errors() == kv4.ERR_SLOT
    want = R.values(x.double().cpu().numpy())
    want[[1, 3, 4, 5]] = 0
    same(k, want[:, 0])
    same(v, want[:, 1])


# ------------------------------------------------------------------ the step


def compare_plan(c, plan, step, want):
    starts, slots, pos = want
    assert step.starts.tolist() == starts
    assert step.slots.tolist() == slots
    assert step.positions.tolist() == pos
    assert c.lens.tolist() == plan.lens
    assert c.table.tolist() == [t + [-1] * (plan.width - len(t)) for t in plan.table]
    assert c.n_free.item() == len(plan.free)
    assert c.free.tolist() == plan.free + [-1] * (plan.n_pages - len(plan.free))


@pytest.mark.parametrize("n_seq,page,width,n_pages,most", [
    (1, 32, 9, 9, 40), (5, 64, 6, 20, 90), (64, 32, 8, 300, 33), (65, 32, 8, 200, 40),
    (300, 64, 4, 700, 50), (1500, 32, 5, 4000, 30), (3, 256, 40, 100, 6000)])
def test_steps_follow_the_lengths(n_seq, page, width, n_pages, most):
    rng = np.random.default_rng(n_seq)
    c = make(n_kv_heads=1, n_pages=n_pages, max_seqs=n_seq, max_len=width * page, page=page)
    plan = R.Plan(n_seq, page, width, n_pages)
    for turn in range(7):
        lens = np.array(plan.lens)
        kind = rng.integers(0, 3, n_seq)
        keep = np.where(kind == 0, lens, np.where(kind == 1, lens - rng.integers(0, lens + 1), lens * (turn % 2)))
        grow = np.where(rng.random(n_seq) < 0.2, 0, rng.integers(0, most + 1, n_seq))
        grow = np.minimum(grow, width * page - keep)
        max_rows = int(grow.sum()) + int(rng.integers(0, 3)) * 5
        want, err = plan.step(grow.tolist(), keep.tolist(), max_rows)
        step = c.step(grow=torch.tensor(grow, dtype=torch.int32).cuda(), keep=keep.tolist(), max_rows=max_rows)
        compare_plan(c, plan, step, want)
        assert c.errors() == err
    step = c.step(keep=[0] * n_seq)                          # everything is put back
    assert step.slots.numel() == 0 and c.n_free.item() == n_pages
    assert sorted(c.free.tolist()) == list(range(n_pages)) and int(c.table.max()) == -1


@pytest.mark.parametrize("n_seq", [4, 80])
def test_a_step_that_cannot_be_done_changes_nothing(n_seq):
    from mirror_sd_amd import kv4
    c = make(n_kv_heads=1, n_pages=2 * n_seq, max_seqs=n_seq, max_len=96, page=32)
    plan = R.Plan(n_seq, 32, 3, 2 * n_seq)
    ones = [33] * n_seq
    compare_plan(c, plan, c.step(grow=ones), plan.step(ones, [0] * n_seq, sum(ones))[0])
    zero = [0] * n_seq
    one = lambda x: [x] + zero[1:]
    for grow, keep, rows_, bits in [
            (one(64), [33] * n_seq, 99, kv4.ERR_LENGTH),     # 97 rows of 96
            (one(-1), [33] * n_seq, 99, kv4.ERR_LENGTH), (one(2**31 - 1), [33] * n_seq, 99, kv4.ERR_LENGTH),
            (zero, one(34), 99, kv4.ERR_LENGTH), (zero, one(-1), 99, kv4.ERR_LENGTH),
            (one(32), [33] * n_seq, 99, kv4.ERR_POOL),       # no page is left
            ([10] * n_seq, [33] * n_seq, 10 * n_seq - 1, kv4.ERR_ROWS),
            ([32] * n_seq, [33] * n_seq, 5, kv4.ERR_ROWS | kv4.ERR_POOL)]:
        want, err = plan.step(grow, keep, rows_)
        assert err == bits
        step = c.step(grow=torch.tensor(grow, dtype=torch.int32).cuda(), keep=keep, max_rows=rows_)
        compare_plan(c, plan, step, want)
        assert c.errors() == bits
    compare_plan(c, plan, c.step(grow=[9] * n_seq), plan.step([9] * n_seq, [33] * n_seq, 9 * n_seq)[0])


def state(c):
    return [t.clone() for t in (c.lens, c.table, c.free, c.n_free)]


@pytest.mark.parametrize("n_seq,spare", [(4, 0), (70, 0), (4, 9000), (1100, 0)])
def test_a_step_that_meets_a_bad_page_changes_nothing(n_seq, spare):
    """Page ids outside the pool where a step would put them back, take them or go on in them: the
    step gives no rows, says so and leaves everything as it was.  (9000 spare rows, 1100 sequences:
    the step in launches.)  Ids that the step does not touch are none of its business."""
    from mirror_sd_amd import kv4
    n_pages = 3 * n_seq + 4
    c = make(n_kv_heads=1, n_pages=n_pages, max_seqs=n_seq, max_len=128, page=32)
    plan = R.Plan(n_seq, 32, 4, n_pages)
    lens = [40 + s % 3 * 15 for s in range(n_seq)]           # 2 or 3 pages, the last partly filled
    c.step(grow=lens)
    plan.step(lens, [0] * n_seq, sum(lens))
    last = n_seq - 1
    places = {
        "put back": lambda: c.table[last, 1:2],
        "taken": lambda: c.free[int(c.n_free) - 1:int(c.n_free)],
        "last of those taken": lambda: c.free[int(c.n_free) - 2:int(c.n_free) - 1],
        "gone on in": lambda: c.table[last, 1:2],
    }
    for what, place in places.items():
        keep, grow = list(lens), [0] * n_seq
        if what == "put back":
            keep[last] = 31
        elif what == "gone on in":
            keep[last], grow[last] = 35, 3                   # rows 35 .. 37 lie in its second page
        else:
            grow[0], grow[last] = 64, 5                      # 2 pages for the first alone
            assert R.pages(keep[last] + 5, 32) == R.pages(keep[last], 32)
        rows_ = sum(grow) + spare
        at = place()
        good = at.clone()
        for page in (-1, n_pages, 2**31 - 1, -2**31):
            at.fill_(page)
            before = state(c)
            step = c.step(grow=grow, keep=keep, max_rows=rows_)
            assert c.errors() == kv4.ERR_PAGE, (what, page)
            assert step.starts.tolist() == [0] * (n_seq + 1), (what, page)
            assert step.slots.tolist() == step.positions.tolist() == [-1] * rows_, (what, page)
            for now, then in zip(state(c), before):
                assert torch.equal(now, then), (what, page)
        at.copy_(good)
    # a bad id in the rows that stay, and below those that are taken
    c.table[last, 0], c.free[0] = -1, n_pages
    keep, grow = list(lens), [0] * n_seq
    keep[0], grow[0] = 33, 2
    step = c.step(grow=grow, keep=keep, max_rows=2 + spare)
    assert c.errors() == 0 and int(step.slots[0]) == int(c.table[0, 1]) * 32 + 1
    c.table[last, 0], c.free[0] = plan.table[last][0], plan.free[0]
    plan.step(grow, keep, 2)
    # and the next step is that of a sound cache
    keep, grow = list(plan.lens), [5] * n_seq
    want, err = plan.step(grow, keep, 5 * n_seq + spare)
    compare_plan(c, plan, c.step(grow=grow, keep=keep, max_rows=5 * n_seq + spare), want)
    assert c.errors() == err == 0


@pytest.mark.parametrize("n_seq", [3, 70, 1000])
def test_steps_that_move_many_pages(n_seq):
    """More pages than a workgroup has threads, put back and taken with few new rows; a bad id among
    the last of them changes nothing."""
    from mirror_sd_amd import kv4
    rng = np.random.default_rng(n_seq)
    width = 3000 // n_seq + 6
    n_pages = n_seq * width + 3
    c = make(n_kv_heads=1, n_pages=n_pages, max_seqs=n_seq, max_len=width * 32, page=32)
    plan = R.Plan(n_seq, 32, width, n_pages)
    full = rng.integers(width * 32 - 90, width * 32 + 1, n_seq).tolist()
    zero = [0] * n_seq
    for few in ((8000 // n_seq) * np.ones(n_seq, int), rng.integers(0, 8, n_seq), np.array(zero)):
        want, err = plan.step(full, zero, sum(full))         # (in launches)
        compare_plan(c, plan, c.step(grow=full, keep=zero), want)
        keep = np.minimum(rng.integers(0, 100, n_seq), np.array(full))
        few = np.minimum(few, width * 32 - keep)
        s, at = n_seq - 1, width - 3
        good = int(c.table[s, at])
        c.table[s, at] = n_pages
        before = state(c)
        step = c.step(grow=few.tolist(), keep=keep.tolist(), max_rows=8192)
        assert c.errors() == kv4.ERR_PAGE and step.starts.tolist() == [0] * (n_seq + 1)
        assert int(step.slots.max()) == -1
        assert all(torch.equal(x, y) for x, y in zip(state(c), before))
        c.table[s, at] = good
        want, err = plan.step(few.tolist(), keep.tolist(), 8192)
        compare_plan(c, plan, c.step(grow=few.tolist(), keep=keep.tolist(), max_rows=8192), want)
        assert c.errors() == err == 0


# ------------------------------------------------------------------ attention


def fill(c, lens, seed, dtype, layer=0, shuffle=True):
    """A cache with lens rows a sequence in scattered pages, and the 64-bit values it holds."""
    if shuffle:
        g = torch.Generator().manual_seed(seed)
        c.free.copy_(torch.randperm(c.n_pages, generator=g).to(torch.int32))
    step = c.step(grow=lens)
    n = sum(lens)
    x = rows(n, c.n_kv_heads, seed, dtype)
    c.append(x[:, 0], x[:, 1], step.slots, layer)
    return x, R.values(x.double().cpu().numpy()), step


def queries(n, heads, seed, dtype):
    g = torch.Generator().manual_seed(seed + 77)
    return (1.5 * torch.randn((n, heads, 128), generator=g)).to(dtype).cuda()


def check(c, q, starts, held, lens, causal, out, lse=None, scale=128 ** -0.5):
    half = torch.finfo(q.dtype).eps / 2
    rows = q.shape[0] * (q.shape[1] // c.n_kv_heads) / min(len(lens), max(1, q.shape[0]))
    at = 0
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        kv = held[at:at + n]
        at += n
        if a == b:
            continue
        o, l, mass, size = R.attend(q[a:b].double().cpu().numpy(), kv[:, 0], kv[:, 1], causal, scale)
        tol, ltol = R.attend_tolerance(o, l, mass, size, n, half, split=rows > 32)
        off = np.abs(out[a:b].double().cpu().numpy() - o)
        assert (off <= tol).all(), (s, float((off / tol).max()))
        if lse is not None:
            got = lse[a:b].double().cpu().numpy()
            empty = np.isneginf(l)
            assert (np.isneginf(got) == empty).all()
            assert (np.abs(got[~empty] - l[~empty]) <= ltol[~empty]).all(), s


CASES = [  # heads, kv, q rows, lens, page
    (4, 2, [1], [1], 32), (4, 2, [1], [31], 32), (4, 4, [1], [32], 64), (8, 1, [1], [33], 32),
    (32, 8, [1], [500], 64), (5, 5, [1, 1], [64, 65], 64), (12, 4, [1, 0, 1, 1], [100, 7, 0, 333], 128),
    (8, 8, [1] * 9, [3, 1, 64, 129, 700, 31, 0, 32, 95], 32), (14, 2, [1, 1], [5000, 3], 256),
    (32, 8, [32], [1500], 64), (40, 8, [32, 32], [700, 33], 64), (16, 2, [16, 4, 0, 1], [90, 4, 50, 260], 32),
    (3, 1, [7, 33, 1], [7, 70, 12], 64), (4, 1, [130], [130], 128), (6, 2, [65, 20], [300, 20], 32),
    (1, 1, [257], [257], 32), (64, 1, [2, 3], [40, 41], 64), (24, 1, [5], [2100], 128),
    (8, 2, [5, 9], [3, 2], 32),                              # more query rows than keys
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv,q_lens,lens,page", CASES)
def test_attend(heads, kv, q_lens, lens, page, causal, dtype):
    c = make(n_kv_heads=kv, max_seqs=len(lens), max_len=max(max(lens), 1), page=page,
             n_pages=sum(R.pages(n, page) for n in lens) + 2)
    _, held, _ = fill(c, lens, sum(lens) + heads, DT[dtype])
    starts = np.concatenate(([0], np.cumsum(q_lens))).tolist()
    q = queries(starts[-1], heads, len(lens), DT[dtype])
    out, lse = c.attend(q, starts, causal=causal, return_lse=True)
    assert c.errors() == 0
    check(c, q, starts, held, lens, causal, out, lse)
    # the same call again gives the same bits (no order of sums is left to chance)
    assert torch.equal(c.attend(q, starts, causal=causal), out)


def test_long_caches():
    """Tens of thousands of keys, one of them far above the rest (fp16 weights of the others lie
    far below 1), and a short sequence beside."""
    for dtype in ("fp16", "bf16"):
        lens = [40007, 65]
        c = make(n_kv_heads=1, max_seqs=2, max_len=40960, page=256, n_pages=170)
        c.free.copy_(torch.arange(170, dtype=torch.int32))
        step = c.step(grow=lens)
        x = rows(sum(lens), 1, 3, DT[dtype])
        q = queries(3, 4, 0, DT[dtype])
        x[12345, 0, 0] = (q[0, 1] * 3).to(x.dtype)          # q.k about 3 * 128 * 2.25 * 128^-0.5 = 76
        x[12345, 1, 0] = 0.0
        c.append(x[:, 0], x[:, 1], step.slots)
        held = R.values(x.double().cpu().numpy())
        out, lse = c.attend(q, [0, 2, 3], return_lse=True, scale=0.02)
        check(c, q, [0, 2, 3], held, lens, False, out, lse, scale=0.02)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("q_rows,heads", [(1, 8), (2, 80), (4, 80), (16, 56), (33, 40)])
def test_all_workers_share_units(q_rows, heads, dtype):
    """Enough keys that every workgroup has some and most units have several (in each of the tiles):
    nine ragged sequences of 70 thousand rows in all, against 64 bits on the GPU."""
    lens = [4100, 16001, 9000, 33, 12345, 0, 7777, 20011, 1500]
    c = make(n_kv_heads=8, max_seqs=9, max_len=20480, page=64, n_pages=sum(R.pages(n, 64) for n in lens))
    step = c.step(grow=lens)
    g = torch.Generator("cuda").manual_seed(q_rows)
    x = torch.randn((sum(lens), 2, 8, 128), generator=g, device="cuda", dtype=torch.float32).to(DT[dtype])
    c.append(x[:, 0], x[:, 1], step.slots)
    k, v = (t.double() for t in c.read(step.slots, dtype=torch.float32))
    m_of = [min(q_rows, n) for n in lens]
    starts = np.concatenate(([0], np.cumsum(m_of))).tolist()
    q = queries(starts[-1], heads, 5, DT[dtype])
    r = heads // 8
    for causal in (False, True):
        out = c.attend(q, starts, causal=causal)
        at = 0
        for s, n in enumerate(lens):
            m = m_of[s]
            if m == 0:
                continue
            see = torch.arange(n, device="cuda") < (n - m + torch.arange(m, device="cuda") + 1)[:, None]
            see = see if causal else torch.ones_like(see)
            for h in range(8):
                kh, vh = k[at:at + n, h].contiguous(), v[at:at + n, h].contiguous()
                qh = q[starts[s]:starts[s + 1], h * r:(h + 1) * r].double()
                group = qh.abs().reshape(m, r, 4, 32).amax(-1).repeat_interleave(32, -1)
                sees = see[:, None].expand(m, r, n).reshape(m * r, n)
                z = (qh.reshape(m * r, 128) @ kh.T * 128 ** -0.5).masked_fill(~sees, -torch.inf)
                top = z.amax(1, keepdim=True)
                w = torch.exp(z - top)
                l = w.sum(1, keepdim=True)
                size = [(y.reshape(m * r, 128) @ kh.abs().T * 128 ** -0.5 * sees).amax(1) for y in (qh.abs(), group)]
                tol, _ = R.attend_tolerance(
                    (w @ vh / l).cpu().numpy(), (top + l.log())[:, 0].cpu().numpy(), (w @ vh.abs() / l).cpu().numpy(),
                    torch.stack(size).cpu().numpy(), n, torch.finfo(q.dtype).eps / 2, split=q_rows * r > 32)
                off = (out[starts[s]:starts[s + 1], h * r:(h + 1) * r].double().reshape(m * r, 128) - w @ vh / l).abs()
                assert (off.cpu().numpy() <= tol).all(), (s, h, causal)
            at += n
    assert c.errors() == 0


def spare_rows(n_rows, n_seq, ratio, tile):
    """Rows of no sequence behind n_rows, so that the call takes tiles of `tile` rows."""
    most = {16: 16, 32: 32, 128: 1 << 20}[tile] * n_seq // ratio
    least = {16: 1, 32: 16 * n_seq // ratio + 1, 128: 32 * n_seq // ratio + 1}[tile]
    assert n_rows <= most, "the rows alone take larger tiles"
    return max(0, least - n_rows)


def many(n_seq, kind):
    """Rows and lengths of n_seq sequences, most of them idle unless kind is "all"."""
    rng = np.random.default_rng(n_seq)
    lens = rng.integers(0, 90, n_seq)
    lens[::17] = rng.integers(90, 1200, len(lens[::17]))
    seams = [i for i in (0, 62, 63, 64, 65, 127, 128, 129, n_seq - 1) if i < n_seq]
    if kind == "all":
        on = np.arange(n_seq)
    elif kind == "seams":
        on = np.array(seams)
    elif kind == "ends":                                    # 64 and more without rows between them
        on = np.array([0, n_seq - 1])
    else:
        on = np.array([n_seq - 1])
    m = np.zeros(n_seq, int)
    m[on] = rng.integers(1, 4, len(on))
    lens[n_seq - 1] = 700
    return m, lens


@pytest.mark.parametrize("tile", [16, 32, 128])
@pytest.mark.parametrize("n_seq,kind", [(65, "all"), (65, "last"), (130, "seams"), (130, "ends"), (200, "all"),
                                        (200, "last"), (1000, "seams"), (1000, "ends"), (1000, "all")])
def test_more_than_64_sequences(n_seq, kind, tile):
    """Work over more sequences than a wave looks at once, idle ones at the seams of 64 and whole 64s
    of them between; the tile size is forced by rows of no sequence, which stay as they were."""
    from mirror_sd_amd import kv4
    m, lens = many(n_seq, kind)
    heads, kv = 4, 2
    c = make(n_kv_heads=kv, max_seqs=n_seq, max_len=1216, page=32, n_pages=int(sum(-(-lens // 32))) + 1)
    _, held, _ = fill(c, lens.tolist(), n_seq, torch.bfloat16)
    starts = np.concatenate(([0], np.cumsum(m))).tolist()
    n = starts[-1] + spare_rows(starts[-1], n_seq, heads // kv, tile)
    q = queries(n, heads, 1, torch.bfloat16)
    for causal in (False, True):
        out, lse = c.attend(q, starts, causal=causal, out=torch.full_like(q, 7.0), return_lse=True)
        check(c, q, starts, held, lens.tolist(), causal, out, lse)
        assert (out[starts[-1]:] == 7.0).all()
    assert c.errors() == 0
    # a length and a row range that do not fit, past the first 64: those sequences have no rows
    bad = n_seq - 1
    a = starts[bad]
    for field in ("lens", "starts"):
        st, keep = list(starts), c.lens.clone()
        if field == "lens":
            c.lens[bad] = 1217
        else:
            st[n_seq] = n + 1
        got = c.attend(q, st, causal=True, out=torch.full_like(q, 7.0))
        assert c.errors() == kv4.ERR_PAGE and (got[a:] == 7.0).all(), field
        check(c, q, starts[:n_seq] + [a], held, lens.tolist(), True, got)
        c.lens.copy_(keep)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("tile,heads,kv,n_seq,m,n", [
    (16, 16, 2, 140, 141, 170), (32, 8, 1, 140, 421, 430), (128, 8, 1, 1, 1100, 1100), (128, 16, 2, 2, 1061, 1300)])
def test_more_than_64_tiles(tile, heads, kv, n_seq, m, n, dtype):
    """A sequence of more tiles than a wave looks at once, an odd number of rows in the last of
    them, between sequences of a row."""
    lens = [5 + s % 40 for s in range(n_seq)]
    rows_ = [1] * n_seq
    at = n_seq // 2
    lens[at], rows_[at] = n, m
    assert -(-m * heads // kv // tile) > 64
    c = make(n_kv_heads=kv, max_seqs=n_seq, max_len=1312, page=32, n_pages=sum(R.pages(l, 32) for l in lens))
    _, held, _ = fill(c, lens, n, DT[dtype])
    starts = np.concatenate(([0], np.cumsum(rows_))).tolist()
    q = queries(starts[-1] + spare_rows(starts[-1], n_seq, heads // kv, tile), heads, 1, DT[dtype])
    for causal in (False, True):
        out, lse = c.attend(q, starts, causal=causal, return_lse=True)
        check(c, q, starts, held, lens, causal, out, lse)
    assert c.errors() == 0


@pytest.mark.parametrize("q_rows,heads", [(1, 2), (5, 8), (30, 12)])
def test_extreme_magnitudes(q_rows, heads):
    """Keys of 2^90 under queries of 2^-88 (and the other way round), values of 2^100: powers of two
    change nothing but the exponents.  A query whose values differ by 2^40 within a group."""
    for up, down in ((90, -88), (-100, 101)):
        c = make(max_seqs=2, n_pages=40, page=32, max_len=512)
        lens = [77, 300]
        step = c.step(grow=lens)
        x = rows(sum(lens), 2, 8, torch.bfloat16)
        x[:, 0] *= 2.0 ** up
        x[:, 1] *= 2.0 ** 100
        c.append(x[:, 0], x[:, 1], step.slots)
        held = R.values(x.double().cpu().numpy())
        q = queries(2 * q_rows, heads, 6, torch.bfloat16)
        q[:, :, ::5] *= 2.0 ** -40
        q *= 2.0 ** down
        starts = [0, q_rows, 2 * q_rows]
        out, lse = c.attend(q, starts, causal=True, return_lse=True)
        check(c, q, starts, held, lens, True, out, lse)
    # an infinity or a NaN in a query is its rows' alone
    q[1, 1, 3], q[-1, 0, 100] = float("inf"), float("nan")
    again = c.attend(q, starts, causal=True)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    bad[1, 1] = bad[-1, 0] = True
    assert torch.isnan(again[bad]).all() and torch.equal(again[~bad], out[~bad])
    assert c.errors() == 0


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("ratio", [20, 300])
@pytest.mark.parametrize("q_rows,heads", [(1, 2), (5, 8), (30, 12)])
def test_queries_with_outlier_channels(q_rows, heads, ratio, dtype):
    """A channel of each group of 32 far above the rest, as norm gains leave them: within the bound of
    the parts of 6 bits past 32 rows, and of the type alone up to there."""
    lens = [77, 700]
    starts = [0, q_rows, 2 * q_rows]
    c = make(max_seqs=2, n_pages=60, page=32)
    _, held, _ = fill(c, lens, ratio, DT[dtype])
    q = queries(2 * q_rows, heads, 6, torch.float32) * min(1.0, 20 / ratio)
    q[:, :, 7::32] *= ratio
    q = q.to(DT[dtype])
    out, lse = c.attend(q, starts, causal=True, return_lse=True)
    check(c, q, starts, held, lens, True, out, lse)
    # and where the rest alone decides: the channel's keys are zero
    x = rows(sum(lens), 2, 5, DT[dtype])
    x[:, 0, :, 7::32] = 0
    c.step(keep=[0, 0])
    c.append(x[:, 0], x[:, 1], c.step(grow=lens).slots)
    out, lse = c.attend(q, starts, causal=True, return_lse=True)
    check(c, q, starts, R.values(x.double().cpu().numpy()), lens, True, out, lse)


@pytest.mark.parametrize("q_rows,heads", [(1, 2), (5, 8), (30, 12)])
@pytest.mark.parametrize("up,down,scale", [(20, -18, None), (30, -20, 2.0 ** -11), (-26, 12, 1400.0), (-60, 12, 2.0 ** 48 / 11),
                                           (15, -14, None), (-20, 8, 300.0)])
def test_keys_past_the_range_of_fp16_queries(q_rows, heads, up, down, scale):
    """Keys that fp16 does not hold (the cache was filled from bf16) under fp16 queries: they weigh as
    they are, whatever the tile, all of them or the values of one group of 32 in some of the rows."""
    lens = [77, 300]
    starts = [0, q_rows, 2 * q_rows]
    scale = 128 ** -0.5 if scale is None else scale
    for part in (slice(0, 128), slice(32, 64)):
        c = make(max_seqs=2, n_pages=40, page=32, max_len=512)
        step = c.step(grow=lens)
        x = rows(sum(lens), 2, 8, torch.bfloat16)
        q = queries(2 * q_rows, heads, 6, torch.float16)
        if part.stop < 128:                                  # the other groups' logits stay small
            x[:, 0] *= 2.0 ** -4 * min(1.0, 128 ** -0.5 / scale)
            x[::3, 0, :, part] = 0                           # (groups of zeros, with an exponent of zero)
        x[:, 0, :, part] *= 2.0 ** up
        q[:, :, part] *= 2.0 ** down
        assert torch.isfinite(q).all()
        c.append(x[:, 0], x[:, 1], step.slots)
        held = R.values(x.double().cpu().numpy())
        out, lse = c.attend(q, starts, causal=True, scale=scale, return_lse=True)
        check(c, q, starts, held, lens, True, out, lse, scale=scale)
    # NaN keys among them
    x[77 + 200, 0, 1, 40] = float("nan")
    c.append(x[:, 0], x[:, 1], step.slots)
    again = c.attend(q, starts, causal=True, scale=scale)
    assert torch.equal(again[:q_rows], out[:q_rows]) and torch.isnan(again[q_rows:, heads // 2:]).all()
    assert torch.equal(again[q_rows:, :heads // 2], out[q_rows:, :heads // 2])
    assert c.errors() == 0


@pytest.mark.parametrize("q_rows,heads", [(1, 2), (5, 8), (30, 12)])
def test_values_past_the_range_of_fp16_queries(q_rows, heads):
    """Small values are rounded to multiples of 2^-23: each is off by 2^-24 at most, and so is their
    mean."""
    lens = [77, 300]
    starts = [0, q_rows, 2 * q_rows]
    q = queries(2 * q_rows, heads, 6, torch.float16)
    for e in (-18, -21, -26, -40):
        c = make(max_seqs=2, n_pages=40, page=32, max_len=512)
        step = c.step(grow=lens)
        x = rows(sum(lens), 2, 8, torch.bfloat16)
        x[:, 1] *= 2.0 ** e
        c.append(x[:, 0], x[:, 1], step.slots)
        held = R.values(x.double().cpu().numpy())
        out = c.attend(q, starts, causal=True)
        for s in range(2):
            kv = held[77 * s:77 + 300 * s]
            a, b = starts[s], starts[s + 1]
            o, l, mass, size = R.attend(q[a:b].double().cpu().numpy(), kv[:, 0], kv[:, 1], True, 128 ** -0.5)
            tol, _ = R.attend_tolerance(o, l, mass, size, lens[s], 2.0 ** -11)
            assert (np.abs(out[a:b].double().cpu().numpy() - o) <= tol + 2.0 ** -24).all(), e
    assert c.errors() == 0


@pytest.mark.parametrize("q_rows,heads", [(1, 2), (5, 8), (30, 12)])
@pytest.mark.parametrize("dtype,most,past", [("fp16", 114688.0, 115712.0), ("bf16", 2.95e38, 3.0e38)])
def test_largest_values_of_the_query_type(q_rows, heads, dtype, most, past):
    """Values up to 7 * 2^14 (fp16 queries; 7 * 2^125 with bf16) count; a group of 32 with one past that
    is NaN for the rows that see it, and reaches no other."""
    lens = [77, 300]
    starts = [0, q_rows, 2 * q_rows]
    q = queries(2 * q_rows, heads, 6, DT[dtype])
    c = make(max_seqs=2, n_pages=40, page=32, max_len=512)
    step = c.step(grow=lens)
    x = rows(sum(lens), 2, 8, torch.bfloat16)
    hidden = 77 + 298 if q_rows > 1 else 40                  # seen by the last two rows, or (page by page) by all
    x[hidden, 1, 1, 5] = most
    x[3, 1, 0, 127] = -most                                  # in a block that all rows see
    c.append(x[:, 0], x[:, 1], step.slots)
    held = R.values(x.double().cpu().numpy())
    good, lse = c.attend(q, starts, causal=True, return_lse=True)
    for s in range(2):
        kv = held[77 * s:77 + 300 * s]
        a, b = starts[s], starts[s + 1]
        o, l, mass, size = R.attend(q[a:b].double().cpu().numpy(), kv[:, 0], kv[:, 1], True, 128 ** -0.5)
        tol, _ = R.attend_tolerance(o, l, mass, size, lens[s], torch.finfo(DT[dtype]).eps / 2)
        fits = np.abs(o) <= (65000 if dtype == "fp16" else 2.0 ** 112 / 300)
        assert (np.abs(good[a:b].double().cpu().numpy() - o) <= tol)[fits].all() and fits.mean() > 0.9
    x[hidden, 1, 1, 5], x[3, 1, 0, 127] = past, -past
    c.append(x[:, 0], x[:, 1], step.slots)
    assert torch.isfinite(x.float()).all()
    again, lse2 = c.attend(q, starts, causal=True, return_lse=True)
    nan = torch.zeros(again.shape, dtype=torch.bool, device="cuda")
    nan[:q_rows, :heads // 2, 96:] = True
    if q_rows > 1:
        nan[-2:, heads // 2:, :32] = True
    else:
        nan[:1, heads // 2:, :32] = True
    assert torch.equal(torch.isnan(again), nan)
    assert torch.equal(again[~nan], good[~nan]) and torch.equal(lse2, lse)
    assert c.errors() == 0


@pytest.mark.parametrize("q_rows,heads", [(1, 2), (5, 8), (30, 12)])
def test_all_keys_absent(q_rows, heads):
    """A sequence all of whose pages are outside the pool is one without keys, however it is cut."""
    from mirror_sd_amd import kv4
    c = make(max_seqs=3, n_pages=200, page=32, max_len=4096)
    lens = [40, 3000, 40]
    _, held, _ = fill(c, lens, 4, torch.float16)
    q = queries(3 * q_rows, heads, 3, torch.float16)
    starts = [0, q_rows, 2 * q_rows, 3 * q_rows]
    good = c.attend(q, starts)
    c.table[1, :60] = -1                                    # keys 0 .. 1919: the first seen is a late one
    out = c.attend(q, starts)
    kv = held[40 + 1920:3040]
    o, l, mass, size = R.attend(q[q_rows:2 * q_rows].double().cpu().numpy(), kv[:, 0], kv[:, 1], False, 128 ** -0.5)
    tol, _ = R.attend_tolerance(o, l, mass, size, 3000, 2.0 ** -11)
    assert (np.abs(out[q_rows:2 * q_rows].double().cpu().numpy() - o) <= tol).all()
    assert c.errors() == kv4.ERR_PAGE
    c.table[1] = -1
    out, lse = c.attend(q, starts, return_lse=True)
    assert c.errors() == kv4.ERR_PAGE
    a, b = starts[1], starts[2]
    assert (out[a:b] == 0).all() and torch.isneginf(lse[a:b]).all()
    assert torch.equal(out[:a], good[:a]) and torch.equal(out[b:], good[b:])


@pytest.mark.parametrize("q_rows", [1, 24])
def test_pool_past_32_bits(q_rows):
    """Pages whose bytes lie past 2^32 from the pool's start, in the second layer too."""
    c = make(n_kv_heads=8, n_pages=17000, max_seqs=2, max_len=1024, page=256, n_layers=2)
    assert c.pool[0].numel() > 2**32 and int(c.n_free) == 17000
    c.free.copy_(torch.arange(17000, dtype=torch.int32))    # page 16999 first
    lens = [300, 700]
    _, held, step = fill(c, lens, 9, torch.float16, layer=1, shuffle=False)
    assert int(step.slots[0]) == 16999 * 256
    q = queries(2 * q_rows, 16, 1, torch.float16)
    out = c.attend(q, [0, q_rows, 2 * q_rows], layer=1, causal=True)
    check(c, q, [0, q_rows, 2 * q_rows], held, lens, True, out)
    assert int(c.pool[0].max()) == 0


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("q_rows,heads", [(1, 4), (6, 4), (40, 6)])
def test_what_a_row_does_not_see(dtype, q_rows, heads):
    """Pool bytes that nobody wrote (all ones: NaN groups), NaN and infinite keys and values past a
    row's last key: none of it reaches the row, all of it reaches the rows that see it."""
    lens = [77, 130, 0, 33]
    c = make(max_seqs=4, n_pages=14, page=64)
    c.pool.fill_(255)
    x, held, step = fill(c, lens, 21, DT[dtype])
    starts = np.concatenate(([0], np.cumsum([min(q_rows, max(n, 1)) for n in lens]))).tolist()
    q = queries(starts[-1], heads, 2, DT[dtype])
    for causal in (False, True):
        out, lse = c.attend(q, starts, causal=causal, return_lse=True)
        check(c, q, starts, held, lens, causal, out, lse)
    if q_rows == 1:
        return
    # sequence 1: its last key but two is NaN, a group of values two before it infinite
    k_at, v_at = 77 + 127, 77 + 125
    x[k_at, 0, :, 3] = float("nan")
    x[v_at, 1, 1, 70] = float("inf")
    c.append(x[:, 0], x[:, 1], step.slots)
    out, lse = c.attend(q, starts, causal=True, return_lse=True)
    want = R.values(x.double().cpu().numpy())
    clean = np.nan_to_num(want, nan=0.0)
    m = starts[2] - starts[1]
    got = out[starts[1]:starts[2]].double().cpu().numpy()
    for t in range(m):
        see = 130 - m + t + 1
        if see > 127:                                       # the NaN key: everything
            assert np.isnan(got[t]).all(), t
            assert np.isnan(lse[starts[1] + t].cpu().numpy()).all()
        elif see > 125:                                     # the values' group 64 .. 95 of kv head 1
            nan = np.zeros((heads, 128), bool)
            nan[heads // 2:, 64:96] = True
            assert (np.isnan(got[t]) == nan).all(), t
        else:
            assert np.isfinite(got[t]).all(), t
    # the other sequences, and the rows before, are what they are without them
    o, l, mass, size = R.attend(q[starts[1]:starts[2]].double().cpu().numpy(), clean[77:207, 0],
                                clean[77:207, 1], True, 128 ** -0.5)
    tol, _ = R.attend_tolerance(o, l, mass, size, 130, torch.finfo(q.dtype).eps / 2)
    before = max(0, m - 5)
    assert (np.abs(got - o)[:before] <= tol[:before]).all()
    got0 = out[:starts[1]].double().cpu().numpy()
    assert np.isfinite(got0).all()


def test_largest_fp16_values():
    """65504 in keys and values: a group's 65504 is held as 65536, past fp16's range, and still
    weighs as such."""
    c = make(n_kv_heads=1, max_seqs=1)
    x = rows(40, 1, 4)
    x[7, 1, 0, 9] = 65504.0
    x[9, 1, 0, 100] = -61500.0
    x[30, 0, 0, 64] = 65504.0
    step = c.step(grow=[40, ])
    c.append(x[:, 0], x[:, 1], step.slots)
    held = R.values(x.double().cpu().numpy())
    assert held.max() == 65536
    q = queries(2, 2, 0, torch.float16) * 0.01
    q[:, :, 64] = 0.0
    out, lse = c.attend(q, [0, 2], return_lse=True)
    check(c, q, [0, 2], held, [40], False, out, lse)


def test_pages_and_ranges_that_do_not_fit():
    from mirror_sd_amd import kv4
    lens = [100, 90, 64]
    c = make(max_seqs=3, n_pages=12, page=32)
    _, held, _ = fill(c, lens, 1, torch.float16)
    q = queries(6, 4, 0, torch.float16)
    starts = [0, 2, 4, 6]
    good = c.attend(q, starts)
    table = c.table.clone()
    for page in (-1, 12, -2**31, 2**31 - 1):
        c.table[1, 1] = page                                # keys 32 .. 63 of sequence 1
        out = c.attend(q, starts)
        assert c.errors() == kv4.ERR_PAGE
        assert torch.equal(out[:2], good[:2]) and torch.equal(out[4:], good[4:])
        kv = np.concatenate((held[100:132], held[164:190]))
        o, l, mass, size = R.attend(q[2:4].double().cpu().numpy(), kv[:, 0], kv[:, 1], False, 128 ** -0.5)
        tol, _ = R.attend_tolerance(o, l, mass, size, 90, 2.0 ** -11)
        assert (np.abs(out[2:4].double().cpu().numpy() - o) <= tol).all()
        c.table.copy_(table)
    # lengths beyond the table, rows beyond q or out of order: those sequences have no rows, and
    # their rows of out stay as they were
    for field, value, bad in [("lens", 1025, 1), ("lens", -1, 1), ("starts", [0, 2, 1, 3], 1),
                              ("starts", [0, 2, 4, 7], 2), ("starts", [-1, 2, 4, 6], 0),
                              ("lens", 2**31 - 1, 1)]:
        st, keep = starts, c.lens.clone()
        if field == "lens":
            c.lens[1] = value
        else:
            st = value
        out = torch.full_like(q, 7.0)
        c.attend(q, st, out=out)
        assert c.errors() == kv4.ERR_PAGE, (field, value)
        assert (out[starts[bad]:starts[bad + 1]][-1] == 7.0).all(), (field, value)
        c.lens.copy_(keep)
    assert torch.equal(c.attend(q, starts), good) and c.errors() == 0


def test_rows_of_no_sequence_stay():
    c = make(max_seqs=3, n_pages=12)
    _, held, _ = fill(c, [40, 0, 50], 1, torch.float16)
    q = queries(9, 4, 0, torch.float16)
    out = torch.full_like(q, 3.0)
    got, lse = c.attend(q, [2, 3, 3, 6], causal=True, out=out, return_lse=True)
    assert got is out and (out[:2] == 3.0).all() and (out[6:] == 3.0).all()
    check(c, q[2:6], [0, 1, 1, 4], held, [40, 0, 50], True, out[2:6], lse[2:6])
    none = c.attend(q, [4, 4, 4, 4], out=torch.full_like(q, 3.0))
    assert (none == 3.0).all() and c.errors() == 0
    assert c.attend(q[:0], [0, 0, 0, 0]).shape == (0, 4, 128)


def test_queries_in_place_of_a_projection():
    c = make(max_seqs=2, n_pages=12, n_kv_heads=2)
    _, held, _ = fill(c, [70, 33], 5, torch.bfloat16)
    wide = torch.randn((5, 6 * 128 + 40), device="cuda").bfloat16()
    q = wide[:, 8:8 + 6 * 128].unflatten(1, (6, 128))
    out = c.attend(q, [0, 3, 5], causal=True)
    assert torch.equal(out, c.attend(q.contiguous(), [0, 3, 5], causal=True))
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(out, c.attend(heads_first, [0, 3, 5], causal=True))
    check(c, q, [0, 3, 5], held, [70, 33], True, out)


@pytest.mark.parametrize("q_rows,heads", [(1, 4), (5, 8), (30, 12)])
def test_results_in_the_queries_place(q_rows, heads):
    c = make(max_seqs=2, n_pages=80, max_len=1500)
    fill(c, [1400, 33], 5, torch.float16)
    q = queries(2 * q_rows, heads, 0, torch.float16)
    starts = [0, q_rows, 2 * q_rows]
    want = c.attend(q, starts, causal=True)
    buf = torch.cat((q, q))
    assert torch.equal(c.attend(buf[:2 * q_rows], starts, causal=True, out=buf[2 * q_rows:]), want)   # side by side
    assert torch.equal(buf[:2 * q_rows], q)
    assert c.attend(q, starts, causal=True, out=q) is q and torch.equal(q, want)


# ------------------------------------------------------------------ together


def reference_step(hist, q, k, v, starts, causal):
    """Plain caches (lists of held rows a sequence) after appending, and attention over them."""
    out = np.zeros(q.shape)
    bounds = []
    for s in range(len(hist)):
        a, b = starts[s], starts[s + 1]
        hist[s] = np.concatenate((hist[s], np.stack((k[a:b], v[a:b]), 1)))
        if a == b:
            continue
        o, l, mass, size = R.attend(q[a:b], hist[s][:, 0], hist[s][:, 1], causal, 128 ** -0.5)
        out[a:b] = o
        bounds.append((a, b, R.attend_tolerance(o, l, mass, size, len(hist[s]), 2.0 ** -11)[0]))
    return out, bounds


def test_drafting_loop():
    """Prompts, then blocks whose rejected rows the next step drops, requests that end and others
    that take their place, over two layers: as a drafting program runs it."""
    rng = np.random.default_rng(2)
    n_seq, layers, kv, heads = 5, 2, 2, 6
    c = make(n_kv_heads=kv, max_seqs=n_seq, n_pages=40, max_len=320, page=32, n_layers=layers)
    hist = [[np.zeros((0, 2, kv, 128)) for _ in range(n_seq)] for _ in range(layers)]
    lens = np.zeros(n_seq, int)
    for turn in range(12):
        if turn % 4 == 0:                                   # a sequence or two begin anew
            keep = np.where(rng.random(n_seq) < 0.4, 0, lens) if turn else lens
            grow = np.where(keep == 0, rng.integers(1, 120, n_seq), 0)
            causal = True
        else:                                               # 8-row blocks, some of the last kept
            keep = np.maximum(lens - rng.integers(0, 8, n_seq) * (turn % 4 > 1), 1)
            grow = np.where(rng.random(n_seq) < 0.2, 0, 8)
            causal = False
        step = c.step(grow=grow.tolist(), keep=keep.tolist(), max_rows=int(grow.sum()) + 3)
        starts = step.starts.tolist()
        n = starts[-1]
        assert n == grow.sum() and step.positions[:n].tolist() == [
            p for s in range(n_seq) for p in range(keep[s], keep[s] + grow[s])]
        lens = keep + grow
        for layer in range(layers):
            hist[layer] = [h[:keep[s]] for s, h in enumerate(hist[layer])]
            x = rows(n + 3, kv, 100 * turn + layer)         # rows past the step's: slot -1
            q = queries(n + 3, heads, turn + layer, torch.float16)
            c.append(x[:, 0], x[:, 1], step.slots, layer)
            out = c.attend(q, step.starts, layer, causal=causal)
            held = R.values(x.double().cpu().numpy())
            want, bounds = reference_step(hist[layer], q.double().cpu().numpy(), held[:, 0], held[:, 1],
                                          starts, causal)
            for a, b, tol in bounds:
                assert (np.abs(out[a:b].double().cpu().numpy() - want[a:b]) <= tol).all(), (turn, layer)
    assert c.errors() == 0 and c.lens.tolist() == lens.tolist()


def test_results_join_over_keys():
    """Attention over two caches joined by their sums equals attention over one with all rows."""
    x = rows(200, 2, 8)
    q = queries(3, 4, 8, torch.float16)
    parts = []
    for a, b in ((0, 200), (0, 77), (77, 200)):
        c = make(max_seqs=1)
        c.append(x[a:b, 0], x[a:b, 1], c.step(grow=[b - a]).slots)
        parts.append(c.attend(q, [0, 3], return_lse=True))
    (o, l), (o1, l1), (o2, l2) = [(a.double(), b.double()) for a, b in parts]
    both = torch.logaddexp(l1, l2)
    joined = o1 * torch.exp(l1 - both)[..., None] + o2 * torch.exp(l2 - both)[..., None]
    # each side is off by its weights' and its result's rounding, 3 half steps of values below 10
    assert float((joined - o).abs().max()) <= 2 * 3 * 2.0 ** -11 * 10 and float((both - l).abs().max()) <= 2.0 ** -9


@pytest.mark.parametrize("heads,n", [(4, 12), (40, 12), (4, 9000)])
def test_captured_steps(heads, n):
    """A step, its rows and its attention in a graph, replayed with other lengths and rows between
    eager work; a second graph beside it.  (40 heads: tiles of 128 rows; 9000 rows, nearly all of
    them spare: a step in several launches.)"""
    caches = [make(max_seqs=3, n_pages=30, page=32) for _ in range(2)]
    grow, keep = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2))
    x = rows(n, 2, 0)
    q = queries(n, heads, 0, torch.float16)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                           # first use outside of a capture
        s = caches[0].step(grow=grow, keep=keep, max_rows=n)
        caches[0].append(x[:, 0], x[:, 1], s.slots)
        caches[0].attend(q, s.starts)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for causal in (False, True):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s = caches[0].step(grow=grow, keep=keep, max_rows=n)
            caches[0].append(x[:, 0], x[:, 1], s.slots)
            out = torch.zeros_like(q)
            caches[0].attend(q, s.starts, causal=causal, out=out)
        graphs.append(g)
        outs.append((s, out))
    rng = np.random.default_rng(0)
    lens = np.zeros(3, int)
    for turn in range(8):
        k = np.maximum(lens - rng.integers(0, 4, 3), 0)
        gr = rng.integers(0, 5, 3)
        lens = k + gr
        grow.copy_(torch.tensor(gr, dtype=torch.int32))
        keep.copy_(torch.tensor(k, dtype=torch.int32))
        x.copy_(rows(n, 2, turn))
        q.copy_(queries(n, heads, turn, torch.float16))
        graphs[turn % 2].replay()
        got, out = outs[turn % 2]
        e = caches[1].step(grow=grow, keep=keep, max_rows=n)
        caches[1].append(x[:, 0], x[:, 1], e.slots)
        want = caches[1].attend(q, e.starts, causal=bool(turn % 2), out=torch.zeros_like(q))
        for a, b in zip(got, e):
            assert torch.equal(a, b), turn
        assert torch.equal(out, want), turn
        torch.cuda.synchronize()
    assert caches[0].errors() == caches[1].errors() == 0 and caches[0].lens.tolist() == lens.tolist()


def test_another_stream():
    c, d = make(max_seqs=2), make(max_seqs=2)
    x, q = rows(90, 2, 0), queries(4, 4, 0, torch.float16)
    d.append(x[:, 0], x[:, 1], d.step(grow=[60, 30]).slots)
    want = d.attend(q, [0, 2, 4])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        s = c.step(grow=[60, 30])
        c.append(x[:, 0], x[:, 1], s.slots)
        got = c.attend(q, [0, 2, 4])
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("spare", [0, 1_200_000])
def test_the_most_sequences(spare):
    """65536 sequences, every third idle, the others of one key: a row's result is that key's value
    (its weight and its sum are one number).  Then 40 keys for the last of them.  (1.2 million spare
    rows: tiles of 32.)"""
    n_seq = 65536
    c = make(n_kv_heads=1, max_seqs=n_seq, max_len=64, n_pages=n_seq + 8, page=32)
    grow = torch.ones(n_seq, dtype=torch.int32, device="cuda")
    grow[1::3] = 0                                            # (the last, 65535, has a row)
    n = int(grow.sum())
    step = c.step(grow=grow, max_rows=n)
    x = rows(n, 1, 3)
    c.append(x[:, 0], x[:, 1], step.slots)
    q = queries(n + spare, 1, 1, torch.float16) if spare == 0 else torch.ones((n + spare, 1, 128), dtype=torch.float16, device="cuda")
    out = c.attend(q, step.starts, causal=True, out=torch.full_like(q, 5.0))
    assert c.errors() == 0 and torch.equal(out[:n], c.read(step.slots)[1]) and (out[n:] == 5.0).all()
    more = torch.zeros_like(grow)
    more[-1] = 39
    last = c.step(grow=more, max_rows=39)
    y = rows(39, 1, 4)
    c.append(y[:, 0], y[:, 1], last.slots)
    again = c.attend(q, step.starts, causal=True)
    assert c.errors() == 0 and torch.equal(again[:n - 1], out[:n - 1])
    held = R.values(torch.cat((x[n - 1:], y)).double().cpu().numpy())
    check(c, q[n - 1:n], [0, 1], held, [40], True, again[n - 1:n])


@pytest.mark.parametrize("heads", [4, 40])
def test_two_calls_at_once(heads):
    """Attention over one cache from two streams, eager and replayed, while a third fills another."""
    c, d = make(max_seqs=3, n_pages=80), make(max_seqs=3, n_pages=80)
    fill(c, [700, 33, 900], 1, torch.float16)
    x = rows(1500, 2, 5)
    qs = [queries(27, heads, i, torch.float16) for i in range(2)]
    starts = torch.tensor([0, 9, 13, 27], dtype=torch.int32, device="cuda")
    want = [c.attend(q, starts, causal=bool(i)) for i, q in enumerate(qs)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        replayed = c.attend(qs[1], starts, causal=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(20):
        got = []
        with torch.cuda.stream(streams[0]):
            got += [(c.attend(qs[0], starts), want[0]) for _ in range(3)]
        with torch.cuda.stream(streams[1]):
            replayed.zero_()
            g.replay()
            got += [(c.attend(qs[1], starts, causal=True), want[1]), (replayed, want[1])]
        with torch.cuda.stream(streams[2]):
            slots = d.step(grow=[500, 500, 500], keep=[0, 0, 0]).slots
            d.append(x[:, 0], x[:, 1], slots)
        torch.cuda.synchronize()
        for a, b in got:
            assert torch.equal(a, b), turn
    assert c.errors() == d.errors() == 0


def test_more_rows_than_a_launch_has_workgroups():
    """2.2 million rows in one call (65535 workgroups of 32 take some of them twice), as in parts."""
    n = 2_200_003
    c, d = (make(n_kv_heads=1, max_seqs=1, n_pages=n // 256 + 9, page=256) for _ in range(2))
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn((n, 2, 1, 128), generator=g, device="cuda", dtype=torch.float16)
    slots = torch.randperm((n // 256 + 9) * 256, generator=g, device="cuda")[:n].to(torch.int32)
    c.append(x[:, 0], x[:, 1], slots)
    for a, b in ((0, 1_000_000), (1_000_000, 2_097_120), (2_097_120, n)):
        d.append(x[a:b, 0], x[a:b, 1], slots[a:b])
    assert torch.equal(c.pool, d.pool)
    k, v = c.read(slots)
    for at in (0, 1_048_575, 2_097_120, n - 40):
        want = R.values(x[at:at + 40].double().cpu().numpy())
        same(k[at:at + 40], want[:, 0])
        same(v[at:at + 40], want[:, 1])
    for a, b in ((0, 1_500_000), (1_500_000, n)):
        pk, pv = c.read(slots[a:b])
        assert torch.equal(k[a:b], pk) and torch.equal(v[a:b], pv)
    assert c.errors() == 0


def test_a_step_of_70_million_rows():
    page, lens = 256, [35_000_123, 1, 0, 35_200_000]
    n_pages = sum(R.pages(n, page) for n in lens) + 1
    c = make(n_kv_heads=1, n_pages=n_pages, max_seqs=4, max_len=36_000_000, page=page)
    step = c.step(grow=lens, max_rows=sum(lens) + 77)
    assert step.starts.tolist() == [0, 35_000_123, 35_000_124, 35_000_124, sum(lens)] and c.errors() == 0
    assert (step.slots[sum(lens):] == -1).all() and (step.positions[sum(lens):] == -1).all()
    at = 0
    for s, n in enumerate(lens):
        pos = torch.arange(n, device="cuda", dtype=torch.int32)
        assert torch.equal(step.positions[at:at + n], pos)
        assert torch.equal(step.slots[at:at + n], c.table[s].long()[pos.long() // page].int() * page + pos % page)
        at += n
    used = torch.cat([c.table[s, :R.pages(n, page)] for s, n in enumerate(lens)])
    assert used.unique().numel() == used.numel() == n_pages - int(c.n_free) and int(used.min()) >= 0
    c.step(keep=[0] * 4)
    assert int(c.n_free) == n_pages and int(c.table.max()) == -1 and c.errors() == 0


def test_errors_of_another_stream():
    """errors() waits for calls on every stream, and clears before any later one."""
    from mirror_sd_amd import kv4
    c = make(n_pages=3)
    x = rows(2, 2, 0)
    bad = torch.tensor([5, 96], dtype=torch.int32, device="cuda")
    ok = bad - 5
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)                    # some 10 ms
            c.append(x[:, 0], x[:, 1], bad)
        assert c.errors() == kv4.ERR_SLOT
        with torch.cuda.stream(side):
            c.append(x[:, 0], x[:, 1], bad)
        assert c.errors() == kv4.ERR_SLOT and c.errors() == 0
    with torch.cuda.stream(side):
        c.append(x[:, 0], x[:, 1], ok)
    assert c.errors() == 0


def test_integers_wider_than_32_bits():
    """Numbers that 32 bits do not hold are out of range, not what their low bits say."""
    from mirror_sd_amd import kv4
    c = make()
    wide = torch.full((4,), 2**32 + 1, dtype=torch.int64, device="cuda")
    step = c.step(grow=wide, max_rows=8)
    assert c.errors() == kv4.ERR_LENGTH and step.starts.tolist() == [0] * 5 and c.lens.tolist() == [0] * 4
    x = torch.ones((4, 2, 128), dtype=torch.float16, device="cuda")
    c.append(x, x, wide)
    assert c.errors() == kv4.ERR_SLOT and int(c.pool.max()) == 0
    c.append(x, x, -wide)
    assert c.errors() == kv4.ERR_SLOT and int(c.pool.max()) == 0
    with pytest.raises(ValueError, match="integers"):
        c.append(x, x, torch.zeros(4, device="cuda"))


def test_refusals_on_the_device():
    c = make()
    with pytest.raises(ValueError, match="max_rows"):
        c.step(grow=torch.zeros(4, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="cpu"):
        c.attend(torch.zeros((1, 4, 128), dtype=torch.float16), [0, 1, 1, 1, 1])
    with pytest.raises(ValueError, match="layer"):
        c.read([0], layer=1)
    assert c.read([], dtype=torch.float32)[0].shape == (0, 2, 128)
    assert c.errors() == 0
