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
    at = 0
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        kv = held[at:at + n]
        at += n
        if a == b:
            continue
        o, l, mass, size = R.attend(q[a:b].double().cpu().numpy(), kv[:, 0], kv[:, 1], causal, scale)
        tol, ltol = R.attend_tolerance(o, l, mass, size, n, half)
        off = np.abs(out[a:b].double().cpu().numpy() - o)
        assert (off <= tol).all(), (s, float((off / tol).max()))
        if lse is not None:
            got = lse[a:b].double().cpu().numpy()
            empty = np.isneginf(l)
            assert (np.isneginf(got) == empty).all()
            assert (np.abs(got - l)[~empty] <= ltol[~empty]).all(), s


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
