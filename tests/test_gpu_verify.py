"""Verification of drafted blocks against plain 64-bit arithmetic: the tokens to the last one, the
chances within a bound derived from the first pass's roundings."""

import numpy as np
import pytest

import verify_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# A chance is p / q of two sums in fp32, rounded once.  A sum: exponents down to -40 matter, each
# rounded three times at most, 3 * 2^-24 * 40 ln 2 = 5.0e-6; powers 2^-23; 128 additions in a thread,
# 7.6e-6, 40 rescalings, 2.4e-6, 8 additions across a wave, 5e-7: 1.6e-5.
REL = 2 * 1.6e-5 + 2.0 ** -23


def call(target, ids, starts, u, temps, draft=None, draft_temps=None):
    from mirror_sd_amd import verify_draft
    v = verify_draft(target, ids, starts, u, temperature=temps, draft_logits=draft,
                     draft_temperature=draft_temps)
    torch.cuda.synchronize()
    return v.accepted.cpu().numpy(), v.next_ids.cpu().numpy(), v.chances.cpu().numpy()


def plain(target, ids, starts, u, temps, draft=None, draft_temps=None):
    host = lambda t: None if t is None else t.double().cpu().numpy()   # noqa: E731
    n_seq = len(starts) - 1
    def each(t):
        if t is None:
            return None
        t = t.cpu().numpy() if isinstance(t, torch.Tensor) else [t] * n_seq
        return [float(np.float32(x)) for x in t]
    return R.verify(host(target), ids.cpu().numpy(), [int(x) for x in starts], u.cpu().numpy(),
                    each(temps), host(draft), each(draft_temps))


def check(target, ids, starts, u, temps, draft=None, draft_temps=None):
    got = call(target, ids, starts, u, temps, draft, draft_temps)
    want = plain(target, ids, starts, u, temps, draft, draft_temps)
    np.testing.assert_array_equal(got[0], want[0])
    np.testing.assert_array_equal(got[1], want[1])
    mine = ~np.isnan(want[2])
    np.testing.assert_allclose(got[2][mine], want[2][mine], rtol=REL, atol=2.0 ** -126)
    return got


def inputs(rows, vocab, target, draft, seed, temp=1.0, near=0.6):
    """Blocks whose draft lies near the target, tokens drawn from the draft."""
    g = torch.Generator().manual_seed(seed)
    n = sum(rows)
    t = 1.5 * torch.randn((n, vocab), generator=g)
    t[torch.arange(n), torch.randint(vocab, (n,), generator=g)] += 7
    d = near * torch.randn((n, vocab), generator=g)
    d[1:] += t[:-1]
    t = t.to(DT[target])
    if draft is None:
        ids = d.argmax(1)
        d = None
    else:
        d = d.to(DT[draft])
        gumbel = -torch.log(-torch.log(torch.rand((n, vocab), generator=g).clamp(min=1e-30)))
        ids = (d.float() / max(temp, 1e-6) + gumbel).argmax(1)
        d = d.cuda()
    starts = [sum(rows[:i]) for i in range(len(rows) + 1)]
    u = torch.rand(n, generator=g)
    return t.cuda(), ids.to(torch.int32).cuda(), starts, u.cuda(), d


@pytest.mark.parametrize("target,draft", [("bf16", "fp32"), ("fp16", "bf16"), ("fp32", "fp16"),
                                          ("bf16", None), ("fp32", None)])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 1000, 2049, 16387, 40000])
def test_tokens_and_chances(target, draft, vocab):
    rows = [5, 1, 0, 9, 2, 16, 3]
    t, ids, starts, u, d = inputs(rows, vocab, target, draft, vocab)
    check(t, ids, starts, u, 1.0, d)


@pytest.mark.parametrize("vocab", [151936, 128257])
@pytest.mark.parametrize("draft", ["bf16", None])
def test_the_largest_vocabularies(vocab, draft):
    t, ids, starts, u, d = inputs([4, 2, 3], vocab, "bf16", draft, 3, temp=0.7)
    check(t, ids, starts, u, 0.7, d)


def test_parts_of_32_kib():
    """Logits past 32 MiB, for which a part of a row is four times as long."""
    t, ids, starts, u, d = inputs([16] * 11, 70001, "bf16", "fp32", 8)
    check(t, ids, starts, u, 1.0, d)


def test_a_temperature_for_each_sequence():
    rows = [6, 6, 6, 6, 6, 6]
    temps = torch.tensor([0.0, 0.3, 1.0, 9e-6, 5.0, 1.7])
    t, ids, starts, u, d = inputs(rows, 3001, "bf16", "bf16", 2)
    check(t, ids, starts, u, temps.cuda(), d)
    check(t, ids, starts, u, temps, d, temps.flip(0))   # greedy drafts of warm targets, and back
    check(t, ids, starts, u, temps, None)


def test_greedy_takes_the_targets_own_choices():
    """Temperature 0: what is kept is what the target alone would have chosen, ties to the lowest id."""
    g = torch.Generator().manual_seed(4)
    t = torch.randint(0, 6, (64, 500), generator=g).to(torch.bfloat16)   # many equal logits
    best = [int(np.argmax(r)) for r in t.float().numpy()]
    ids = torch.tensor([3] + best[:-1], dtype=torch.int32)
    ids[20] += 1
    ids[33] = 499
    u = torch.rand(64, generator=g)
    accepted, next_ids, chances = call(t.cuda(), ids.cuda(), [0, 16, 32, 64], u.cuda(), 0.0)
    assert accepted.tolist() == [15, 3, 0]
    assert next_ids.tolist() == [best[15], best[19], best[32]]
    assert set(chances.tolist()) <= {0.0, 1.0}


def test_draws_at_the_borders_of_equal_weights():
    """1024 equal logits and numbers that are multiples of 1 / 1024: every sum is exact, and the
    first running sum that exceeds u is token 1024 u."""
    n = 256
    t = torch.full((n, 1024), -3.5, dtype=torch.float16)
    u = torch.arange(n).float() * 4 / 1024
    accepted, next_ids, _ = call(t.cuda(), torch.zeros(n, dtype=torch.int32).cuda(), list(range(n + 1)),
                                 u.cuda(), 0.5)
    assert accepted.tolist() == [0] * n and next_ids.tolist() == [4 * i for i in range(n)]
    below = torch.nextafter(u[1:], torch.zeros(1)).cuda()
    _, next_ids, _ = call(t[1:].cuda(), torch.zeros(n - 1, dtype=torch.int32).cuda(), list(range(n)), below, 0.5)
    assert next_ids.tolist() == [4 * i - 1 for i in range(1, n)]


@pytest.mark.parametrize("vocab", [4096, 100003])
def test_draws_of_flat_distributions(vocab):
    """Every token nearly as likely as its neighbours: sums of 32 bits would miss some."""
    g = torch.Generator().manual_seed(vocab)
    n = 96
    t = (0.01 * torch.randn((n, vocab), generator=g)).to(torch.float32).cuda()
    u = torch.rand(n, generator=g).cuda()
    check(t, torch.zeros(n, dtype=torch.int32).cuda(), list(range(n + 1)), u, 1.0)


def test_tests_too_close_for_32_bits():
    """Numbers one step of fp32 on either side of p / q."""
    rows = [2] * 60
    t, ids, starts, _, d = inputs(rows, 5000, "bf16", "bf16", 6, near=2.0)
    u = torch.rand(120)
    want = plain(t, ids, starts, u, 1.0, d)[2][1::2]
    for step in (-1.0, 2.0):
        c = torch.from_numpy(want).float()
        u[1::2] = torch.where(c < 1, torch.nextafter(c, torch.full_like(c, step)), c * 0.5)
        check(t, ids, starts, u.cuda(), 1.0, d)
        check(t, ids, starts, u.cuda(), 1.0, None)


def test_masked_tokens_and_rows_without_a_distribution():
    rows = [4] * 14
    t, ids, starts, u, d = inputs(rows, 3000, "fp32", "fp32", 9)
    t, d = t.clone(), d.clone()
    inf, low = float("inf"), torch.finfo(torch.float32).min
    t[0:4, 100:2900] = -inf            # most of the vocabulary masked, some of it drafted
    t[4:8, :2048] = -inf               # parts with nothing in them
    t[8:12, 7:] = low
    t[12:16] = low                     # all alike
    t[16:20] = -inf
    t[20:24, 2999] = -inf
    t[24:28, 5] = inf
    t[28:32, 1234] = float("nan")
    d[33, 8] = float("nan")
    d[38:40] = -inf
    d[40:44, 1000:] = -inf
    t[44:48] = -inf
    t[44:48, 17] = 2.0                 # one token left
    t[48:52, 3] = 3e38                 # near the end of the range
    t[52:56] = 3e38
    for temps in (1.0, 0.0, 0.02):
        check(t, ids, starts, u, temps, d)
        check(t, ids, starts, u, temps, None)
    accepted, next_ids, _ = call(t, ids, starts, u, 1.0, d)
    assert next_ids[4] == -1 and accepted[4] == 0 and next_ids[6] == -1 and next_ids[7] == -1
    assert next_ids[11] == 17


@pytest.mark.parametrize("temp", [1e-5, 1e-3, 50.0, 1e30])
def test_temperatures_far_from_one(temp):
    t, ids, starts, u, d = inputs([5, 4, 3], 2500, "fp32", "fp32", 11)
    check(t, ids, starts, u, temp, d)
    check(t, ids, starts, u, temp, None)


def test_ids_outside_the_vocabulary():
    t, ids, starts, u, d = inputs([4, 4, 4], 900, "bf16", "bf16", 12)
    ids = ids.clone()
    ids[1], ids[6], ids[9] = -1, 900, 2**31 - 1
    got = check(t, ids, starts, u, 1.0, d)
    check(t, ids, starts, u, 1.0, None)
    assert got[0][0] == 0 and got[0][2] == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_rows_apart_and_at_any_address(dtype):
    """Views with a row stride, whose rows begin anywhere; what lies beside them is NaN."""
    t, ids, starts, u, d = inputs([3, 5, 2], 4099, dtype, dtype, 13)
    want = call(t, ids, starts, u, 1.0, d)
    for left, right in ((0, 1), (1, 0), (3, 4), (5, 8)):
        wide = torch.full((10, left + 4099 + right), float("nan"), dtype=DT[dtype], device="cuda")
        draft = wide.clone()
        wide[:, left:left + 4099] = t
        draft[:, left:left + 4099] = d
        got = call(wide[:, left:left + 4099], ids, starts, u, 1.0, draft[:, left:left + 4099])
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])
        np.testing.assert_allclose(got[2], want[2], rtol=REL)   # (parts begin elsewhere)
    got = call(t.t().contiguous().t(), ids, starts, u, 1.0, d)  # columns apart: copied
    np.testing.assert_array_equal(got[1], want[1])


def test_rows_of_no_sequence_and_ranges_that_do_not_fit():
    t, ids, _, u, d = inputs([4, 4, 4, 4], 1200, "fp16", "fp16", 14)
    check(t, ids, [2, 5, 5, 9], u, 1.0, d)                 # rows before and behind
    got = call(t, ids, [0, 4, 99, 16], u, 1.0, d)
    assert got[0][1] == 0 and got[1][1] == -1 and got[1][2] == -1
    got = call(t, ids, [-3, 4, 8], u, 1.0, d)
    assert got[1][0] == -1
    assert got[1][1] == plain(t, ids, [4, 8], u, 1.0, d)[1][0]
    # no rows at all
    got = call(t[:0], ids[:0], [0, 0, 0], u[:0], 1.0, d[:0])
    assert got[0].tolist() == [0, 0] and got[1].tolist() == [-1, -1]


def test_many_sequences_and_long_blocks():
    g = torch.Generator().manual_seed(15)
    rows = torch.randint(0, 4, (5000,), generator=g).tolist()
    t, ids, starts, u, d = inputs(rows, 33, "bf16", "bf16", 15)
    check(t, ids, starts, u, 1.0, d)
    t, ids, starts, u, d = inputs([3000, 1, 2000], 60, "fp16", "fp16", 16, near=0.02)
    check(t, ids, starts, 0.5 * u, 1.0, d)


def test_kept_tokens_are_distributed_as_the_targets():
    """Two-token blocks from one draft row and one target row, 200 thousand times: the first new
    token's frequencies are the target's within five standard deviations."""
    n = 200000
    g = torch.Generator().manual_seed(17)
    p, q = torch.randn(12, generator=g), torch.randn(12, generator=g)
    ids = torch.zeros(2 * n, dtype=torch.int32)
    ids[1::2] = torch.multinomial(torch.softmax(q, 0), n, replacement=True, generator=g)
    t = p.repeat(2 * n, 1).cuda()
    u = torch.rand(2 * n, generator=g).cuda()
    accepted, next_ids, _ = call(t, ids.cuda(), torch.arange(0, 2 * n + 1, 2)[:65537], u, 1.0,
                                 q.repeat(2 * n, 1).cuda())
    got = np.where(accepted > 0, ids[1::2].numpy()[:65536], next_ids)
    freq = np.bincount(got, minlength=12) / 65536
    want = torch.softmax(p.double(), 0).numpy()
    assert (np.abs(freq - want) <= 5 * np.sqrt(want * (1 - want) / 65536)).all()


def test_a_captured_call_is_replayed_with_other_numbers():
    from mirror_sd_amd import verify_draft
    t, ids, starts, u, d = inputs([8, 5, 8], 20011, "bf16", "bf16", 18)
    starts = torch.tensor(starts, dtype=torch.int32).cuda()
    temps = torch.ones(3).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        verify_draft(t, ids, starts, u, temperature=temps, draft_logits=d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        v = verify_draft(t, ids, starts, u, temperature=temps, draft_logits=d)
    for k in range(4):
        t2, ids2, _, u2, d2 = inputs([8, 5, 8], 20011, "bf16", "bf16", 19 + k)
        for dst, src in ((t, t2), (ids, ids2), (u, u2), (d, d2)):
            dst.copy_(src)
        temps.copy_(torch.tensor([1.0, 0.0, 0.5 + 0.2 * k]))
        graph.replay()
        torch.cuda.synchronize()
        want = call(t2, ids2, starts, u2, temps, d2)
        for x, y in zip(v, want):
            np.testing.assert_array_equal(x.cpu().numpy(), y)


def test_two_calls_on_two_streams():
    a = inputs([32] * 4, 50001, "bf16", "bf16", 21)
    b = inputs([7] * 9, 50001, "fp32", None, 22)
    from mirror_sd_amd import verify_draft
    want = [call(*a[:4], 1.0, a[4]), call(*b[:4], 0.8, b[4])]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (x, temp) in enumerate(((a, 1.0), (b, 0.8))):
            with torch.cuda.stream(streams[i]):
                got[i].append(verify_draft(*x[:4], temperature=temp, draft_logits=x[4]))
    torch.cuda.synchronize()
    for i in range(2):
        for v in got[i]:
            for x, y in zip(v, want[i]):
                np.testing.assert_array_equal(x.cpu().numpy(), y)


def test_inputs_of_other_kinds():
    t, ids, starts, u, d = inputs([4, 3], 700, "fp32", "fp32", 23)
    want = call(t, ids, starts, u, 0.9, d)
    got = call(t, ids.long().cpu(), torch.tensor(starts), u.double().cpu(), torch.tensor([0.9, 0.9]), d)
    for x, y in zip(got, want):
        np.testing.assert_array_equal(x, y)


def test_a_number_next_to_one_in_64_bits():
    """0.99999999 is 1 in 32 bits: it is taken as the largest number below."""
    t = torch.zeros((1, 8), device="cuda")
    _, next_ids, _ = call(t, torch.zeros(1, dtype=torch.int32).cuda(), [0, 1],
                          torch.tensor([1 - 1e-12], dtype=torch.float64), 1.0)
    assert next_ids.tolist() == [7]


def test_refusals():
    from mirror_sd_amd import verify_draft
    t, ids, starts, u, d = inputs([4, 3], 700, "fp32", "fp32", 24)
    for bad in (dict(target_logits=t[0]), dict(target_logits=t.double()), dict(ids=ids[:-1]),
                dict(ids=ids.float()), dict(starts=starts[:1]), dict(uniforms=u[:-1]),
                dict(uniforms=ids), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=float("inf")), dict(temperature=torch.ones(3)),
                dict(draft_logits=d[:, :-1]), dict(draft_logits=d.cpu()),
                dict(draft_temperature=-0.5), dict(target_logits=t.cpu())):
        args = dict(target_logits=t, ids=ids, starts=starts, uniforms=u, temperature=1.0, draft_logits=d)
        args.update(bad)
        with pytest.raises(ValueError):
            verify_draft(**args)


def test_logits_that_grow_along_a_row():
    """References that are raised again and again, over many rounds of a part and past the range
    in which exponents are made in one step."""
    n, vocab = 6, 30011
    steps = torch.arange(vocab).float()
    t = torch.stack([steps * k for k in (1e-4, 1e-2, 1.0, 50.0, -3.0, 1e34)]).clamp(max=3.4e38)
    u = torch.rand(n, generator=torch.Generator().manual_seed(25))
    ids = torch.tensor([5, vocab - 1, vocab - 2, vocab - 1, vocab - 1, 0], dtype=torch.int32)
    for temp in (1.0, 300.0, 1e30):
        check(t.cuda(), ids.cuda(), [0, 2, 4, 6], u.cuda(), temp)
        check(t.flip(1).contiguous().cuda(), ids.cuda(), list(range(7)), u.cuda(), temp)


@pytest.mark.parametrize("vocab,rows", [(2**20 + 3, [2, 1]), (2**24, [2]), (300007, [9] * 40)])
def test_rows_of_many_parts(vocab, rows):
    """Rows of more parts than a wave has lanes, of more than 256 in the draw, and of parts at their
    longest."""
    g = torch.Generator(device="cuda").manual_seed(26)
    n = sum(rows)
    t = (2 * torch.randn((n, vocab), generator=g, device="cuda")).to(torch.bfloat16)
    d = t.roll(1, 0)
    ids = torch.randint(vocab, (n,), generator=g, device="cuda").to(torch.int32)
    u = torch.rand(n, generator=g, device="cuda")
    starts = [sum(rows[:i]) for i in range(len(rows) + 1)]
    some = range(len(rows)) if n < 10 else range(0, len(rows), 13)
    got = call(t, ids, starts, u, 1.0, d), call(t, ids, starts, u, 0.8, None)
    for s in some:
        a, b = starts[s], starts[s + 1]
        for v, temp, draft in ((got[0], 1.0, d), (got[1], 0.8, None)):
            want = plain(t[a:b], ids[a:b], [0, b - a], u[a:b], temp, None if draft is None else draft[a:b])
            assert v[0][s] == want[0][0] and v[1][s] == want[1][0]
            np.testing.assert_allclose(v[2][a:b], want[2], rtol=REL, atol=2.0 ** -126)


def test_logits_past_32_bits():
    """300 rows of 2^24 tokens, 10 GB: the last sequence's rows begin past 2^32 values."""
    n, vocab = 300, 2**24
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB")
    t = torch.empty((n, vocab), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(27)
    t.normal_(generator=g).mul_(2)
    ids = torch.randint(vocab, (n,), generator=g, device="cuda").to(torch.int32)
    u = torch.rand(n, generator=g, device="cuda")
    u[299] = 0.0                       # its token passes
    starts = list(range(0, 299, 2)) + [298, 300]
    got = call(t, ids, starts, u, 1.0)
    want = plain(t[298:], ids[298:], [0, 2], u[298:], 1.0)
    assert got[0][-1] == want[0][0] == 1 and got[1][-1] == want[1][0]
    np.testing.assert_allclose(got[2][298:], want[2], rtol=REL)


def test_numbers_outside_of_their_range():
    """Numbers that are not of [0, 1): some token of the vocabulary that has weight, never another."""
    t = torch.full((6, 500), -float("inf"))
    t[:, 100:400] = torch.randn((6, 300), generator=torch.Generator().manual_seed(28))
    for u in (-1.0, 1.0, 7.0, float("inf"), float("nan"), -float("inf")):
        _, next_ids, _ = call(t.cuda(), torch.zeros(6, dtype=torch.int32).cuda(), list(range(7)),
                              torch.full((6,), u).cuda(), 1.0)
        assert ((next_ids >= 100) & (next_ids < 400)).all(), u


def test_two_graphs_in_one_pool():
    """Two captured calls whose workspaces share memory, replayed in turn."""
    from mirror_sd_amd import verify_draft
    a = inputs([8, 3], 30011, "bf16", "bf16", 29)
    b = inputs([2, 9, 4], 9001, "fp32", None, 30)
    want = [call(*a[:4], 1.0, a[4]), call(*b[:4], 0.6, b[4])]
    graphs, got = [], []
    dev = [[x if isinstance(x, torch.Tensor) else torch.tensor(x, dtype=torch.int32).cuda() for x in c[:4]]
           for c in (a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c, temp, d in ((dev[0], 1.0, a[4]), (dev[1], 0.6, b[4])):
            verify_draft(*c, temperature=temp, draft_logits=d)
    torch.cuda.current_stream().wait_stream(side)
    for c, temp, d in ((dev[0], 1.0, a[4]), (dev[1], 0.6, b[4])):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            got.append(verify_draft(*c, temperature=temp, draft_logits=d))
        graphs.append(graph)
    for i in (0, 1, 1, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        for x, y in zip(got[i], want[i]):
            np.testing.assert_array_equal(x.cpu().numpy(), y)


def test_ranges_that_overlap():
    """Starts that go back: any results, but counts of the sequence's rows and tokens of the vocabulary."""
    t, ids, _, u, d = inputs([6, 3, 8, 4], 5000, "bf16", "fp16", 31)
    starts = [0, 6, 3, 9, 1, 21, 20]
    for draft in (None, d):
        accepted, next_ids, _ = call(t, ids, starts, u, 1.0, draft)
        for s, (a, x) in enumerate(zip(accepted, next_ids)):
            rows = starts[s + 1] - starts[s]
            assert 0 <= a < max(rows, 1) and -1 <= x < 5000
            assert rows > 0 or x == -1
