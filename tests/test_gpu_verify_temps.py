"""Temperatures of a verification that are no temperatures, or lie on the GPU."""

import numpy as np
import pytest

from test_gpu_verify import REL, call, inputs, plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

INF, NAN = float("inf"), float("nan")
ROWS = [4, 1, 5, 3, 1, 2, 6]
# sequences 1, 2, 4 and 5: negative, NaN, infinite, the smallest number below zero
TEMPS = [0.7, -1.0, NAN, 0.0, INF, -1e-45, 1.3]
BAD = [1, 2, 4, 5]


def others(got, want, starts, skip):
    """Every sequence but those of `skip` as in the plain verification."""
    for s in range(len(starts) - 1):
        if s in skip:
            continue
        a, b = starts[s], starts[s + 1]
        assert (got[0][s], got[1][s]) == (want[0][s], want[1][s]), s
        np.testing.assert_allclose(got[2][a:b], want[2][a:b], rtol=REL, atol=2.0 ** -126)


@pytest.mark.parametrize("vocab", [900, 40000])
@pytest.mark.parametrize("draft", ["bf16", None])
def test_entries_on_the_gpu_that_are_no_temperatures(vocab, draft):
    """Their sequences' rows have no distribution: nothing accepted, -1 drawn; the others are as ever."""
    t, ids, starts, u, d = inputs(ROWS, vocab, "bf16", draft, 40)
    good = torch.tensor([1.0 if s in BAD else x for s, x in enumerate(TEMPS)])
    want = plain(t, ids, starts, u, good, d)
    got = call(t, ids, starts, u, torch.tensor(TEMPS).cuda(), d)
    others(got, want, starts, BAD)
    for s in BAD:
        a, b = starts[s], starts[s + 1]
        assert got[0][s] == 0 and got[1][s] == -1
        assert got[2][a:b].tolist() == [1.0] + [0.0] * (b - a - 1)


def test_draft_temperatures_on_the_gpu_that_are_none():
    """The drafted rows have no distribution: the first of them is rejected and -1 drawn; a sequence
    without drafted rows needs none."""
    t, ids, starts, u, d = inputs(ROWS, 3001, "fp16", "fp32", 41)
    good = torch.tensor([1.0 if s in BAD else x for s, x in enumerate(TEMPS)])
    want = plain(t, ids, starts, u, 0.9, d, good)
    got = call(t, ids, starts, u, 0.9, d, torch.tensor(TEMPS).cuda())
    several = [s for s in BAD if ROWS[s] > 1]
    others(got, want, starts, several)
    for s in several:
        a, b = starts[s], starts[s + 1]
        assert got[0][s] == 0 and got[1][s] == -1
        assert got[2][a:b].tolist() == [1.0] + [0.0] * (b - a - 1)


def test_host_tensors_are_refused_as_numbers_are():
    from mirror_sd_amd import verify_draft
    t, ids, starts, u, d = inputs([4, 3], 700, "fp32", "fp32", 42)
    for x in (-1.0, NAN, INF, -INF, -1e-30):
        for dtype in (torch.float32, torch.float64, torch.bfloat16):
            temps = torch.tensor([0.5, x], dtype=dtype)
            with pytest.raises(ValueError, match="finite"):
                verify_draft(t, ids, starts, u, temperature=temps)
            with pytest.raises(ValueError, match="finite"):
                verify_draft(t, ids, starts, u, draft_logits=d, draft_temperature=temps)
    with pytest.raises(ValueError, match="finite"):   # past fp32
        verify_draft(t, ids, starts, u, temperature=torch.tensor([0.5, 1e39], dtype=torch.float64))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.int64])
def test_a_number_on_the_gpu_is_one_for_all(dtype):
    t, ids, starts, u, d = inputs(ROWS, 3001, "bf16", "bf16", 43)
    for x, y in ((0, 2), (2, 0)) if dtype == torch.int64 else ((0.5, 1.25), (0.0, 0.75)):
        want = call(t, ids, starts, u, float(x), d, float(y))
        got = call(t, ids, starts, u, torch.tensor(x, dtype=dtype).cuda(), d, torch.tensor(y, dtype=dtype).cuda())
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a, b)


def test_a_number_on_the_gpu_that_is_no_temperature():
    t, ids, starts, u, d = inputs(ROWS, 900, "bf16", "bf16", 44)
    for x in (-0.5, NAN, INF):
        got = call(t, ids, starts, u, torch.tensor(x).cuda(), d)
        assert not got[0].any() and (got[1] == -1).all()
    with pytest.raises(ValueError):
        call(t, ids, starts, u, torch.tensor(1j).cuda(), d)


def test_a_captured_call_takes_a_number_on_the_gpu():
    """It is not read back: a graph can be captured with it, and follows what it holds."""
    from mirror_sd_amd import verify_draft
    t, ids, starts, u, d = inputs([5, 3], 5003, "fp16", "fp16", 45)
    starts = torch.tensor(starts, dtype=torch.int32).cuda()
    temp = torch.tensor(1.0).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        verify_draft(t, ids, starts, u, temperature=temp, draft_logits=d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        v = verify_draft(t, ids, starts, u, temperature=temp, draft_logits=d)
    for x in (1.0, 0.0, 0.5, 2.0, 0.5):
        temp.fill_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(v, call(t, ids, starts, u, x, d)):
            np.testing.assert_array_equal(a.cpu().numpy(), b)
