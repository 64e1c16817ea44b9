"""Groups named for blocks of so many rows that their sequences are attended apart: results as without
groups, and boundaries that do not fit reported as everywhere."""

import pytest

from test_gpu_kv4_shared import check_rows, ends, family, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("rows", [17, 40])   # of a kv head: tiles of 32, of 128
def test_boundaries_are_looked_at(rows):
    from mirror_sd_amd import kv4
    c, held, groups = family(2, 32, [3, 2], [100, 70], [rows + s for s in range(5)], torch.float16)
    starts = ends([rows] * 5)
    q = queries(5 * rows, 2, rows, torch.float16)
    want = c.attend(q, starts, causal=True)
    check_rows(q, starts, held, True, want)
    for bad in ([0, 4, 3, 5], [-1, 3, 5], [0, 3, 6], [3, 0], [0, 2**31 - 1], [-2**31, 5]):
        assert torch.equal(c.attend(q, starts, causal=True, groups=bad), want)
        assert c.errors() == kv4.ERR_PAGE, bad
    for good in (groups, [0, 5], [2, 2, 4], [5, 5], [0, 0], [0, 1, 2, 3, 4, 5]):
        assert torch.equal(c.attend(q, starts, causal=True, groups=good), want)
        assert c.errors() == 0, good


@pytest.mark.parametrize("at", [1, 255, 256, 700, 899])
def test_many_boundaries(at):
    """900 groups, one boundary among them out of order."""
    from mirror_sd_amd import kv4
    n = 900
    c, _, _ = family(1, 32, [n], [32], [1] * n, torch.bfloat16)
    q = queries(17 * n, 1, 5, torch.bfloat16)
    starts = ends([17] * n)
    want = c.attend(q, starts)
    groups = list(range(n + 1))
    assert torch.equal(c.attend(q, starts, groups=groups), want) and c.errors() == 0
    groups[at] = groups[at + 1] + 1
    assert torch.equal(c.attend(q, starts, groups=groups), want)
    assert c.errors() == kv4.ERR_PAGE


def test_a_captured_call_reports_each_time():
    from mirror_sd_amd import kv4
    c, held, _ = family(1, 32, [4], [200], [20] * 4, torch.float16)
    starts = torch.tensor(ends([20] * 4), dtype=torch.int32, device="cuda")
    groups = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    q = queries(80, 2, 6, torch.float16)
    want = c.attend(q, starts, causal=True, groups=groups)
    check_rows(q, ends([20] * 4), held, True, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.attend(q, starts, causal=True, groups=groups)
    for bounds, err in (([0, 4], 0), ([4, 0], kv4.ERR_PAGE), ([0, 3], 0), ([0, 5], kv4.ERR_PAGE), ([1, 1], 0)):
        groups.copy_(torch.tensor(bounds))
        graph.replay()
        assert c.errors() == err and torch.equal(out, want)
