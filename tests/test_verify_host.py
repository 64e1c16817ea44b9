"""Verification of drafted blocks without a GPU: refusals of the C entry points, the workspace, the
plain implementation that the GPU tests compare with."""

import ctypes

import numpy as np
import pytest

import verify_ref as R
from mirror_sd_amd import _lib

torch = pytest.importorskip("torch")

FAKE = 4096   # aligned, never read


def args(**o):
    a = dict(target=FAKE, draft=FAKE, target_row=1000, draft_row=1000, target_dtype=2, draft_dtype=0,
             n_rows=8, vocab=1000, n_seq=2, temp=1.0, draft_temp=0.7, ids=FAKE, starts=FAKE,
             uniforms=FAKE, temps=None, draft_temps=None, accepted=FAKE, next_ids=FAKE, chances=FAKE,
             ws=FAKE, ws_bytes=0)
    a.update(o)
    return _lib.DflVerify(*a.values())


@pytest.mark.parametrize("bad", [
    dict(n_rows=-1), dict(n_rows=2**24 + 1), dict(vocab=0), dict(vocab=2**24 + 1), dict(n_seq=0),
    dict(n_seq=65537), dict(target_dtype=3), dict(draft_dtype=-1), dict(target=None), dict(ids=None),
    dict(starts=None), dict(uniforms=None), dict(accepted=None), dict(next_ids=None),
    dict(chances=None), dict(target_row=999), dict(draft_row=0), dict(target=FAKE + 1),
    dict(draft=FAKE + 2), dict(temp=-1.0), dict(temp=float("nan")), dict(temp=float("inf")),
    dict(draft_temp=-1e-9), dict(n_rows=2**24, vocab=2**24, target_row=2**24, draft_row=2**24),
    dict(ws=None), dict(ws=FAKE + 8), dict(ws_bytes=-1)])
def test_refuses_before_device_work(bad):
    L = _lib.load()
    good = args()
    good.ws_bytes = L.dfl_verify_ws(ctypes.byref(good))
    assert good.ws_bytes > 0
    bad = args(**{"ws_bytes": good.ws_bytes, **bad})
    assert L.dfl_verify(ctypes.byref(bad), None) == _lib.DFL_EINVAL
    assert L.dfl_last_error().startswith(b"dfl_verify: ")
    assert L.dfl_verify(None, None) == _lib.DFL_EINVAL


def test_workspace_grows_with_the_call():
    L = _lib.load()
    size = lambda **o: L.dfl_verify_ws(ctypes.byref(args(**o)))   # noqa: E731
    assert 0 < size(draft=None) < size() < size(n_rows=100) < size(n_rows=100, n_seq=50)
    assert size(vocab=0) == 0 and L.dfl_verify_ws(None) == 0
    # scratch stays far below the logits that it is made from
    big = size(n_rows=2048, n_seq=64, vocab=151936, target_row=151936, draft_row=151936)
    assert big < 2048 * 151936 * 6 / 100


def test_refusals_of_the_python_function():
    from mirror_sd_amd import verify_draft
    t = torch.zeros(4, 10)
    with pytest.raises(ValueError, match="GPU"):
        verify_draft(t, [0] * 4, [0, 4], torch.zeros(4))
    with pytest.raises(ValueError, match="vocab"):
        verify_draft(t[0], [0] * 4, [0, 4], torch.zeros(4))
    with pytest.raises(ValueError, match="fp32"):
        verify_draft(t.double(), [0] * 4, [0, 4], torch.zeros(4))


# ------------------------------------------------------------------ the plain implementation


def test_plain_distributions():
    inf = float("inf")
    np.testing.assert_allclose(R.distribution([0.0, np.log(3.0)], 1.0), [0.25, 0.75])
    np.testing.assert_allclose(R.distribution([0.0, np.log(3.0)], 0.5), [0.1, 0.9])
    assert R.distribution([1.0, 5.0, 5.0], 0.0).tolist() == [0, 1, 0]
    assert R.distribution([-inf, 2.0], 1.0).tolist() == [0, 1]
    for row in ([-inf, -inf], [0.0, inf], [0.0, float("nan")]):
        assert R.distribution(row, 1.0) is None and R.distribution(row, 0.0) is None


def test_plain_draws():
    assert [R.draw(np.array([1.0, 0.0, 2.0, 1.0]), u) for u in (0.0, 0.24, 0.25, 0.74, 0.75, 0.99)] == \
        [0, 0, 2, 2, 3, 3]
    assert R.draw(np.array([0.0, 0.0, 1.0]), 0.0) == 2


def test_plain_verdicts():
    """Two tokens: p = (1/4, 3/4), q = (3/4, 1/4).  Token 0 passes with chance 1/3, else 1 is drawn."""
    p, q = np.log([[0.25, 0.75]] * 3), np.log([[0.75, 0.25]] * 3)
    for u, accepted in ((0.32, 2), (0.34, 0)):
        a, n, c = R.verify(p, [1, 0, 1], [0, 3], [0.5, u, 0.9], [1.0], q)
        assert a[0] == accepted and n[0] == 1
        np.testing.assert_allclose(c, [1, 1 / 3, 1])
    # a greedy draft: the chance is p's, and the rejected token is not drawn again
    a, n, c = R.verify(p, [1, 0, 1], [0, 3], [0.0, 0.3, 0.8], [1.0])
    assert a[0] == 0 and n[0] == 1
    np.testing.assert_allclose(c, [1, 0.25, 0.75])
    a, n, _ = R.verify(p, [1, 1, 0], [0, 3], [0.1, 0.3, 0.2], [1.0])
    assert a[0] == 2 and n[0] == 0
