"""The paged 4-bit cache without a GPU: index maps, the split of the work and the argument rules (a
host program), refusals of the C entry points and of the Python class, the plain implementation
that the GPU tests compare with."""

import ctypes
import os
import subprocess

import numpy as np
import pytest

import kv4_ref as R
from mirror_sd_amd import _lib

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("flags", [[], ["-g", "-Xarch_host", "-fsanitize=address", "-Xarch_host",
                                        "-fsanitize=undefined", "-Xarch_host",
                                        "-fno-sanitize-recover=undefined"]])
def test_host_program(tmp_path, flags):
    import shutil
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    exe = str(tmp_path / "check_kv4_host")
    r = subprocess.run([hipcc, "--offload-arch=gfx950", "-std=c++17", "-O1", *flags, "-I",
                        os.path.join(ROOT, "mirror-sd_amd", "csrc"),
                        os.path.join(ROOT, "tests", "check_kv4_host.hip"), "-o", exe],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


FAKE = ctypes.c_void_p(4096)   # aligned, never read


def test_entry_points_refuse_before_device_work():
    L = _lib.load()

    def step(**o):
        a = dict(n_seq=2, page=64, width=4, n_pages=9, keep=FAKE, grow=FAKE, lens=FAKE, table=FAKE,
                 free=FAKE, n_free=FAKE, max_rows=3, starts=FAKE, slots=FAKE, positions=FAKE,
                 scratch=FAKE, err=FAKE)
        a.update(o)
        return L.dfl_kv4_step(*a.values(), None)

    def append(**o):
        a = dict(k=FAKE, k_row=1024, k_head=128, v=FAKE, v_row=1024, v_head=128, dtype=1, rows=3,
                 n_kv=8, page=64, n_pages=9, slots=FAKE, pool=FAKE, err=FAKE)
        a.update(o)
        return L.dfl_kv4_append(*a.values(), None)

    def read(**o):
        a = dict(slots=FAKE, rows=3, n_kv=8, page=64, n_pages=9, pool=FAKE, dtype=1, k=FAKE, v=FAKE,
                 err=FAKE)
        a.update(o)
        return L.dfl_kv4_read(*a.values(), None)

    def attend(**o):
        a = dict(q=FAKE, out=FAKE, lse=None, q_row=4096, q_head=128, dtype=1, n_rows=3, n_heads=32,
                 n_kv=8, n_seq=2, causal=0, scale=0.1, starts=FAKE, lens=FAKE, table=FAKE, width=4,
                 page=64, n_pages=9, pool=FAKE, ws=FAKE,
                 ws_bytes=L.dfl_kv4_attend_ws(3, 32, 8, 2), err_flags=FAKE)
        a.update(o)
        return L.dfl_kv4_attend(ctypes.byref(_lib.DflKv4Attn(**a)), None)

    odd = ctypes.c_void_p(4104)
    for call, bad, needle in [
            (step, dict(page=48), "page rows"), (step, dict(page=16), "page rows"),
            (step, dict(page=0), "page rows"), (step, dict(page=-64), "page rows"),
            (step, dict(n_seq=0), "sequences"), (step, dict(width=0), "width"),
            (step, dict(n_pages=1 << 25), "pool pages"), (step, dict(max_rows=-1), "negative"),
            (step, dict(table=None), "null"), (step, dict(err=None), "null"),
            (append, dict(dtype=3), "dtype"), (append, dict(rows=-1), "negative"),
            (append, dict(k=odd), "aligned"), (append, dict(v_row=1028), "strides"),
            (append, dict(slots=None), "null"), (append, dict(n_kv=0), "kv heads"),
            (read, dict(dtype=-1), "dtype"), (read, dict(v=None), "null"),
            (read, dict(page=33), "page rows"),
            (attend, dict(dtype=0), "dtype"), (attend, dict(n_heads=30), "multiple"),
            (attend, dict(n_heads=0), "multiple"), (attend, dict(scale=0.0), "scale"),
            (attend, dict(scale=float("nan")), "scale"), (attend, dict(q_row=4100), "strides"),
            (attend, dict(ws_bytes=16), "workspace"), (attend, dict(ws=None), "workspace"),
            (attend, dict(out=None), "null"), (attend, dict(q=odd), "aligned"),
            (attend, dict(n_seq=70000), "sequences")]:
        assert call(**bad) == _lib.DFL_EINVAL, (call.__name__, bad)
        assert needle in L.dfl_last_error().decode(), (bad, L.dfl_last_error())
    assert L.dfl_kv4_attend(None, None) == _lib.DFL_EINVAL
    # nothing to do is no error, and no launch
    assert append(rows=0) == read(rows=0) == attend(n_rows=0) == _lib.DFL_OK
    assert L.dfl_kv4_step_scratch(0) == 0 and L.dfl_kv4_step_scratch(5) >= 15
    assert L.dfl_kv4_attend_ws(0, 32, 8, 2) == 0 and L.dfl_kv4_attend_ws(3, 30, 8, 2) == 0


def _cache(**kw):
    """A cache object without a device: what its checks see before any call."""
    from mirror_sd_amd.kv4 import KV4Cache
    c = KV4Cache.__new__(KV4Cache)
    c.n_kv_heads, c.max_seqs, c.n_layers, c.page, c.n_pages, c.width = 2, 3, 2, 32, 5, 4
    c.device = torch.device("cpu")
    c.pool = torch.zeros((2, 5, 2, 1, 4352), dtype=torch.uint8)
    c._codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    return c


def test_cache_refuses_what_does_not_fit():
    from mirror_sd_amd.kv4 import KV4Cache
    for bad in (dict(page=48), dict(page=16), dict(n_kv_heads=0), dict(n_pages=0), dict(max_seqs=0),
                dict(max_len=0), dict(n_layers=0), dict(max_seqs=65537), dict(n_pages=2**26),
                dict(device="cpu")):
        with pytest.raises(ValueError):
            KV4Cache(**dict(dict(n_kv_heads=2, n_pages=4, max_seqs=2, max_len=64), **bad))
    c = _cache()
    k = torch.zeros((4, 2, 128), dtype=torch.float16)
    slots = torch.zeros(4, dtype=torch.int32)
    for args in [(k[:, :1], k, slots), (k, k[:3], slots), (k, k.float(), slots), (k.double(), k.double(), slots),
                 (k[:, :, :64], k[:, :, :64], slots), (k[0], k[0], slots), (k.to("meta"), k, slots)]:
        with pytest.raises(ValueError):
            c.append(*args)
    q = torch.zeros((4, 6, 128), dtype=torch.float16)
    starts = torch.zeros(4, dtype=torch.int32)
    for args, kw in [((q.float(), starts), {}), ((q[:, :5], starts), {}), ((q[:, :0], starts), {}),
                     ((q, starts), dict(out=q[:3])), ((q, starts), dict(out=q.bfloat16())),
                     ((q, starts), dict(out=torch.zeros((4, 12, 128), dtype=torch.float16)[:, ::2]))]:
        with pytest.raises(ValueError):
            c.attend(*args, **kw)
    with pytest.raises(ValueError):
        c.read(slots, dtype=torch.int8)
    for t, n in [(torch.zeros(3), 3), (torch.zeros((3, 1), dtype=torch.int32), 3),
                 (torch.zeros(2, dtype=torch.int32), 3), (torch.zeros(3, dtype=torch.bool), 3)]:
        with pytest.raises(ValueError):
            c._ints(t, n, "grow")
    for layer in (-1, 2):
        with pytest.raises(ValueError):
            c._layer(layer)
    with pytest.raises(ValueError):
        c.step(grow=[1, 2, 3], max_rows=-1)


def test_counts_from_the_host_are_what_they_say():
    """Lists and arrays: what 32 bits do not hold stays out of range (not its low bits, and never the
    -1 that skips a row), fractions and truth values are refused as on the device."""
    c = _cache()
    lo, hi = -2**31, 2**31 - 1
    for given, want in [([3, -1], [3, -1]), ([], []), ((5,), [5]), (range(3), [0, 1, 2]), ([2**32 + 5, -2**40], [hi, lo]),
                        (np.array([2**32 + 5, -2**32 - 1, 7]), [hi, lo, 7]), (np.array([7, -1], np.int16), [7, -1]),
                        (np.array([7, 2**32 - 1], np.uint32), [7, hi]), (np.array([2**16 - 1], np.uint16), [65535]),
                        (np.zeros(0, np.int64), [])]:
        got = c._ints(given, None, "slots")
        assert got.dtype == torch.int32 and got.tolist() == want, given
    for bad in ([0.5], np.array([2.0]), np.zeros(2), [True], np.array([False]), np.array([1], np.uint64)):
        with pytest.raises(ValueError, match="integers"):
            c._ints(bad, None, "slots")
    with pytest.raises(ValueError, match="integers"):
        c.step(grow=[0.5, 0.25, 0.25])


def test_results_over_queries_that_are_still_read_are_refused():
    c = _cache()
    starts = torch.zeros(4, dtype=torch.int32)
    buf = torch.zeros((9, 6, 128), dtype=torch.float16)
    for q, out in [(buf[:4], buf[1:5]), (buf[3:7], buf[:4]), (buf[:8:2], buf[4:8]),
                   (buf.view(9, 768)[:, :512].unflatten(1, (4, 128)), buf.view(-1)[512:512 + 9 * 512].view(9, 4, 128)[:9])]:
        with pytest.raises(ValueError, match="overlap"):
            c.attend(q, starts, out=out)


def test_rows_are_read_in_place_where_they_can_be():
    c = _cache()
    wide = torch.zeros((5, 1024), dtype=torch.float16)
    k = wide[:, 128:384].unflatten(1, (2, 128))
    assert c._rows(k, 2, "k") is k
    assert c._rows(torch.zeros((2, 9, 128)).transpose(0, 1), 2, "k").stride() == (128, 1152, 1)
    for odd in (wide[:, 1:257].unflatten(1, (2, 128)), torch.zeros((5, 260))[:, :256].unflatten(1, (2, 128)),
                torch.zeros((5, 128, 2)).transpose(1, 2)):
        got = c._rows(odd, 2, "k")
        assert got is not odd and got.is_contiguous() and torch.equal(got, odd)


def test_plain_rows_against_every_choice():
    """The plain row format against a search: of all exponents without clipping by more than half a
    step the smallest, and the nearest code, an even one of two as near."""
    rng = np.random.default_rng(0)
    for trial in range(300):
        x = rng.standard_normal(128) * 2.0 ** rng.integers(-30, 30)
        if trial % 3 == 0:
            x = np.round(x / np.abs(x).max() * 28) / 4 * 2.0 ** rng.integers(-20, 20)
        got = R.values(x)
        for g in range(4):
            part, out = x[32 * g:32 * g + 32], got[32 * g:32 * g + 32]
            top = np.abs(part).max()
            e = next(e for e in range(-127, 128) if top <= 7 * 2.0 ** e)
            for a, b in zip(part, out):
                d = np.abs(np.abs(a) / 2.0 ** e - R.GRID)
                best = [c for c in range(8) if d[c] == d.min()]
                c = best[0] if len(best) == 1 or best[0] % 2 == 0 else best[1]
                assert b == np.copysign(R.GRID[c] * 2.0 ** e, a)


def test_plain_attention_against_torch():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 6, 128), (9, 2, 128), (9, 2, 128)))
    for causal in (False, True):
        out, lse, _, (size, _) = R.attend(q.numpy(), k.numpy(), v.numpy(), causal, 0.1)
        s = torch.einsum("mhd,nhd->hmn", q, k.repeat_interleave(3, 1)) * 0.1
        if causal:
            s = s.masked_fill(torch.ones(5, 9, dtype=torch.bool).triu(5), -float("inf"))
        want = torch.einsum("hmn,nhd->mhd", torch.softmax(s, -1), v.repeat_interleave(3, 1))
        np.testing.assert_allclose(out, want.numpy(), rtol=1e-12, atol=1e-12)
        np.testing.assert_allclose(lse, torch.logsumexp(s, -1).T.numpy(), rtol=1e-12)
        assert (size > 0).all()
    out, lse, _, _ = R.attend(q.numpy(), k[:3].numpy(), v[:3].numpy(), True, 0.1)
    assert (out[:2] == 0).all() and np.isneginf(lse[:2]).all() and np.isfinite(lse[2:]).all()
