"""Sequences that share pages without a GPU: what a step asks, workspaces and argument rules (a host
program), refusals of the C entry points and of the Python class, the plain step that the GPU tests
compare with."""

import ctypes
import os
import random
import subprocess

import pytest

from kv4_ref import Plan
from kv4_shared_ref import SharedPlan
from mirror_sd_amd import _lib

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 4096   # aligned, never read


@pytest.mark.parametrize("flags", [[], ["-g", "-Xarch_host", "-fsanitize=address", "-Xarch_host",
                                        "-fsanitize=undefined", "-Xarch_host",
                                        "-fno-sanitize-recover=undefined"]])
def test_host_program(tmp_path, flags):
    import shutil
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    exe = str(tmp_path / "check_kv4_shared_host")
    r = subprocess.run([hipcc, "--offload-arch=gfx950", "-std=c++17", "-O1", *flags, "-I",
                        os.path.join(ROOT, "mirror-sd_amd", "csrc"),
                        os.path.join(ROOT, "tests", "check_kv4_shared_host.hip"), "-o", exe],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


@pytest.mark.parametrize("bad,needle", [
    (dict(page=48), "page rows"), (dict(n_seq=0), "sequences"), (dict(width=0), "width"),
    (dict(n_pages=1 << 26), "pool pages"), (dict(max_rows=-1), "negative"), (dict(n_kv=0), "kv heads"),
    (dict(n_layers=0), "layers"), (dict(layer_bytes=100), "bytes"), (dict(table=None), "null"),
    (dict(refs=None), "null"), (dict(scratch=None), "null"), (dict(positions=None), "null slot map"),
    (dict(pool=FAKE + 8), "aligned"), (dict(n_seq=65536, width=1 << 13), "2^29")])
def test_fork_refuses_before_device_work(bad, needle):
    L = _lib.load()
    a = dict(n_seq=2, page=64, width=4, n_pages=9, max_rows=3, n_kv=8, n_layers=2, parent=None,
             keep=FAKE, grow=FAKE, lens=FAKE, table=FAKE, refs=FAKE, n_free=FAKE, starts=FAKE,
             slots=FAKE, positions=FAKE, pool=FAKE, layer_bytes=9 * 8 * 2 * 4352, scratch=FAKE,
             err_flags=FAKE)
    a.update(bad)
    assert L.dfl_kv4_fork(ctypes.byref(_lib.DflKv4Fork(**a)), None) == _lib.DFL_EINVAL
    assert needle in L.dfl_last_error().decode()
    assert L.dfl_kv4_fork(None, None) == _lib.DFL_EINVAL
    assert L.dfl_kv4_fork_scratch(0, 4, 9, 0) == L.dfl_kv4_fork_scratch(2, 0, 9, 0) == 0
    assert L.dfl_kv4_fork_scratch(2, 4, 9, 1) == L.dfl_kv4_fork_scratch(2, 4, 9, 0) + 8


def test_shared_attention_refuses_before_device_work():
    L = _lib.load()

    def call(groups=FAKE, n_groups=2, **o):
        a = dict(q=FAKE, out=FAKE, lse=None, q_row=4096, q_head=128, dtype=1, n_rows=3, n_heads=32,
                 n_kv=8, n_seq=3, causal=0, scale=0.1, starts=FAKE, lens=FAKE, table=FAKE, width=4,
                 page=64, n_pages=9, pool=FAKE, ws=FAKE,
                 ws_bytes=L.dfl_kv4_attend_shared_ws(3, 32, 8, 3, 2), err_flags=FAKE)
        a.update(o)
        return L.dfl_kv4_attend_shared(ctypes.byref(_lib.DflKv4Attn(**a)), groups, n_groups, None)

    for bad, needle in [(dict(groups=None), "groups"), (dict(n_groups=0), "groups"),
                        (dict(n_groups=4), "groups"), (dict(dtype=0), "dtype"),
                        (dict(n_heads=30), "multiple"), (dict(ws=None), "workspace"),
                        (dict(ws_bytes=L.dfl_kv4_attend_ws(3, 32, 8, 3)), "workspace"),
                        (dict(q=FAKE + 2), "aligned"), (dict(table=None), "null")]:
        assert call(**bad) == _lib.DFL_EINVAL, bad
        assert needle in L.dfl_last_error().decode(), (bad, L.dfl_last_error())
    assert L.dfl_kv4_attend_shared(None, FAKE, 1, None) == _lib.DFL_EINVAL
    assert call(n_rows=0) == _lib.DFL_OK
    for args in ((0, 32, 8, 3, 2), (3, 30, 8, 3, 2), (3, 32, 8, 3, 0), (3, 32, 8, 3, 4)):
        assert L.dfl_kv4_attend_shared_ws(*args) == 0


def test_refusals_of_the_cache():
    from mirror_sd_amd.kv4 import KV4Cache
    c = KV4Cache.__new__(KV4Cache)
    c.refs, c.max_seqs = None, 3
    with pytest.raises(ValueError, match="shared"):
        c.step(grow=[1, 1, 1], parent=[0, 0, 0])
    with pytest.raises(ValueError):
        KV4Cache(n_kv_heads=1, n_pages=4, max_seqs=2, max_len=64, device="cpu", shared=True)


# ------------------------------------------------------------------ the plain step


def test_plain_steps_without_parents_hold_what_the_plain_step_holds():
    """Lengths, slots' rows and errors are those of the step of sequences that share nothing."""
    rng = random.Random(1)
    a, b = SharedPlan(5, 32, 8, 30), Plan(5, 32, 8, 30)
    for _ in range(50):
        keep = [rng.randint(0, n) for n in a.lens]
        grow = [min(256 - k, rng.choice([0, 1, rng.randint(0, 120)])) for k in keep]
        (starts, _, pos), copies, err = a.step(grow, keep, None, 400)
        (starts2, _, pos2), err2 = b.step(grow, keep, 400)
        assert (starts, pos, err, a.lens) == (starts2, pos2, err2, b.lens) and not copies
        assert [len(t) for t in a.table] == [len(t) for t in b.table]
        held = [p for t in a.table for p in t]
        assert len(held) == len(set(held))


def test_plain_forks():
    p = SharedPlan(3, 32, 8, 20)
    p.step([40, 0, 0], None, None, 40)
    assert p.table == [[0, 1], [], []]
    # two go on from the first, all write into its page: the first stays
    _, copies, err = p.step([1, 1, 1], [40, 40, 40], [0, 0, 0], 3)
    assert err == 0 and copies == [(1, 2, 8), (1, 3, 8)] and p.table == [[0, 1], [0, 2], [0, 3]]
    assert p.refs()[:5] == [3, 1, 1, 1, 0]
    # a holder that only keeps: the one that writes copies
    _, copies, err = p.step([0, 2, 0], [41, 35, 20], [0, 0, 0], 2)
    assert err == 0 and copies == [(1, 2, 3)] and p.table == [[0, 1], [0, 2], [0]]
    assert p.step([250, 250, 250], None, None, 999)[2] == 8 and p.step([200] * 3, None, None, 999)[2] == 16
