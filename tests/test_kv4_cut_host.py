"""Which tiles attention over shared keys takes for the shapes that the GPU tests run: without this a
changed rule could leave a kernel without any test."""

import os
import shutil
import subprocess

import pytest

from kv4_shared_shapes import TILES_32, TILES_128

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    exe = str(tmp_path_factory.mktemp("cut") / "check_kv4_cut_host")
    r = subprocess.run([hipcc, "--offload-arch=gfx950", "-std=c++17", "-O1", "-I",
                        os.path.join(ROOT, "mirror-sd_amd", "csrc"),
                        os.path.join(ROOT, "tests", "check_kv4_cut_host.hip"), "-o", exe],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]

    def run(calls):
        r = subprocess.run([exe, *(str(x) for c in calls for x in c)], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0
        return [tuple(map(int, line.split())) for line in r.stdout.splitlines()]
    return run


@pytest.mark.parametrize("shapes,own,shared,apart", [(TILES_32, 32, 32, False), (TILES_128, 16, 128, True)])
def test_tiles_of_the_shapes(cut, shapes, own, shared, apart):
    calls = [(sum(q), heads, kv, len(q), len(sizes)) for heads, kv, _, sizes, _, _, q in shapes.values()]
    got = cut(calls)
    for name, c in zip(shapes, got):
        assert c[:2] == (own, shared) and (c[3] > 0) == apart, (name, c)


def test_borders_of_the_rule(cut):
    """16 rows a kv head and sequence; 128 and 512 a group."""
    got = cut([(8, 16, 1, 8, 1), (8, 17, 1, 8, 1), (127, 1, 1, 127, 1), (128, 1, 1, 128, 1), (511, 1, 1, 511, 1),
               (512, 1, 1, 512, 1), (1024, 1, 1, 1024, 3), (1024, 1, 1, 1024, 9)])
    assert [c[:2] for c in got] == [(32, 32), (0, 0), (16, 16), (32, 32), (32, 32), (16, 128), (32, 32), (16, 16)]
