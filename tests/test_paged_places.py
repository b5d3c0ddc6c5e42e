"""Whose tile a workgroup's place is, on the CPU; and no index of the attention kernels that goes through a floating-point value."""
import os
import subprocess

import pytest

from edgeforge_amd import build as hipbuild

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def compiler():
    if not os.path.exists(hipbuild.HIPCC):
        pytest.skip("no hipcc")


def test_places_of_requests(tmp_path):
    exe = str(tmp_path / "places")
    r = subprocess.run([hipbuild.HIPCC, "--offload-arch=gfx950", "--offload-host-only", "-std=c++17", "-O1", f"-I{hipbuild.CSRC}",
                        os.path.join(ROOT, "tests", "cpp", "places.hip"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("source", ["attn_few", "attn_tiles", "attn_mixed", "paging"])
def test_no_integer_by_way_of_a_double(source):
    """min and max of an unsigned and a signed value are a double's in device code: 2^32 - 1 then passes an int."""
    r = subprocess.run([hipbuild.HIPCC, *hipbuild.DEVICE_FLAGS, "-Werror=float-conversion", "--cuda-device-only", "-fsyntax-only",
                        os.path.join(hipbuild.CSRC, source + ".hip")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
