"""The most positions of a request: on the CPU, nothing is launched (a call that is in order asks for ef_hip_init)."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
import ctypes as C, sys
from edgeforge_amd import _lib as L
P, lib, wrong = 0x10000, L.lib(), []
def attend(page, ld):
    pool = L.ef_hip_page_pool(P, P, L.F16, 9, page, 2, 64, 0)
    b = L.ef_hip_paged_batch(P, P, P, ld, 1, 8, 1, 100)
    return lib.ef_hip_paged_attention(P, 256, P, 256, 4, C.byref(pool), C.byref(b), 0.125, P, 1 << 40, None)
most = 2 ** 31 - 1024
for page in (1, 2, 16, 256, 512, 1024):
    for ld, want in ((most // page, L.ESTATE), (most // page + 1, L.EINVAL), ((2 ** 31 - 1) // page + 1, L.EINVAL)):
        got = attend(page, ld)
        if got != want: wrong.append((page, ld, got, (lib.ef_hip_last_error() or b"").decode()))
sys.exit(print(wrong) or (1 if wrong else 0))
"""


def test_positions_near_two_to_the_31_are_refused():
    """The kernels look two steps ahead in 32 bits: past 2^31 they would read before the table and never end."""
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
