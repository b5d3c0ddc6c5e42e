"""What the entry points of paged serving refuse, and where their kernels look for a page: on the CPU, before
anything is launched (a call that is in order gets as far as asking for ef_hip_init)."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from edgeforge_amd import _lib as L
from edgeforge_amd import build as hipbuild

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000  # an address: nothing is read before the call is refused

PROGRAM = r"""
import ctypes as C, sys
from edgeforge_amd import _lib as L
P = 0x10000
lib = L.lib()
pool = dict(k_dev=P, v_dev=P, qtype=L.F16, n_pages=9, page_size=16, KV=2, hd=64, page_stride=0)
plan = dict(cached=P, new=P, n_seqs=3, page_size=16, n_pages=9, table=P, ld=4, free=P, n_free=P, n_free_out=P, kv_len=P,
            row_start=P, pos=P, slot=P, max_rows=8, status=P, stream=None)
append = dict(q=P, ldq=256, q_out=P, ldqo=256, heads=4, k=P, ldk=128, k_out=None, ldko=0, v=P, ldv=128, rows=3, pos=P, cos=P,
              sin=P, n_pos=64, slot=P, pool=None, stream=None)
paged = dict(q=P, ldq=256, out=P, ldo=256, heads=4, pool=None, batch=None, scale=0.125, ws=P, ws_bytes=1 << 40, stream=None)
batch = dict(row_start_dev=P, kv_len_dev=P, table_dev=P, table_ld=4, n_seqs=3, max_rows=8, max_new=4, max_kv=64)
packed = dict(q=P, ldq=256, k=P, ldk=128, v=P, ldv=128, qtype=L.BF16, out=P, ldo=256, heads=4, KV=2, hd=64, row_start=P,
              n_seqs=3, max_rows=8, scale=0.125, ws=P, ws_bytes=1 << 40, stream=None)
tables = dict(theta=1e4, hd=64, n_pos=8, cos=P, sin=P)

def call(name, args, change):
    p = L.ef_hip_page_pool(**{**pool, **{k[5:]: v for k, v in change.items() if k.startswith("pool_")}})
    b = L.ef_hip_paged_batch(**{**batch, **{k[6:]: v for k, v in change.items() if k.startswith("batch_")}})
    a = {**args, **{k: v for k, v in change.items() if not k.startswith(("pool_", "batch_"))}}
    if "pool" in a and "pool" not in change: a["pool"] = C.byref(p)
    if "batch" in a and "batch" not in change: a["batch"] = C.byref(b)
    rc = getattr(lib, name)(*a.values())
    return rc, (lib.ef_hip_last_error() or b"").decode()

bad_pool = [dict(pool_k_dev=None), dict(pool_v_dev=None), dict(pool_qtype=L.Q8_0), dict(pool_n_pages=0), dict(pool_n_pages=1 << 31),
            dict(pool_page_size=0), dict(pool_page_size=12), dict(pool_page_size=2048), dict(pool_KV=0), dict(pool_hd=0),
            dict(pool_hd=60), dict(pool_hd=264), dict(pool_page_stride=100), dict(pool_page_stride=16 * 128 + 4),
            dict(pool_page_stride=1 << 50), dict(pool_k_dev=P + 8), dict(pool_v_dev=P + 2), dict(pool=None)]
refused = {
    "ef_hip_page_plan": (plan, [{k: None} for k in ("cached", "new", "table", "free", "n_free", "n_free_out", "kv_len", "row_start",
                                                    "pos", "slot", "status")] +
        [dict(n_seqs=0), dict(n_seqs=(1 << 20) + 1), dict(page_size=0), dict(page_size=3), dict(page_size=2048), dict(n_pages=0),
         dict(n_pages=1 << 31), dict(ld=0), dict(ld=1 << 28), dict(n_seqs=1 << 20, ld=1 << 12), dict(max_rows=1 << 31)]),
    "ef_hip_rope_tables": (tables, [dict(theta=0.0), dict(hd=63), dict(hd=0), dict(n_pos=0), dict(n_pos=1 << 23), dict(cos=None), dict(sin=None)]),
    "ef_hip_rope_append": (append, bad_pool + [{k: None} for k in ("q", "q_out", "k", "v", "pos", "cos", "sin", "slot")] +
        [dict(heads=0), dict(ldq=252), dict(ldq=258), dict(ldqo=255), dict(ldk=124), dict(ldv=127), dict(k_out=P + 64, ldko=64),
         dict(k_out=P + 4, ldko=128), dict(q=P + 4), dict(q_out=P + 8), dict(k=P + 4), dict(v=P + 12), dict(cos=P + 4), dict(n_pos=0),
         dict(ldq=512), dict(k_out=P, ldko=256), dict(rows=1 << 40)]),
    "ef_hip_paged_attention": (paged, bad_pool + [{k: None} for k in ("q", "out", "batch")] +
        [dict(batch_row_start_dev=None), dict(batch_kv_len_dev=None), dict(batch_table_dev=None), dict(batch_table_ld=0),
         dict(batch_table_ld=1 << 28), dict(batch_n_seqs=0), dict(batch_max_rows=1 << 31), dict(heads=0), dict(heads=3),
         dict(ldq=252), dict(ldq=250), dict(ldo=128), dict(q=P + 4), dict(out=P + 8), dict(scale=0.0), dict(scale=-1.0),
         dict(scale=float("inf")), dict(scale=float("nan"))]),
    "ef_hip_packed_attention": (packed, [{k: None} for k in ("q", "k", "v", "out", "row_start")] +
        [dict(qtype=L.Q4_0), dict(hd=0), dict(hd=36), dict(hd=264), dict(heads=0), dict(heads=3), dict(KV=0), dict(n_seqs=0),
         dict(max_rows=1 << 31), dict(ldq=252), dict(ldk=64), dict(ldk=132), dict(ldv=120), dict(k=P + 8), dict(v=P + 2),
         dict(out=P + 4), dict(scale=0.0), dict(scale=float("nan"))]),
}
wrong = []
for name, (args, changes) in refused.items():
    rc, msg = call(name, args, {})
    if rc != L.ESTATE:
        wrong.append((name, "in order", rc, msg))
    for change in changes:
        rc, msg = call(name, args, change)
        if rc != L.EINVAL or not msg:
            wrong.append((name, change, rc, msg))
print(wrong)
sys.exit(1 if wrong else 0)
"""


def test_refusals():
    """In a process of its own, which has not called ef_hip_init."""
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_workspace_bytes_of_bad_sizes_is_zero():
    lib = L.lib()
    pool = L.ef_hip_page_pool(P, P, L.Q8_0, 9, 16, 2, 64, 0)
    assert lib.ef_hip_paged_attention_workspace_bytes(4, C.byref(pool), 1, 1, 1, 64) == 0
    assert lib.ef_hip_paged_attention_workspace_bytes(4, None, 1, 1, 1, 64) == 0
    assert lib.ef_hip_packed_attention_workspace_bytes(3, 2, 64, L.F32, 1, 1) == 0


def test_pages_and_requests_on_the_cpu(tmp_path):
    if not os.path.exists(hipbuild.LIB):
        pytest.skip("libedgeforge_hip.so not built")
    exe = str(tmp_path / "pages")
    r = subprocess.run([hipbuild.HIPCC, "--offload-arch=gfx950", "--offload-host-only", "-std=c++17", "-O1",
                        f"-I{hipbuild.CSRC}", os.path.join(ROOT, "tests", "cpp", "pages.hip"), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
