"""Some of a batch's requests by pointers into its plan: row_start[0] above zero.  Rows of the requests before and behind stay as
they were, whatever the workspace holds."""
import numpy as np
import pytest
import torch

from tests.test_gpu_paged import TYPES, TYPE_IDS, Dev, Packed, Paged, check, i32

pytestmark = pytest.mark.gpu


class At:
    def __init__(self, dev, skip):
        self.ptr = dev.ptr + 4 * skip


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new,kv", [([1, 1, 1, 1], [900, 700, 1200, 5]), ([3, 4, 2, 5], [900, 700, 1200, 77]), ([90, 70, 100, 30], [900, 700, 1200, 77]),
                                    ([1, 90, 1, 3], [900, 700, 1200, 77]), ([1, 1, 1, 1], [900, 30000, 100, 5])],
                         ids=["decode", "few", "tiles", "mixed", "many_ranges"])
@pytest.mark.parametrize("a,b,fill", [(1, 3, 0x02), (2, 4, 0x02), (1, 2, 0xFF)])
def test_requests_a_to_b(hip, qtype, new, kv, a, b, fill):
    print(f"[case] part {qtype} {new} {kv} {a}:{b} fill={fill}", flush=True)
    p = Paged(hip, 33, qtype, 8, 2, 64, 16, new, kv)
    H, ld = p.H, p.H * p.hd
    first, last = int(p.start[a]), int(p.start[b])
    want = p.want()[first:last]
    dq, out = Dev(torch.from_numpy(p.q.reshape(p.rows, ld))), Dev(torch.full((p.rows, ld), 5.0))
    table, start, lens = i32(p.table), i32(p.start), i32(p.kv)
    args = (b - a, p.rows, max(new[a:b]), max(kv[a:b]))
    ws = Dev(torch.full((max(hip.paged_attention_workspace_bytes(H, p.pool, *args), 16),), fill, dtype=torch.uint8))
    torch.cuda.synchronize()
    hip.paged_attention(dq, ld, out, ld, H, p.pool, At(table, a * p.ld), p.ld, At(start, a), At(lens, a), *args, float(p.scale), ws=ws)
    hip.sync()
    got = out.np().reshape(p.rows, H, p.hd)
    assert (got[:first] == 5.0).all() and (got[last:] == 5.0).all()
    check(got[first:last], want, f"requests {a} to {b}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("way", ["rows", "prepared"])
def test_prompts_a_to_b(hip, monkeypatch, qtype, hd, way):
    monkeypatch.setenv("EF_HIP_PACKED_ATTENTION", way)
    print(f"[case] part packed {qtype} hd={hd} {way}", flush=True)
    p = Packed(hip, 34, qtype, 4, 2, hd, [150, 70, 0, 130, 60])
    p.run()
    q, k, v, out, start, ws, (ldq, ldk, ldv, n) = p.dev
    a, b = 1, 4
    out.t.fill_(5.0)
    part = At(start, a)
    torch.cuda.synchronize()
    hip.packed_attention(q, ldq, k, ldk, v, ldv, qtype, out, ldq, 4, 2, hd, part, b - a, n, float(1.0 / np.sqrt(hd)), ws=ws)
    hip.sync()
    got, first, last = out.np()[:, :4 * hd].reshape(n, 4, hd), int(p.start[a]), int(p.start[b])
    assert (got[:first] == 5.0).all() and (got[last:] == 5.0).all()
    check(got[first:last], p.want()[first:last], "prompts")
