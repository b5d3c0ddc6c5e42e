"""max_rows inside a request: the rows before it are as without the cut, whatever kernel takes them, those behind it are
neither read nor written."""
import numpy as np
import pytest
import torch

from tests.test_gpu_paged import TYPES, TYPE_IDS, Dev, Packed, Paged, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new,kv,max_rows", [([1, 1, 1], [300, 77, 5], 2), ([5, 4, 6], [300, 77, 200], 7), ([5, 4], [600, 500], 1),
                                             ([100, 90], [300, 777], 131), ([100, 1, 60], [300, 77, 200], 103), ([100, 1, 60], [300, 77, 2000], 140),
                                             ([200], [900], 3), ([40, 3], [40, 3], 41)],
                         ids=["decode", "few", "few_one", "tiles", "mixed_few_left", "mixed", "tiles_three_left", "prompts"])
def test_rows_before_the_cut(hip, qtype, new, kv, max_rows):
    hd = 64 if len(new) == 3 else 128
    print(f"[case] cut {qtype} hd={hd} {new} {kv} at {max_rows}", flush=True)
    p = Paged(hip, hd + max_rows, qtype, 8, 2, hd, 16, new, kv)
    H, ld = p.H, p.H * hd
    want = p.want()[:max_rows]
    q = np.full((p.rows, ld), np.nan, np.float32)
    q[:max_rows] = p.q[:max_rows].reshape(max_rows, -1)
    args = (len(kv), max_rows, max(new), max(kv))
    ws = Dev(torch.full((max(hip.paged_attention_workspace_bytes(H, p.pool, *args), 16),), 0xFF, dtype=torch.uint8))
    dq, out = Dev(torch.from_numpy(q)), Dev(torch.full((p.rows, ld), 5.0))
    table, start, lens = (Dev(torch.tensor(np.asarray(v, np.int32))) for v in (p.table, p.start, p.kv))
    torch.cuda.synchronize()
    hip.paged_attention(dq, ld, out, ld, H, p.pool, table, p.ld, start, lens, *args, float(p.scale), ws=ws)
    hip.sync()
    got = out.np().reshape(p.rows, H, hd)
    assert (got[max_rows:] == 5.0).all()
    check(got[:max_rows], want, f"cut at {max_rows}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("way", ["rows", "prepared"])
@pytest.mark.parametrize("max_rows", [1, 50, 131, 190])
def test_prompts_before_the_cut(hip, monkeypatch, qtype, way, max_rows):
    monkeypatch.setenv("EF_HIP_PACKED_ATTENTION", way)
    print(f"[case] cut packed {qtype} {way} at {max_rows}", flush=True)
    p = Packed(hip, max_rows, qtype, 4, 2, 64, [50, 100, 0, 70])
    want = p.want()[:max_rows]
    nan = float("nan")
    q, k, v = (torch.full((p.rows, w), nan, dtype=t) for w, t in ((256, torch.float32), (128, p.k.dtype), (128, p.k.dtype)))
    q[:max_rows] = torch.from_numpy(p.q).reshape(p.rows, -1)[:max_rows]
    k[:max_rows], v[:max_rows] = p.k.view(p.rows, -1)[:max_rows], p.v.view(p.rows, -1)[:max_rows]
    dq, dk, dv, out, start = Dev(q), Dev(k), Dev(v), Dev(torch.full((p.rows, 256), 5.0)), Dev(torch.from_numpy(p.start))
    need = hip.packed_attention_workspace_bytes(4, 2, 64, qtype, 4, max_rows)
    ws = Dev(torch.full((max(need, 16),), 0xFF, dtype=torch.uint8))
    torch.cuda.synchronize()
    hip.packed_attention(dq, 256, dk, 128, dv, 128, qtype, out, 256, 4, 2, 64, start, 4, max_rows, 0.125, ws=ws)
    hip.sync()
    got = out.np().reshape(p.rows, 4, 64)
    assert (got[max_rows:] == 5.0).all()
    check(got[:max_rows], want, f"cut at {max_rows}")
