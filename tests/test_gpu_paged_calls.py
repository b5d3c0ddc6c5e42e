"""Calls of paged serving beside the ordinary ones: more heads to a KV head than the few-rows kernel takes, packed prompts captured and
replayed, packed calls at once on two streams, requests that share their first pages."""
import numpy as np
import pytest
import torch

from edgeforge_amd import _lib as L
from tests import _data as D
from tests.test_gpu_paged import TYPES, TYPE_IDS, Packed, Paged, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new,kv", [([1], [700]), ([1, 1, 2], [300, 5, 77]), ([40, 1], [300, 90])], ids=["one", "decode", "mixed"])
def test_71_heads_over_one(hip, qtype, new, kv):
    p = Paged(hip, 71, qtype, 71, 1, 64, 16, new, kv)
    check(p.run(), p.want(), f"71 heads {new}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
def test_packed_prompts_replayed_with_other_lengths(hip, monkeypatch, qtype):
    """A captured packed call (prepared tiles and all) over fixed bounds, replayed over other prompts with eager work in between."""
    monkeypatch.setenv("EF_HIP_PACKED_ATTENTION", "prepared")
    p = Packed(hip, 3, qtype, 8, 2, 64, [300, 1, 0, 99])
    p.run()
    q, k, v, out, start, ws, (ldq, ldk, ldv, n) = p.dev
    side, graph, own = torch.cuda.Stream(), torch.cuda.CUDAGraph(), hip.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        p.launch(torch.cuda.current_stream().cuda_stream)
    r = D.rng(4)
    for it in range(6):
        cuts = np.sort(r.integers(0, p.rows + 1, 3))
        start.t.copy_(torch.tensor([0, *cuts, p.rows], dtype=torch.int32))
        k.t[:p.rows].normal_()
        out.t.fill_(5.0)
        torch.cuda.synchronize()
        p.launch(own)
        own.sync()
        eager = out.t.clone()
        out.t.fill_(5.0)
        ws.t.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.t, eager), it
        assert (out.t[:p.rows, :512] != 5.0).all() and (out.t[p.rows:] == 5.0).all()


def test_two_packed_calls_on_two_streams(hip, monkeypatch):
    monkeypatch.setenv("EF_HIP_PACKED_ATTENTION", "prepared")
    s1, s2 = hip.Stream(), hip.Stream()
    a, b = Packed(hip, 61, L.F32, 32, 4, 64, [700, 200]), Packed(hip, 62, L.BF16, 8, 2, 128, [900])
    ra, rb = a.run(), b.run()
    for _ in range(4):
        for x in (a, b):
            x.dev[3].t.fill_(5.0)
            x.dev[5].t.fill_(0xFF)
        torch.cuda.synchronize()
        a.launch(s1)
        b.launch(s2)
        s1.sync()
        s2.sync()
        assert np.array_equal(a.fetch(), ra) and np.array_equal(b.fetch(), rb)


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 2, 1]])
def test_requests_that_share_pages(hip, qtype, new):
    """Block tables that name the same pages: a common beginning, kept once."""
    p = Paged(hip, 7, qtype, 8, 2, 64, 16, new, [200, 177, 128])
    for r in (1, 2):
        p.table[r, :6] = p.table[0, :6]
        p.k[r][:96], p.v[r][:96] = p.k[0][:96], p.v[0][:96]
    check(p.run(table=p.table), p.want(), f"shared {new}")
