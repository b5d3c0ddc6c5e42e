"""FP32 decodes are no further from float64 than a plain FP32 computation is: products with the library's FP32 matrix product, softmax
and sums in FP32, on inputs whose scores share a part of about 3, as trained models' do (that part's size is what the score's
roundings are relative to, so that long sums of it show)."""
import numpy as np
import pytest
import torch

from edgeforge_amd import _lib as L
from tests.test_gpu_paged import U, Paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,KV,hd,new,kv", [(32, 4, 64, [1], [2047]), (32, 8, 128, [1, 1], [900, 700]), (8, 4, 256, [1, 1], [900, 800]), (16, 2, 64, [4], [1500])],
                         ids=["64", "128", "256", "64-few"])
def test_error_against_a_plain_computation(hip, H, KV, hd, new, kv):
    own, plain = [], []
    for seed in range(5):
        p = Paged(hip, 100 + seed, L.F32, H, KV, hd, 16, new, kv)
        common = np.zeros(hd, np.float32)
        common[:4] = np.sqrt(3.0 * np.sqrt(hd) / 4.0)
        p.q += common
        for r, n in enumerate(kv):
            p.k[r] = (p.k[r] + common).astype(np.float32).astype(np.float64)
            for j in range(n):
                pg, off = p.place(r, j)
                p.kp.t[pg].view(KV, 16, hd)[:, off] = torch.from_numpy(p.k[r][j]).float().cuda()
        want = p.want()
        own.append(np.linalg.norm(p.run() - want) / np.linalg.norm(want))
        got = np.zeros_like(want)
        for r, n in enumerate(new):
            k, v = (torch.from_numpy(x[r]).float().cuda() for x in (p.k, p.v))
            for i in range(n):
                q = torch.from_numpy(p.q[p.start[r] + i]).cuda()
                m = kv[r] - n + i + 1
                for h in range(H):
                    g = h // (H // KV)
                    s = (k[:m, g].contiguous() @ q[h]) * p.scale
                    w = torch.exp(s - s.max())
                    got[p.start[r] + i, h] = ((w @ v[:m, g].contiguous()) / w.sum()).double().cpu().numpy()
        plain.append(np.linalg.norm(got - want) / np.linalg.norm(want))
    print(f"{H}/{KV}/{hd}: {np.mean(own) / U:.1f} u, plain {np.mean(plain) / U:.1f} u", flush=True)
    assert np.mean(own) < np.mean(plain)
