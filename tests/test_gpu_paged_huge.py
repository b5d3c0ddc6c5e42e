"""Values near FP32's largest, whose weighted sum before the division would pass it: the mean is finite, and right.

Equal weights and values, or random ones, of the same sign: the mean of n values is off by the weights' 60 u (test_gpu_paged_dims.py) at most."""
import numpy as np
import pytest
import torch

from edgeforge_amd import _lib as L
from tests.test_gpu_paged import TORCH, U, Packed, Paged, prepared  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def close(got, want, what):
    assert np.isfinite(got).all(), what
    rel = np.abs(got.astype(np.float64) / want - 1).max()
    print(f"{what}: {rel / U:.1f} u", flush=True)
    assert rel < 60 * U, what


def values(v, how):
    return np.abs(v) % 0.49 + 0.5 if how == "spread" else np.full_like(v, 0.99)


@pytest.mark.parametrize("qtype", [L.F32, L.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("size,how", [(2.0 ** 128, "same"), (2.0 ** 119, "spread")], ids=["largest", "sums"])
@pytest.mark.parametrize("new,kv", [([1, 1], [700, 2]), ([4, 2], [700, 77]), ([100, 70], [700, 90]), ([100, 1], [230, 1500])],
                         ids=["decode", "few", "tiles", "mixed"])
def test_paged(hip, qtype, hd, size, how, new, kv):
    print(f"[case] huge {qtype} hd={hd} {size} {how} {new}", flush=True)
    p = Paged(hip, hd, qtype, 4, 2, hd, 16, new, kv)
    for r, n in enumerate(kv):
        v = torch.from_numpy(values(p.v[r], how) * size).to(TORCH[qtype])
        p.v[r] = v.double().numpy()
        for j in range(n):
            pg, off = p.place(r, j)
            p.vp.t[pg].view(2, 16, hd)[:, off] = v[j].cuda()
    close(p.run(), p.want(), f"{size}")


@pytest.mark.parametrize("qtype", [L.F32, L.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("size,how", [(2.0 ** 128, "same"), (2.0 ** 119, "spread")], ids=["largest", "sums"])
def test_packed(hip, prepared, qtype, hd, size, how):  # noqa: F811
    print(f"[case] huge packed {qtype} hd={hd} {size} {how}", flush=True)
    p = Packed(hip, hd, qtype, 4, 2, hd, [150, 2, 1])
    p.v = torch.from_numpy(values(p.v.double().numpy(), how) * size).to(TORCH[qtype])
    close(p.run(), p.want(), f"{size}")


def test_a_huge_range_beside_an_ordinary_one(hip):
    """Ranges of positions that are joined: sums near FP32's largest in each of them."""
    p = Paged(hip, 5, L.F32, 4, 1, 64, 16, [1], [9000])
    v = np.abs(p.v[0]) % 0.5 + 0.5
    v *= np.where(np.arange(9000) < 4000, 2.0 ** 100, 2.0 ** 120)[:, None, None]
    v32 = torch.from_numpy(v).float()
    p.v[0] = v32.double().numpy()
    for j in range(9000):
        pg, off = p.place(0, j)
        p.vp.t[pg].view(1, 16, 64)[:, off] = v32[j].cuda()
    close(p.run(), p.want(), "ranges")
