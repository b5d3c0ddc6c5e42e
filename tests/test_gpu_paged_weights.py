"""Small weights before large values: positions far below a row's largest score whose values outweigh that.

A weight's two halves hold it to 2^-25, and a row's largest weight is kept at 2^13 or more: what a weight is off by is
2^-38 of the largest at most, beside what it is off by itself.  That is 60 u where the exponent's argument is up to 14
(test_gpu_paged_dims.py).  Here it is up to 21 / ln 2 = 31: its rounding is half an ulp of 16 .. 32, 16 u, for 8, and c2's two roundings
(1.5 u relative) make 47 u of it for 21: ln 2 (16 + 47) = 44 u for 20: 84 u.  The top positions' scores are exact where their other dims are zero ("exact").  Otherwise
they are sums around the gap, whose hd roundings are at its size and at random: each within half an ulp, that is u gap at most,
evenly, so with a standard deviation of u gap / sqrt(3), together sqrt(hd / 3) u gap.  The largest of the some 10^3 sums of
a test is at 3.3 standard deviations, 2 sqrt(hd) u gap, and every weight is relative to theirs.
A component: 84 u (+ 2 sqrt(hd) gap u) of sum_j p_j |v_jd|, and 2^-38 sum_j |v_jd| p_max."""
import numpy as np
import pytest
import torch

from edgeforge_amd import _lib as L
from tests.test_gpu_paged import TORCH, TYPES, TYPE_IDS, U, Packed, Paged, prepared  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

# e^-18 = 2^-26; whether the top scores are exact
GAP = pytest.mark.parametrize("gap,exact", [(18.0, True), (21.0, False)], ids=["18-exact", "21-sums"])


def check_rows(got, q, k, v, seen, scale, gap, exact, what):
    worst, off = 0.0, (84 + (0 if exact else 2 * np.sqrt(q.shape[2]) * gap)) * U
    for i in range(len(q)):
        n = seen(i)
        for h in range(q.shape[1]):
            g = h // (q.shape[1] // k.shape[1])
            s = k[:n, g] @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            size = np.abs(v[:n, g])
            tol = off * (p @ size) + 2.0 ** -38 * p.max() * size.sum(0)
            worst = max(worst, (np.abs(got[i, h] - p @ v[:n, g]) / tol).max())
    print(f"{what}: worst component {worst:.2f} of its tolerance", flush=True)
    assert worst < 1.0, what


def keys_apart(k, q, top, gap, exact, hd):
    """Scores around 0, those of the positions `top` higher by `gap`."""
    k *= 0.25
    if exact:
        k[top] = 0.0
    k[..., 0] = 0.0
    k[top, ..., 0] = gap / 4 * np.sqrt(hd)
    q[..., 0] = 4.0


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("hd", [64, 256])
@GAP
@pytest.mark.parametrize("new,kv", [([1, 1], [230, 77]), ([4, 2], [230, 77]), ([100, 70], [230, 90]), ([100, 1], [230, 77])],
                         ids=["decode", "few", "tiles", "mixed"])
def test_paged(hip, qtype, hd, gap, exact, new, kv):
    print(f"[case] weights {qtype} hd={hd} gap={gap} {new}", flush=True)
    p = Paged(hip, hd, qtype, 4, 2, hd, 16, new, kv)
    for r, n in enumerate(kv):
        keys_apart(p.k[r], p.q, [1, 5], gap, exact, hd)
        p.v[r][16:48] *= 2.0 ** 13
        for j in range(n):
            pg, off = p.place(r, j)
            for pool, host in ((p.kp, p.k), (p.vp, p.v)):
                view = pool.t[pg].view(2, 16, hd)
                view[:, off] = torch.from_numpy(host[r][j]).to(TORCH[qtype]).cuda()
                host[r][j] = view[:, off].double().cpu().numpy()
    got = p.run().astype(np.float64)
    for r, n in enumerate(new):
        a = p.start[r]
        check_rows(got[a:a + n], p.q[a:a + n].astype(np.float64), p.k[r], p.v[r], lambda i: kv[r] - n + i + 1, p.scale, gap, exact, f"request {r}")


@pytest.mark.parametrize("hd", [64, 256])
@GAP
def test_packed_f16(hip, hd, gap, exact):
    _packed(hip, L.F16, hd, gap, exact, 13)


@pytest.mark.parametrize("qtype", [L.F32, L.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 256])
@GAP
@pytest.mark.parametrize("bits", [9, 16])
def test_packed(hip, prepared, qtype, hd, gap, exact, bits):  # noqa: F811
    _packed(hip, qtype, hd, gap, exact, bits)


# A whole tile's values 2^40 times the others', at weights of e^-35 = 2^-50: taken in FP32, so no weight is lost.  The exponent's argument is
# up to 50: its rounding is half an ulp of 32 .. 64, 32 u, c2's roundings 75 u of it: ln 2 (32 + 75) = 74 u for 20 of the 60 u.
@pytest.mark.parametrize("qtype", [L.F32, L.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("first", [0, 64, 128])
def test_packed_tile_far_larger(hip, prepared, qtype, hd, first):  # noqa: F811
    print(f"[case] far larger tile {qtype} hd={hd} at {first}", flush=True)
    p = Packed(hip, hd, qtype, 4, 2, hd, [200])
    k, v = p.k.double().numpy(), p.v.double().numpy()
    keys_apart(k, p.q, [(first + 64) % 192 + 1, (first + 64) % 192 + 5], 35.0, True, hd)
    v[first:first + 64] *= 2.0 ** 40
    p.k, p.v = torch.from_numpy(k).to(TORCH[qtype]), torch.from_numpy(v).to(TORCH[qtype])
    q, k, v, got, worst = p.q.astype(np.float64), p.k.double().numpy(), p.v.double().numpy(), p.run().astype(np.float64), 0.0
    for i in range(p.rows):
        for h in range(4):
            s = k[:i + 1, h // 2] @ q[i, h] / np.sqrt(hd)
            w = np.exp(s - s.max())
            w /= w.sum()
            worst = max(worst, (np.abs(got[i, h] - w @ v[:i + 1, h // 2]) / (114 * U * (w @ np.abs(v[:i + 1, h // 2])))).max())
    print(f"worst component {worst:.2f} of its tolerance", flush=True)
    assert worst < 1.0


def _packed(hip, qtype, hd, gap, exact, bits):
    print(f"[case] weights packed {qtype} hd={hd} gap={gap} {bits}", flush=True)
    p = Packed(hip, hd, qtype, 4, 2, hd, [200])
    k, v = p.k.double().numpy(), p.v.double().numpy()
    keys_apart(k, p.q, [1, 5], gap, exact, hd)
    v[64:128] *= 2.0 ** bits
    p.k, p.v = torch.from_numpy(k).to(TORCH[qtype]), torch.from_numpy(v).to(TORCH[qtype])
    check_rows(p.run().astype(np.float64), p.q.astype(np.float64), p.k.double().numpy(), p.v.double().numpy(), lambda i: i + 1, 1.0 / np.sqrt(hd), gap, exact, "packed")
