"""FP32 keys and values, and BF16 ones prepared as FP16 tiles, whose sizes differ from dim to dim and from row to row:
every component of the output against float64, as its own dim's size has it.

Values are v = r_j c_d n_jd with n ~ N(0, 1), weights spread over the positions.  Tolerance of a component, in units of
u = 2^-24, relative to sum_j p_j |v_jd|: a weight's own error is below 48 u (the score's sums, the exponent's rounding, exp2,
the sum; derived in test_gpu_paged.py's tolerances for weights that nothing averages) and value parts keep 22 bits
(4 u) or more, the output's own sums 8 u: 60 u.  What a part's smallest step drops is at most u of the largest value of its row
times the largest of its dim over the largest of the tile, 4.5 * 4.5 / 3 < 7 times r_j c_d with N(0, 1): 7 u relative to
sum_j p_j r_j c_d.  Weights of less than 2^-14 of a row's largest, at 2^-36 of it, change a sum by less than u where rows differ by
2^12 and less (what is taken from tiles), as N(0, 1) scores hardly have any.  A key's dims are seen through the scores only: the same
bounds on the outputs, as the score's error is relative to sum_d |q_d| max_j |k_jd|, which the tests keep at its usual size."""
import numpy as np
import pytest
import torch

from edgeforge_amd import _lib as L
from tests.test_gpu_paged import TORCH, U, Packed, Paged, prepared  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

# 2 to the power of: value dims, value rows, one key dim (the queries are zero there), other key dims (queries the other way)
HOW = {"v_dims_9": (9, 0, 0, 0), "v_dims_16": (16, 0, 0, 0), "v_dims_40": (40, 0, 0, 0), "v_both_12": (12, 12, 0, 0), "k_dim_14": (0, 0, 14, 0),
       "k_dim_30": (0, 0, 30, 0),
       "k_dims": (0, 0, 0, 12), "zero_dims": (3, 0, 0, 0), "late_dims": (3, 0, 0, 0), "late_small_dims": (30, 0, 0, 0)}


def factors(how, rows, hd):
    """zero_dims: some hold nothing else; late_..: some hold something in the last rows of 64 only."""
    v_dim, v_row, k_dim, k_dims = HOW[how]
    d, j = np.arange(hd), np.arange(rows)
    c = 2.0 ** -(v_dim * (d % 3) / 2.0).round()
    r = 2.0 ** -(v_row * (j % 5 == 2))
    kf = 2.0 ** -(k_dims * (d % 2))
    qf = 1.0 / kf
    if k_dim:
        kf[hd // 3], qf[hd // 3] = 2.0 ** k_dim, 0.0
    rc = r[:, None, None] * c
    if how == "zero_dims":
        rc[..., d % 4 == 1] = 0.0
        kf = kf * (d % 5 != 3)
    elif how.startswith("late"):
        rc = rc * np.where((d % 3 == 2) & (j % 64 < 40)[:, None, None], 0.0, 1.0)
    return rc, kf, qf


def component_check(got, q, k, v, rc, scale, seen_of, what):
    rows, H, hd = q.shape
    KV, worst = k.shape[1], 0.0
    for i in range(rows):
        n = seen_of(i)
        for h in range(H):
            g = h // (H // KV)
            s = k[:n, g] @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            tol = 60 * U * (p @ np.abs(v[:n, g])) + 7 * U * (p @ np.broadcast_to(rc, v.shape)[:n, g])
            worst = max(worst, (np.abs(got[i, h] - p @ v[:n, g]) / np.maximum(tol, 1e-300)).max())
    print(f"{what}: worst component {worst:.2f} of its tolerance", flush=True)
    assert worst < 1.0, what


@pytest.mark.parametrize("qtype", [L.F32, L.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("how", HOW)
def test_packed_dims(hip, prepared, qtype, hd, how):  # noqa: F811
    print(f"[case] dims packed {'prepared' if prepared else 'rows'} {qtype} hd={hd} {how}", flush=True)
    p = Packed(hip, hd, qtype, 2, 1, hd, [150])
    rc, kf, qf = factors(how, p.rows, hd)
    p.v = (p.v.double() * torch.from_numpy(rc)).to(TORCH[qtype])
    p.k = (p.k.double() * torch.from_numpy(kf)).to(TORCH[qtype])
    p.q = (p.q * qf).astype(np.float32)
    got = p.run().astype(np.float64)
    component_check(got, p.q.astype(np.float64), p.k.double().numpy(), p.v.double().numpy(), rc, 1.0 / np.sqrt(hd), lambda i: i + 1, how)


@pytest.mark.parametrize("hd,new", [(96, [90]), (128, [90]), (64, [2])], ids=["96-chunk", "128-chunk", "64-few"])
@pytest.mark.parametrize("how", HOW)
def test_paged_dims(hip, hd, how, new):
    kv = [230]
    print(f"[case] dims paged hd={hd} {how} {new}", flush=True)
    p = Paged(hip, hd, L.F32, 2, 1, hd, 16, new, kv)
    rc, kf, qf = factors(how, kv[0], hd)
    for j in range(kv[0]):
        pg, off = p.place(0, j)
        for pool, host, f in ((p.kp, p.k, kf), (p.vp, p.v, rc[j, 0])):
            pool.t[pg].view(1, 16, hd)[0, off] *= torch.from_numpy(f.astype(np.float32)).cuda()
            host[0][j] *= f
    p.q = (p.q * qf).astype(np.float32)
    got = p.run().astype(np.float64)
    component_check(got, p.q.astype(np.float64), p.k[0], p.v[0], rc, 1.0 / np.sqrt(hd), lambda i: kv[0] - new[0] + i + 1, how)
