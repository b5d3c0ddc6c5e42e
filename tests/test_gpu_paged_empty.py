"""Rows whose scores are all -inf: exact zeros as for a row that sees nothing, and their neighbours as ever."""
import numpy as np
import pytest

from tests.test_gpu_paged import TYPES, TYPE_IDS, Packed, Paged, check, prepared  # noqa: F401 (a fixture)
from edgeforge_amd import _lib as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("new,kv", [([1, 1], [130, 77]), ([5, 2], [130, 77]), ([100, 70], [130, 77]), ([100, 1], [130, 77])],
                         ids=["decode", "few", "tiles", "mixed"])
def test_paged(hip, qtype, hd, new, kv):
    print(f"[case] all -inf {qtype} hd={hd} {new} {kv}", flush=True)
    p = Paged(hip, hd + new[0], qtype, 4, 1, hd, 16, new, kv)
    want = p.want()
    for j in range(kv[0]):
        p.put("k", 0, j, 0, 0, -np.inf)
    p.q[:new[0], :, 0] = np.abs(p.q[:new[0], :, 0]) + 1.0  # -inf times a positive value: every score of request 0
    got = p.run()
    assert (got[:new[0]] == 0.0).all()
    check(got[new[0]:], want[new[0]:], "beside")


@pytest.mark.parametrize("qtype", [L.F32, L.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_packed(hip, prepared, qtype, hd):  # noqa: F811
    _packed(hip, qtype, hd)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_packed_f16(hip, hd):
    _packed(hip, L.F16, hd)


def _packed(hip, qtype, hd):
    print(f"[case] all -inf packed {qtype} hd={hd}", flush=True)
    p = Packed(hip, hd, qtype, 4, 2, hd, [130, 77])
    want = p.want()
    p.k[:130, :, 0] = -np.inf
    p.q[:130, :, 0] = np.abs(p.q[:130, :, 0]) + 1.0
    got = p.run()
    assert (got[:130] == 0.0).all()
    check(got[130:], want[130:], "beside")
