"""What PagedEngine looks at before a step counts its positions: on the CPU, nothing is launched."""
import numpy as np
import pytest

from edgeforge_amd import hip as H
from edgeforge_amd import model as M
from edgeforge_amd.model import Config, PagedEngine


class _Model:
    def __init__(self, hd):
        self.cfg = Config(D=4 * hd, F=64, H=4, KV=4, hd=hd, V=100, L=1, max_pos=64)


def _launched(*a, **k):
    raise AssertionError("went on to the device")


@pytest.mark.parametrize("change", [dict(page_size=12), dict(page_size=0), dict(page_size=2048), dict(pages=0)])
def test_sizes_that_no_step_takes_are_refused_first(monkeypatch, change):
    monkeypatch.setattr(H, "init", _launched)
    with pytest.raises(ValueError, match="page"):
        PagedEngine(_Model(64), **{"pages": 4, **change})


@pytest.mark.parametrize("hd", [20, 264])
def test_head_sizes_are_refused_first(monkeypatch, hd):
    monkeypatch.setattr(H, "init", _launched)
    with pytest.raises(ValueError, match="head size"):
        PagedEngine(_Model(hd), pages=4)


def _engine(rows):
    e = object.__new__(PagedEngine)
    e.cfg, e.seqs, e.rows, e.max_seq, e.lens, e.stream = _Model(64).cfg, 2, rows, 1 << 20, np.zeros(2, np.int32), None
    e.pools, e.page_size, e.pages = [None], 16, 9
    return e


def test_more_rows_than_a_product_takes_are_refused(monkeypatch):
    e = _engine(1 << 17)
    e._plan = e._workspace = _launched
    with pytest.raises(ValueError, match="65535 rows"):
        e.step({0: [1] * 65536})
    with pytest.raises(ValueError, match="windows"):
        e.score([[1] * 65537])
    assert M.MOST_ROWS == 65535


def test_a_workspace_that_cannot_be_had_leaves_the_lengths(monkeypatch):
    """The allocation comes before the plan."""
    e = _engine(16)
    monkeypatch.setattr(H, "paged_attention_workspace_bytes", lambda *a: 1 << 20)

    def short(need):
        raise MemoryError("workspace")
    e._workspace, e._plan = short, _launched
    with pytest.raises(MemoryError):
        e.step({0: [1, 2, 3]})
    assert not e.lens.any()
