"""A step that fails after its plan: requests, pages and lengths as before it, and the step taken again is right."""
import numpy as np
import pytest

from edgeforge_amd import _lib as L
from edgeforge_amd import hip as H
from edgeforge_amd.model import Config, DeviceModel, PagedEngine
from oracle.model import OracleModel
from tests import _data as D

pytestmark = pytest.mark.gpu

CFG = Config(D=256, F=512, H=4, KV=2, hd=64, V=512, L=3, max_pos=160)


def _state(e):
    return e.lens.tolist(), e._len.numpy().tolist(), e.free_pages(), e._free.numpy()[:e.free_pages()].tolist()


@pytest.mark.parametrize("where", ["attention", "append", "head", "status", "interrupt"])
def test_a_failed_step_is_taken_back(hip, monkeypatch, where):
    print(f"[case] failed step at {where}", flush=True)
    dm = DeviceModel.synthetic(CFG, seed=61)
    om = OracleModel(dm)
    prompts = [[int(v) for v in D.rng(i).integers(0, CFG.V, n)] for i, n in enumerate((21, 40))]
    want = [om.run_once(p, 3, threads=2) for p in prompts]
    eng = PagedEngine(dm, 12, page_size=8, seqs=3, rows=64)
    eng.step({0: prompts[0], 2: prompts[1][:17]})
    before = _state(eng)
    held = [eng._table.numpy()[r, :-(-n // 8)].tolist() for r, n in enumerate(before[0])]
    calls = {"n": 0}

    def failing(f, at, error):
        def g(*a, **k):
            calls["n"] += 1
            if calls["n"] == at:
                raise error
            return f(*a, **k)
        return g

    step = {0: [int(want[0][0][0])], 2: prompts[1][17:]}
    with monkeypatch.context() as m:
        if where == "attention":
            m.setattr(H, "paged_attention", failing(H.paged_attention, 2, L.HipError(L.EINVAL, "refused")))
        elif where == "append":
            m.setattr(H, "rope_append", failing(H.rope_append, 1, L.HipError(L.EINVAL, "refused")))
        elif where == "head":
            m.setattr(eng, "_head_of", failing(eng._head_of, 1, MemoryError("logits")))
        elif where == "status":
            m.setattr(eng._status, "numpy", failing(eng._status.numpy, 1, L.HipError(L.EINVAL, "copy")))
        else:
            m.setattr(H, "paged_attention", failing(H.paged_attention, 3, KeyboardInterrupt()))
        with pytest.raises((L.HipError, MemoryError, KeyboardInterrupt)):
            eng.step(step)
    assert _state(eng) == before
    assert [eng._table.numpy()[r, :-(-n // 8)].tolist() for r, n in enumerate(before[0])] == held
    assert eng.step(step) == [0, 2]
    logits = eng.logits.numpy()
    for row, ref in ((0, want[0][1][1]), (1, want[1][1][0])):
        assert np.abs(logits[row] - ref).max() / max(1.0, np.abs(ref).max()) < 1e-4
    eng.release(0, 2)
    assert eng.free_pages() == 12
