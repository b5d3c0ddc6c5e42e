"""PagedEngine on streams of its own: two of them over one model, their steps in turn, logits read and sampled on their stream."""
import numpy as np
import pytest

from edgeforge_amd.model import Config, DeviceModel, PagedEngine
from oracle.model import OracleModel
from tests import _data as D

pytestmark = pytest.mark.gpu

CFG = Config(D=256, F=512, H=4, KV=2, hd=64, V=512, L=3, max_pos=160)


def test_two_engines_on_two_streams(hip):
    dm = DeviceModel.synthetic(CFG, seed=61)
    om = OracleModel(dm)
    prompts = [[int(v) for v in D.rng(i).integers(0, CFG.V, n)] for i, n in enumerate((21, 40, 3, 90))]
    want = [om.run_once(p, 5, threads=2) for p in prompts]
    engines, rngs, outs = [], [], []
    for e in range(2):
        engines.append(PagedEngine(dm, 40, page_size=8, seqs=2, rows=160, stream=hip.Stream()))
        rngs.append(hip.RngStates([1, 2]))
        outs.append(hip.DeviceArray((2,), np.int32))
    tokens = [{0: prompts[2 * e], 1: prompts[2 * e + 1]} for e in range(2)]
    for step in range(5):
        for e, eng in enumerate(engines):  # both in flight before either is read
            eng.step(tokens[e])
            hip.sample(eng.logits, CFG.V, dict(temperature=0.0), outs[e], batch=2, rng=rngs[e], stream=eng.stream)
        for e, eng in enumerate(engines):
            logits, ids = eng.logits.numpy(eng.stream), outs[e].numpy(eng.stream)
            for r in range(2):
                ref = want[2 * e + r]
                assert np.abs(logits[r] - ref[1][step]).max() / max(1.0, np.abs(ref[1][step]).max()) < 1e-4
                assert ids[r] == int(ref[0][step])
                tokens[e][r] = [int(ref[0][step])]
    for eng in engines:
        eng.release(0, 1)
        assert eng.free_pages() == 40


def test_windows_scored_on_a_stream(hip):
    dm = DeviceModel.synthetic(CFG, seed=5)
    windows = [D.rng(i).integers(0, CFG.V, n).astype(np.int32) for i, n in enumerate((2, 90, 33))]
    a = PagedEngine(dm, 4, page_size=8, seqs=16, rows=128)
    b = PagedEngine(dm, 4, page_size=8, seqs=16, rows=128, stream=hip.Stream())
    for x, y in zip(a.score(windows), b.score(windows)):
        assert np.array_equal(x, y)
