"""Requests of different lengths served together (model.PagedEngine): the plan, RoPE into pages, attention over pages
and the packed products in a run, as a server uses them, against the CPU oracle's Transformer, one request at a time."""
import numpy as np
import pytest

from edgeforge_amd import _lib as L
from edgeforge_amd.model import Config, DeviceModel, Engine, PagedEngine, PagesShort
from oracle.model import OracleModel
from tests import _data as D

pytestmark = pytest.mark.gpu

SMALL = Config(D=256, F=512, H=4, KV=2, hd=64, V=512, L=3, max_pos=160)
WIDE = Config(D=256, F=512, H=2, KV=1, hd=128, V=300, L=2, max_pos=96)
ODD = Config(D=96, F=160, H=4, KV=4, hd=24, V=200, L=2, max_pos=64)


def _model(cfg):
    dm = DeviceModel.synthetic(cfg, seed=61, q8={(0, "wk"), (1, "w_down")})
    return dm, OracleModel(dm)


def _err(a, b):
    return float(np.abs(a - b).max() / max(1.0, np.abs(b).max()))


class Request:
    def __init__(self, om, prompt, n):
        self.prompt, self.n, self.fed, self.got = [int(v) for v in prompt], n, 0, []
        self.want, self.logits, _, _ = om.run_once(self.prompt, n, threads=2)

    def next(self, chunk):
        """The ids of the next step, and whether its logits pick a token."""
        if self.fed < len(self.prompt):
            part = self.prompt[self.fed:self.fed + chunk]
            self.fed += len(part)
            return part, self.fed == len(self.prompt)
        return [self.got[-1]], True


def _serve(eng, requests, chunk, arrive, V, tol):
    """Requests arrive over the steps, wait for a free slot, and leave; every pick's logits against the oracle's."""
    waiting, running, step, worst = list(enumerate(requests)), {}, 0, 0.0
    while waiting or running:
        while waiting and waiting[0][0] * arrive <= step and len(running) < eng.seqs:
            slot = min(set(range(eng.seqs)) - set(running))
            running[slot] = waiting.pop(0)[1]
        tokens, picks = {}, {}
        for slot, r in running.items():
            tokens[slot], picks[slot] = r.next(chunk)
        order = eng.step(tokens)
        assert order == sorted(tokens)
        logits = eng.logits.numpy()
        done = []
        for row, slot in enumerate(order):
            r = running[slot]
            if not picks[slot]:
                continue
            worst = max(worst, _err(logits[row], r.logits[len(r.got)]))
            assert worst < tol, (step, slot, worst)
            r.got.append(int(r.want[len(r.got)]))  # the oracle's path, so that a near tie cannot part them
            if tol <= 1e-4:
                assert int(np.argmax(logits[row])) == r.got[-1], (step, slot)
            if len(r.got) == r.n:
                done.append(slot)
        if done:
            eng.release(*done)
            for slot in done:
                del running[slot]
        step += 1
    return worst


@pytest.mark.parametrize("cfg", [SMALL, WIDE, ODD], ids=["small", "wide", "odd"])
@pytest.mark.parametrize("page,chunk", [(1, 7), (8, 100), (16, 5), (64, 30)])
def test_requests_served_together_match_the_oracle(hip, cfg, page, chunk):
    dm, om = _model(cfg)
    print(f"[case] served together hd={cfg.hd} page={page} chunk={chunk}", flush=True)
    g = D.rng(page)
    reqs = [Request(om, g.integers(0, cfg.V, int(n)), int(m)) for n, m in zip([1, 33, 7, 50, 2, 19, 40], [9, 4, 12, 3, 8, 6, 5])]
    pages = 4 * -(-60 // page)
    eng = PagedEngine(dm, pages, page_size=page, seqs=3, rows=256)
    worst = _serve(eng, reqs, chunk, arrive=2, V=cfg.V, tol=1e-4)
    print(f"worst logits error {worst:.2e}", flush=True)
    assert eng.free_pages() == pages and not eng.lens.any()


# Keys and values are off by half a step of their type at most, relative to their own size.  The attention's output, a
# weighted mean of values with weights whose exponents the keys' roundings shift by as much relative to the
# scores' size, is then off by at most two to three half steps of its size; it is added to the residual stream layer by
# layer (three of them), and the final norm and head are linear in what is left: 3 layers * 3 half steps, twice that for the
# feed-forward blocks' share of it.
@pytest.mark.parametrize("kv_type,half", [(L.F16, 2.0 ** -11), (L.BF16, 2.0 ** -8)], ids=["f16", "bf16"])
def test_pages_of_16_bits(hip, kv_type, half):
    dm, om = _model(SMALL)
    g = D.rng(9)
    reqs = [Request(om, g.integers(0, SMALL.V, int(n)), 6) for n in (3, 60, 21, 44)]
    eng = PagedEngine(dm, 40, page_size=16, seqs=4, rows=200, kv_type=kv_type)
    worst = _serve(eng, reqs, 64, arrive=1, V=SMALL.V, tol=18 * half)
    print(f"worst logits error {worst:.2e}", flush=True)


def test_pages_run_short_and_come_back(hip):
    dm, om = _model(SMALL)
    g = D.rng(3)
    eng = PagedEngine(dm, 6, page_size=8, seqs=4, rows=64)
    a, b = Request(om, g.integers(0, SMALL.V, 20), 4), Request(om, g.integers(0, SMALL.V, 30), 3)
    eng.step({0: a.prompt})
    before = (eng.lens.copy(), eng.free_pages(), eng._table.numpy(), eng._free.numpy())
    with pytest.raises(PagesShort, match="1 pages"):
        eng.step({1: b.prompt})
    after = (eng.lens.copy(), eng.free_pages(), eng._table.numpy(), eng._free.numpy())
    assert all(np.array_equal(x, y) for x, y in zip(before, after))
    eng.step({0: [int(a.want[0])]})  # the other request goes on
    assert _err(eng.logits.numpy()[0], a.logits[1]) < 1e-4
    eng.release(0)
    assert eng.free_pages() == 6
    eng.step({1: b.prompt})
    assert _err(eng.logits.numpy()[0], b.logits[0]) < 1e-4
    with pytest.raises(ValueError, match="slot"):
        eng.step({4: [1]})
    with pytest.raises(ValueError, match="rows"):
        eng.step({2: [1] * 65})
    with pytest.raises(ValueError, match="max_seq"):
        eng.step({2: [1] * 161})
    assert eng.step({}) == []


def test_sampling_from_a_step(hip):
    """hip.sample on the step's logits, per request its own generator, as the engine samples."""
    dm, om = _model(SMALL)
    cfg = dict(temperature=0.8, top_k=40, top_p=0.95, repetition_penalty=1.0)
    prompts = [[int(v) for v in D.rng(i).integers(0, SMALL.V, n)] for i, n in enumerate((5, 17, 9))]
    want = []
    for i, p in enumerate(prompts):
        e = Engine(dm, max_seq=64)
        want.append(e.generate([p], 6, sampler=cfg, rng=hip.RngStates([11 + i]))[0][0].tolist())
        e.close()
    eng = PagedEngine(dm, 30, page_size=8, seqs=3, rows=64)
    rng, out = hip.RngStates([11, 12, 13]), hip.DeviceArray((3,), np.int32)
    tokens, got = {i: p for i, p in enumerate(prompts)}, [[], [], []]
    for _ in range(6):
        eng.step(tokens)
        hip.sample(eng.logits, SMALL.V, cfg, out, batch=3, rng=rng)
        ids = out.numpy()
        for i in range(3):
            got[i].append(int(ids[i]))
            tokens[i] = [int(ids[i])]
    assert got == want


@pytest.mark.parametrize("rows", [64, 1300])
def test_windows_scored_together(hip, rows):
    """PagedEngine.score of windows of different lengths == Engine.score of each (2e-4, as the quality harness)."""
    cfg = Config(D=256, F=512, H=4, KV=2, hd=64, V=512, L=2, max_pos=700)
    dm = DeviceModel.synthetic(cfg, seed=5)
    lens = [2, 40, 9, 65, 33] if rows == 64 else [600, 2, 401, 77, 300, 650]
    windows = [D.rng(i).integers(0, cfg.V, n).astype(np.int32) for i, n in enumerate(lens)]
    eng = PagedEngine(dm, 4, page_size=8, seqs=16, rows=rows, max_seq=max(lens))
    got = eng.score(windows)
    for w, g in zip(windows, got):
        one = Engine(dm, max_seq=w.size)
        want = one.score(w)
        one.close()
        assert g.shape == want.shape and np.abs(g - want).max() < 2e-4, np.abs(g - want).max()


def test_model_from_a_file(hip, tmp_path):
    """The same over a model loaded from an .efq file."""
    from edgeforge_amd.qfile import EfqModel
    from oracle.efq import write_efq
    from oracle.model import HostModel
    cfg = Config(D=256, F=512, H=4, KV=2, hd=64, V=500, L=2, max_pos=64)
    hm = HostModel(cfg, seed=71)
    path = str(tmp_path / "m.efq")
    write_efq(path, cfg, hm.efq_tensors())
    m = EfqModel.load_efq(path)
    om = OracleModel(hm)
    r = [Request(om, D.rng(i).integers(0, cfg.V, n), 4) for i, n in enumerate((5, 20))]
    eng = PagedEngine(m, 12, page_size=8, seqs=2, rows=64)
    _serve(eng, r, 16, 1, cfg.V, 1e-4)
    del eng
    m.free()
