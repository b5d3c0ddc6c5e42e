"""Paged serving on the GPU: the plan against a plain simulation, RoPE and the store into pages, attention over
pages and over packed prompts against a float64 softmax.

Everything the kernels must not read is NaN: pages nobody owns, positions past a request's last, later rows of
a chunk are infinite, and rows behind the last request hold a mark that has to stay.

Tolerances.  Relative 2-norm per (row, head) against float64, in units of u = 2^-24 (FP32's half step).  With N(0, 1)
queries and keys the terms of a score, q_i k_i scale, add up at random: a rounding of each partial sum (hd of
them, standard deviation of the sums at most 1) gives at most sqrt(hd) / 2 <= 8 u, operand splits that keep 22 bits
or more and their dropped products another 4 u.  The exponent's argument (within about 10 of the maximum, where the
weight is) is rounded at its own size, up to 8 u where p is small and below 2 u where it is not; exp2 is off by
2 u.  Errors of the p_j are independent, so an output of many of them averages them; one that a single position
dominates has that position's error cancel against the sum's.  The sum over positions adds at most 64 chunk
sums at random (8 u / 2).  Together below 16 u where the softmax spreads, and below 32 u in the worst single row.
Stored keys and values: one rounding, half a step of their type, of the FP32 result, which is itself off by at most
2 u of the larger of its two products."""
import numpy as np
import pytest
import torch

from edgeforge_amd import _lib as L
from tests import _data as D

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
WORST, TYPICAL = 32 * U, 16 * U
NP = {L.F32: np.float32, L.F16: np.float16}
TORCH = {L.F32: torch.float32, L.F16: torch.float16, L.BF16: torch.bfloat16}
HALF_STEP = {t: torch.finfo(d).eps / 2 for t, d in TORCH.items()}
TYPES = [L.F32, L.F16, L.BF16]
TYPE_IDS = ["f32", "f16", "bf16"]


class Dev:
    """A torch tensor as the hip module takes it."""

    def __init__(self, t):
        self.t = t.contiguous().cuda()
        self.ptr, self.nbytes = self.t.data_ptr(), self.t.numel() * self.t.element_size()

    def np(self):
        return self.t.cpu().numpy()


def i32(v):
    return Dev(torch.tensor(np.asarray(v, np.int32)))


# ---- the plan --------------------------------------------------------------------------------------------
def simulate(cached, new, page, n_pages, table, free, n_free, max_rows):
    """The documented plan, request by request."""
    table, free = table.copy(), free.copy()
    n, ld = table.shape
    held = [-(-max(int(c), 0) // page) for c in cached]
    bad = [c < 0 or c + max(x, 0) > ld * page for c, x in zip(cached.astype(int), new.astype(int))]
    give = [[p for p in table[r, :held[r]] if 0 <= p < n_pages] if new[r] < 0 and not bad[r] else [] for r in range(n)]
    take = [0 if bad[r] or new[r] < 0 else -(-int(cached[r] + new[r]) // page) - held[r] for r in range(n)]
    rows = [0 if bad[r] else max(int(new[r]), 0) for r in range(n)]
    n1 = n_free + sum(map(len, give))
    status = [max(0, sum(take) - n1), sum(bad), max(0, sum(rows) - max_rows), 0]
    if not 0 <= n_free <= n_pages or n1 > n_pages:
        status[0], status[3] = 0, 1
    pos, slot = np.zeros(max_rows, np.int32), np.full(max_rows, -1, np.int64)
    if any(status):
        return table, free, n_free, cached.copy(), np.zeros(n + 1, np.int32), pos, slot, status
    top = n_free
    for g in give:
        free[top:top + len(g)] = g
        top += len(g)
    for r in range(n):
        for j in range(take[r]):
            top -= 1
            table[r, held[r] + j] = free[top]
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    kv = np.where(new < 0, 0, cached + np.maximum(new, 0)).astype(np.int32)
    for r in range(n):
        for i in range(rows[r]):
            p = int(cached[r]) + i
            pos[start[r] + i] = p
            e = table[r, p // page]
            slot[start[r] + i] = int(e) * page + p % page if 0 <= e < n_pages else -1
    return table, free, top, kv, start, pos, slot, status


def plan_state(seed, n, page, ctx, most, spare, ld_extra=1):
    """Random lengths, a table of scattered pages and a stack of the free ones."""
    g = D.rng(seed)
    cached = g.integers(0, ctx + 1, n).astype(np.int32)
    new = g.integers(0, most + 1, n).astype(np.int32)
    new[g.random(n) < 0.15] = -1
    held = -(-cached // page)
    need = np.where(new < 0, 0, -(-(cached + np.maximum(new, 0)) // page) - held)
    n_pages = int(held.sum() + max(need.sum(), 1) + spare)
    ids = g.permutation(n_pages).astype(np.int32)
    ld = int((held + need).max()) + ld_extra
    table = np.full((n, ld), -7, np.int32)
    at = 0
    for r in range(n):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    free = np.full(n_pages, -9, np.int32)
    free[:n_pages - at] = ids[at:]
    return cached, new, n_pages, table, free, n_pages - at


def run_plan(hip, cached, new, page, n_pages, table, free, n_free, max_rows, in_place=False, stream=None):
    d = dict(cached=i32(cached), new=i32(new), table=i32(table), free=i32(free), n_free=i32([n_free]))
    out = d["n_free"] if in_place else i32([-1])
    kv = d["cached"] if in_place else i32(np.full(len(cached), -1))
    start, pos, slot, status = i32(np.full(len(cached) + 1, -1)), i32(np.full(max_rows, -1)), Dev(torch.full((max_rows,), -5)), i32([9] * 4)
    torch.cuda.synchronize()
    hip.page_plan(d["cached"], d["new"], len(cached), page, n_pages, d["table"], table.shape[1], d["free"], d["n_free"], out, kv, start,
                  pos, slot, max_rows, status, stream=stream)
    hip.sync(stream)
    return (d["table"].np(), d["free"].np(), int(out.np()[0]), kv.np(), start.np(), pos.np(), slot.np(), status.np().tolist())


def same_plan(got, want):
    for name, g, w in zip(("table", "free", "n_free", "kv_len", "row_start", "pos", "slot", "status"), got, want):
        assert np.array_equal(np.asarray(g), np.asarray(w)), (name, g, w)


# requests on both sides of one pass of the workgroup (1024) and of what it keeps in LDS (4096); rows on both sides
# of what it fills by itself (4096); pages given or taken on both sides of what it keeps (4096)
@pytest.mark.parametrize("n,page,ctx,most", [(1, 16, 0, 1), (1, 1, 5, 3), (64, 16, 900, 1), (63, 8, 100, 200), (1023, 32, 300, 2),
                                             (1024, 16, 64, 1), (1025, 16, 64, 1), (2500, 4, 30, 9), (4096, 16, 20, 1), (4097, 16, 20, 2),
                                             (700, 32, 4000, 30), (3, 1024, 5000, 3000),
                                             (200, 1, 300, 2), (200, 1, 4, 60), (900, 2, 90, 40)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(hip, n, page, ctx, most, in_place):
    print(f"[case] plan n={n} page={page} ctx={ctx} most={most} in_place={in_place}", flush=True)
    cached, new, n_pages, table, free, n_free = plan_state(n + page, n, page, ctx, most, spare=3)
    rows = int(np.maximum(new, 0).sum())
    for max_rows in {max(rows, 1), rows + 77}:
        want = simulate(cached, new, page, n_pages, table, free, n_free, max_rows)
        assert want[-1] == [0, 0, 0, 0]
        same_plan(run_plan(hip, cached, new, page, n_pages, table, free, n_free, max_rows, in_place), want)


@pytest.mark.parametrize("n", [9, 1500])
@pytest.mark.parametrize("fault", ["missing", "negative", "wide", "rows", "free", "free_negative", "given"])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_that_does_not_fit_changes_nothing(hip, n, fault, in_place):
    print(f"[case] plan n={n} fault={fault} in_place={in_place}", flush=True)
    page = 8
    cached, new, n_pages, table, free, n_free = plan_state(77, n, page, 60, 20, spare=0)
    max_rows = int(np.maximum(new, 0).sum()) + 5
    if fault == "missing":
        new[0], cached[0], n_free = 12, 0, 0
        new[new < 0] = 0
        free[:] = -1
    elif fault == "negative":
        cached[4], cached[7] = -1, -2 ** 31
    elif fault == "wide":
        new[2] = 2 ** 31 - 1
    elif fault == "rows":
        max_rows -= 9
    elif fault == "free":
        n_free = n_pages + 1
    elif fault == "free_negative":
        n_free = -3
    else:
        new[:], n_free = -1, n_pages  # more given back than there are pages
        cached[0] = 9
    want = simulate(cached, new, page, n_pages, table, free, n_free, max_rows)
    assert any(want[-1]) and want[4].max() == 0 and want[6].max() == -1
    same_plan(run_plan(hip, cached, new, page, n_pages, table, free, n_free, max_rows, in_place), want)


def test_plan_keeps_lost_pages_out(hip):
    """Table entries that are no page: not given back, and no slot."""
    cached, new = np.array([40, 33, 20], np.int32), np.array([-1, 9, 3], np.int32)
    table = np.array([[3, -1, 99, 5, 1, 0], [2, 4, 6, 7, -5, 0], [8, 2 ** 31 - 1, -1, 0, 0, 0]], np.int32)
    free, page, n_pages = np.array([10, 11, 400] + [-1] * 9, np.int32), 8, 12
    want = simulate(cached, new, page, n_pages, table, free, 3, 14)
    assert want[-1] == [0, 0, 0, 0] and want[2] == 5
    same_plan(run_plan(hip, cached, new, page, n_pages, table, free, 3, 14), want)


def test_many_steps_hold_every_page_once(hip):
    """Requests that grow, end and start again: pages are never held twice and never lost, step after step."""
    g, n, page, n_pages, ld = D.rng(5), 37, 4, 400, 24
    cached, table, free, n_free = np.zeros(n, np.int32), np.full((n, ld), -1, np.int32), np.arange(n_pages, dtype=np.int32), n_pages
    for step in range(40):
        new = g.integers(0, 7, n).astype(np.int32)
        new[g.random(n) < 0.1] = -1
        new = np.where(cached + new > ld * page, -1, new).astype(np.int32)
        want = simulate(cached, new, page, n_pages, table, free, n_free, 300)
        got = run_plan(hip, cached, new, page, n_pages, table, free, n_free, 300, in_place=step % 2 == 0)
        same_plan(got, want)
        table, free, n_free, cached = got[0], got[1], got[2], got[3]
        held = [p for r in range(n) for p in table[r, :-(-int(cached[r]) // page)]]
        assert sorted(held + free[:n_free].tolist()) == list(range(n_pages)), step


# ---- RoPE and append ---------------------------------------------------------------------------------------
def test_rope_tables_are_the_engines(hip):
    import oracle as O  # noqa: F401
    cos, sin = hip.rope_tables(10000.0, 64, 50)
    inv = np.array([np.float32(1) / np.float32(np.float32(10000.0) ** np.float32(np.float32(2 * i) / np.float32(64))) for i in range(32)])
    ang = (np.arange(50, dtype=np.float32)[:, None] * inv).astype(np.float64)
    # angles up to 49, off by up to two roundings (pow, division): 49 * 2 * 2^-24, and a rounding of the result
    assert np.abs(cos.numpy() - np.cos(ang)).max() < 50 * 2 * U + U
    assert np.abs(sin.numpy() - np.sin(ang)).max() < 50 * 2 * U + U


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("H,KV,hd,page,rows", [(32, 4, 64, 16, 7), (5, 1, 8, 1, 33), (3, 3, 80, 4, 130), (8, 2, 256, 1024, 3), (1, 1, 128, 64, 1)])
@pytest.mark.parametrize("where", ["fused", "in_place", "apart"])
def test_rope_append(hip, qtype, H, KV, hd, page, rows, where):
    print(f"[case] append {TYPE_IDS[TYPES.index(qtype)]} H={H} KV={KV} hd={hd} page={page} rows={rows} {where}", flush=True)
    g = torch.Generator().manual_seed(rows + hd)
    nq, nk, n_pos = H * hd, KV * hd, 100
    n_pages = -(-rows // page) + 2
    ld = nq + 2 * nk + (4 if where == "apart" else 0)
    x = torch.randn(rows, ld, generator=g)
    ang = torch.rand(n_pos, hd // 2, generator=g, dtype=torch.float64) * 6
    cos, sin = ang.cos().float(), ang.sin().float()
    pos = torch.randint(0, n_pos, (rows,), generator=g, dtype=torch.int32)
    slot = torch.randperm(n_pages * page, generator=g)[:rows].to(torch.int64)
    if rows > 5:  # rows without a slot, slots outside the pool, positions outside the tables
        slot[1], slot[2], slot[3] = -1, n_pages * page, 2 ** 40
        pos[4], pos[5] = -1, n_pos
    pad = 16
    stride = KV * page * hd + pad
    mark = 7.0
    kp, vp = (Dev(torch.full((n_pages, stride), mark, dtype=TORCH[qtype])) for _ in range(2))
    dx, dpos, dslot, dc, ds = Dev(x), Dev(pos), Dev(slot), Dev(cos), Dev(sin)
    pool = hip.PagePool(n_pages, page, KV, hd, qtype, k=kp, v=vp, page_stride=stride)
    qo = dx.ptr if where == "in_place" else Dev(torch.full((rows, nq + 8), mark))
    ko = {"fused": None, "in_place": dx.ptr + 4 * nq, "apart": Dev(torch.full((rows, nk), mark))}[where]
    torch.cuda.synchronize()
    hip.rope_append(dx, ld, qo, ld if where == "in_place" else nq + 8, H, dx.ptr + 4 * nq, ld, dx.ptr + 4 * (nq + nk), ld, rows, dpos, dc, ds,
                    n_pos, dslot, pool, k_out=ko, ldko=ld if where == "in_place" else nk)
    hip.sync()
    known = ((pos >= 0) & (pos < n_pos)).numpy()
    c64, s64 = (t[pos.clamp(0, n_pos - 1).long()].double().numpy()[:, None] for t in (cos, sin))

    def turned(part, heads):
        p = part.double().numpy().reshape(rows, heads, hd)
        a, b = p[..., :hd // 2], p[..., hd // 2:]
        size = np.concatenate([np.abs(a * c64) + np.abs(b * s64), np.abs(b * c64) + np.abs(a * s64)], -1)
        return np.concatenate([a * c64 - b * s64, b * c64 + a * s64], -1), size

    q64, qs = turned(x[:, :nq], H)
    k64, ks = turned(x[:, nq:nq + nk], KV)
    v64 = x[:, nq + nk:nq + 2 * nk].double().numpy().reshape(rows, KV, hd)
    got_q = (dx.np()[:, :nq] if where == "in_place" else qo.np()[:, :nq]).reshape(rows, H, hd)
    assert (np.abs(got_q - q64) <= 2 * U * qs)[known].all() and np.isnan(got_q[~known]).all()
    if where != "in_place":
        assert (qo.np()[:, nq:] == mark).all()
    if where != "fused":
        got_k = (dx.np()[:, nq:nq + nk] if where == "in_place" else ko.np()).reshape(rows, KV, hd)
        assert (np.abs(got_k - k64) <= 2 * U * ks)[known].all() and np.isnan(got_k[~known]).all()
    for dev, val, size in ((kp, k64, ks), (vp, v64, 0 * v64)):
        flat = dev.t.float().cpu().numpy().astype(np.float64)
        assert (flat[:, KV * page * hd:] == mark).all()
        pages = flat[:, :KV * page * hd].reshape(n_pages, KV, page, hd).transpose(0, 2, 1, 3).reshape(n_pages * page, KV, hd)
        stored = np.zeros(n_pages * page, bool)
        for r in range(rows):
            at = int(slot[r])
            if known[r] and 0 <= at < n_pages * page:
                stored[at] = True
                tiny = 2.0 ** -25 if qtype == L.F16 else 0.0  # half the smallest step of FP16
                tol = np.abs(val[r]) * HALF_STEP[qtype] + 2 * U * size[r] * (1 + HALF_STEP[qtype]) + tiny
                assert (np.abs(pages[at] - val[r]) <= tol * (1 + 2.0 ** -20)).all(), (r, at)
        assert (pages[~stored] == mark).all()


# ---- attention -----------------------------------------------------------------------------------------
def softmax_ref(q, k, v, scale):
    """q [H][hd], k / v [n][KV][hd] in float64."""
    H, hd = q.shape
    KV = k.shape[1]
    out = np.zeros((H, hd))
    if not len(k):
        return out
    for h in range(H):
        g = h // (H // KV)
        s = k[:, g] @ q[h] * scale
        p = np.exp(s - s.max())
        out[h] = p @ v[:, g] / p.sum()
    return out


class Paged:
    """Requests over pages: everything they do not own is NaN."""

    def __init__(self, hip, seed, qtype, H, KV, hd, page, new, kv, pad=0, scale=None, spread=1.0):
        g = D.rng(seed)
        self.hip, self.qtype, self.H, self.KV, self.hd, self.page = hip, qtype, H, KV, hd, page
        self.new, self.kv, self.scale = list(new), list(kv), scale or 1.0 / np.sqrt(hd)
        held = [-(-n // page) for n in kv]
        self.n_pages, self.ld = sum(held) + 3, max(max(held), 1) + 1
        ids = g.permutation(self.n_pages)
        self.table = np.full((len(kv), self.ld), -1, np.int64)
        stride = KV * page * hd + pad
        kp, vp = (torch.full((self.n_pages, stride), float("nan"), dtype=TORCH[qtype]) for _ in range(2))
        self.k, self.v = [], []
        at = 0
        for r, n in enumerate(kv):
            self.table[r, :held[r]] = ids[at:at + held[r]]
            at += held[r]
            k = torch.from_numpy(g.standard_normal((n, KV, hd), dtype=np.float32) * np.float32(spread)).to(TORCH[qtype])
            v = torch.from_numpy(g.standard_normal((n, KV, hd), dtype=np.float32)).to(TORCH[qtype])
            for t, pool in ((k, kp), (v, vp)):
                view = pool[:, :KV * page * hd].view(self.n_pages, KV, page, hd)
                for b in range(held[r]):
                    part = t[b * page:(b + 1) * page]
                    view[self.table[r, b], :, :len(part)] = part.permute(1, 0, 2)
            self.k.append(k.double().numpy())
            self.v.append(v.double().numpy())
        self.kp, self.vp = Dev(kp), Dev(vp)
        self.pool = hip.PagePool(self.n_pages, page, KV, hd, qtype, k=self.kp, v=self.vp, page_stride=stride)
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.start[-1])
        self.q = g.standard_normal((self.rows, H, hd), dtype=np.float32)

    def place(self, r, j):
        """(page, offset) of position j of request r."""
        return self.table[r, j // self.page], j % self.page

    def put(self, which, r, j, g, d, value):
        pool, host = (self.kp, self.k) if which == "k" else (self.vp, self.v)
        pg, off = self.place(r, j)
        at = (pg, (g * self.page + off) * self.hd + d)
        pool.t[at] = value
        host[r][j, g, d] = pool.t[at].item()  # as the pool's type holds it

    def run(self, behind=3, max_new=None, max_kv=None, pad=4, stream=None, table=None):
        """Outputs [rows][H][hd]; `behind` more rows have to stay as they were."""
        H, hd = self.H, self.hd
        ldq = H * hd + pad
        q = np.full((self.rows + behind, ldq), np.nan, np.float32)
        q[:self.rows, :H * hd] = self.q.reshape(self.rows, -1)
        dq, out = Dev(torch.from_numpy(q)), Dev(torch.full((self.rows + behind, ldq), 5.0))
        dt, ds, dk = i32(self.table if table is None else table), i32(self.start), i32(self.kv)
        args = (len(self.kv), self.rows + behind, max_new or max(1, max(self.new)), max_kv or max(1, max(self.kv)))
        need = self.hip.paged_attention_workspace_bytes(H, self.pool, *args)
        ws = Dev(torch.full((max(need, 16),), 0xFF, dtype=torch.uint8))  # NaN
        self.dev = (dq, out, dt, ds, dk, ws, args, ldq)
        torch.cuda.synchronize()
        self.launch(stream)
        self.hip.sync(stream)
        return self.fetch()

    def launch(self, stream=None):
        dq, out, dt, ds, dk, ws, args, ldq = self.dev
        self.hip.paged_attention(dq, ldq, out, ldq, self.H, self.pool, dt, self.ld, ds, dk, *args, float(self.scale), ws=ws, stream=stream)

    def fetch(self):
        o = self.dev[1].np()
        assert (o[self.rows:] == 5.0).all() and (o[:, self.H * self.hd:] == 5.0).all(), "rows or columns outside the call were written"
        return o[:self.rows, :self.H * self.hd].reshape(self.rows, self.H, self.hd)

    def want(self, lost=()):
        """lost: (request, page index) pairs that are no page."""
        out = np.zeros((self.rows, self.H, self.hd))
        for r, n in enumerate(self.new):
            real = np.array([(r, j // self.page) not in lost for j in range(self.kv[r])], bool)
            for i in range(n):
                seen = max(0, self.kv[r] - n + i + 1)
                keep = real[:seen]
                row = self.start[r] + i
                out[row] = softmax_ref(self.q[row].astype(np.float64), self.k[r][:seen][keep], self.v[r][:seen][keep], self.scale)
        return out


def check(got, want, what="", worst=WORST):
    """Relative 2-norms per (row, head); rows that see nothing are zero."""
    got, want = got.astype(np.float64), np.asarray(want)
    norm = np.linalg.norm(want, axis=-1)
    err = np.linalg.norm(got - want, axis=-1)
    assert (got[norm == 0] == 0).all(), what
    rel = (err / np.where(norm == 0, 1, norm))[norm > 0]
    if rel.size:
        print(f"{what} relative error: worst {rel.max() / U:.1f} u, rms {np.sqrt((rel ** 2).mean()) / U:.1f} u", flush=True)
        assert rel.max() < worst and np.sqrt((rel ** 2).mean()) < TYPICAL, what


SHAPES = [(32, 4, 64), (8, 2, 128), (4, 4, 64), (6, 1, 80), (2, 1, 256), (20, 1, 8), (7, 1, 96), (70, 2, 64)]


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("H,KV,hd", SHAPES)
@pytest.mark.parametrize("page", [1, 16, 128])
def test_decode(hip, qtype, H, KV, hd, page):
    """One new token each, contexts of one position to several splits, around tiles and pages."""
    kv = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 700]
    print(f"[case] decode {qtype} H={H} KV={KV} hd={hd} page={page}", flush=True)
    p = Paged(hip, H + hd + page, qtype, H, KV, hd, page, [1] * len(kv), kv)
    check(p.run(), p.want(), f"decode {qtype} {H}/{KV}/{hd} page {page}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("H,KV,hd", SHAPES)
@pytest.mark.parametrize("page", [8, 64])
def test_chunks(hip, qtype, H, KV, hd, page):
    """Chunks of every size in one call: whole prompts, continuations, single tokens, none at all."""
    new = [1, 0, 5, 17, 70, 1, 3, 130, 2, 33]
    kv = [1, 0, 5, 40, 71, 300, 3, 131, 64, 290]
    print(f"[case] chunks {qtype} H={H} KV={KV} hd={hd} page={page}", flush=True)
    p = Paged(hip, H * hd + page, qtype, H, KV, hd, page, new, kv)
    check(p.run(), p.want(), f"chunks {qtype} {H}/{KV}/{hd} page {page}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("H,KV,hd", [(32, 4, 64), (8, 8, 128), (4, 1, 96)])
def test_few_tokens(hip, qtype, n, H, KV, hd):
    """As many new tokens as a step that verifies guesses has."""
    kv = [n, n + 1, 50, 333, 1200]
    print(f"[case] few {qtype} n={n} H={H} KV={KV} hd={hd}", flush=True)
    p = Paged(hip, n * hd, qtype, H, KV, hd, 16, [n] * len(kv), kv)
    check(p.run(), p.want(), f"few {qtype} {n} {H}/{KV}/{hd}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new,kv", [([1], [5003]), ([1, 1, 1], [3000, 1, 4999]), ([40], [2600]), ([200, 1], [2100, 3001])])
def test_long(hip, qtype, new, kv):
    print(f"[case] long {qtype} {new} {kv}", flush=True)
    p = Paged(hip, 31, qtype, 8, 2, 64, 32, new, kv)
    check(p.run(), p.want(), f"long {qtype} {new} {kv}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("bounds", [(1, 1), (1, 100000), (1000, 100000), (1000, 1)])
def test_bounds_are_only_bounds(hip, qtype, bounds):
    """max_new and max_kv above and below the lengths: the same results."""
    p = Paged(hip, 8, qtype, 8, 2, 64, 16, [1, 9, 40, 0, 1], [900, 9, 310, 0, 33])
    check(p.run(max_new=bounds[0], max_kv=bounds[1]), p.want(), f"bounds {bounds}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new", [[1, 1, 1, 1, 1], [3, 1, 2, 1, 4], [60, 1, 90, 1, 30]])
def test_lost_pages(hip, qtype, new):
    """Page numbers outside the pool, of every kind: their positions take no part; a row with none left is zero."""
    kv = [200, 16, 130, 5, 61]
    p = Paged(hip, 12, qtype, 8, 2, 64, 16, new, kv)
    lost = {(0, 0), (0, 1), (0, 7), (0, 12), (1, 0), (2, 8), (3, 0), (4, 1)}
    table = p.table.copy()
    for i, (r, b) in enumerate(sorted(lost)):
        table[r, b] = [-1, p.n_pages, 2 ** 31 - 1, -2 ** 31, p.n_pages + 5][i % 5]
    check(p.run(table=table), p.want(lost), f"lost pages {new}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new,kv", [([4, 3], [2, 0]), ([70, 40], [30, 0]), ([1, 1], [0, 7]), ([9], [1])])
def test_rows_that_see_nothing(hip, qtype, new, kv):
    """More new rows than positions: the first rows see nothing and get zeros."""
    p = Paged(hip, 21, qtype, 8, 2, 64, 16, new, kv)
    check(p.run(), p.want(), f"empty rows {new} {kv}")


def test_lengths_past_the_table_are_cut(hip):
    """A kv_len that the table cannot hold reads no further than the table."""
    p = Paged(hip, 22, L.F16, 8, 2, 64, 16, [1, 1], [64, 40])
    want = p.want()
    p.ld = 4
    p.table = p.table[:, :4]
    p.kv[0] = 10 ** 9
    got = p.run()
    assert np.isfinite(got).all()
    check(got, want, "cut")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new,kv", [([1, 1], [300, 77]), ([4, 2], [300, 77]), ([100, 80], [300, 80])])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("which", ["k", "v"])
def test_infinities_stay_with_the_rows_that_see_them(hip, qtype, new, kv, value, which):
    p = Paged(hip, 40, qtype, 8, 2, 64, 16, new, kv)
    spots = [(0, 299, 0, 5), (0, 250, 1, 63), (1, kv[1] - 1, 1, 0)]
    for r, j, g, d in spots:
        p.put(which, r, j, g, d, value)
    got, G = p.run(), p.H // p.KV
    with np.errstate(all="ignore"):
        want = p.want()
    touched = np.zeros(got.shape, bool)
    for r, j, g, d in spots:
        for i in range(new[r]):
            if kv[r] - new[r] + i >= j:
                heads = touched[p.start[r] + i, g * G:g * G + G]
                if which == "v":
                    heads[:, d] = True
                else:
                    heads[:] = True
    clean = ~touched.any(-1)
    assert np.isfinite(got[clean]).all()
    check(np.where(clean[..., None], got, 0), np.where(clean[..., None], want, 0), f"{which} {value}")
    if which == "v":
        assert np.array_equal(got[touched], np.full(touched.sum(), value, np.float32), equal_nan=True)
        part = touched.any(-1)[..., None] & ~touched  # the other dims of the rows that see it
        assert np.isfinite(got[part]).all() and np.abs(got[part] - want[part]).max() < 64 * U
    else:
        # a key of one infinite value: the score is infinite, its weight 0 or the row NaN as the formula has it
        assert np.array_equal(np.isnan(got[touched]), np.isnan(want[touched]))
        fine = touched & np.isfinite(want)
        assert np.abs(got[fine] - want[fine]).max(initial=0) < 64 * U


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new", [[1, 1], [3, 2], [90, 65]])
def test_large_and_small_values(hip, qtype, new):
    """Queries and keys far from 1 (the type's large and tiny values), values of very different sizes."""
    p = Paged(hip, 44, qtype, 8, 2, 64, 16, new, [200, 66])
    big = 2.0 ** 9 if qtype == L.F16 else 2.0 ** 40
    for pool, host, f in ((p.kp, p.k, big), (p.vp, p.v, 1.0 / big)):
        pool.t.mul_(f)
        for r in range(2):
            host[r] *= f
    if qtype == L.F16:  # products of subnormal halves lose bits in the pool itself: take what it holds
        for r in range(2):
            for j in range(p.kv[r]):
                pg, off = p.place(r, j)
                p.v[r][j] = p.vp.t[pg, :2 * 16 * 64].view(2, 16, 64)[:, off].double().cpu().numpy()
    p.q *= np.float32(1.0 / big)
    p.put("v", 0, 3, 0, 9, 3e4)  # beside values of 2^-9 and less
    got, want = p.run(), p.want()
    check(got, want, f"large {qtype} {new}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("offset", [10.0, 40.0])
@pytest.mark.parametrize("new,kv", [([1], [2000]), ([150], [1100])])
def test_scores_with_a_common_part(hip, qtype, offset, new, kv):
    """Scores around an offset, as trained models have, on one dim that no rounding of q or k touches."""
    p = Paged(hip, 50, qtype, 8, 2, 64, 16, new, kv)
    for r in range(len(kv)):
        for j in range(kv[r]):
            for g in range(2):
                p.put("k", r, j, g, 63, 8.0)
    p.q[..., 63] = offset  # scale 1 / 8
    got, want = p.run(), p.want()
    # the score's own roundings are at the offset's size: sqrt(partial sums) / 2 of 2^-24 * offset, as absolute errors
    # of the exponent; the rest as above
    norm = np.linalg.norm(want, axis=-1)
    rel = np.linalg.norm(got - want, axis=-1) / norm
    print(f"offset {offset}: worst {rel.max() / U:.1f} u", flush=True)
    assert rel.max() < WORST + 4 * offset * U


@pytest.mark.parametrize("new,kv", [([1, 1], [300, 40]), ([70, 2], [300, 40])])
def test_offsets_past_32_bits(hip, new, kv):
    """Pages behind the first 2^32 values of the pool (8 GiB each of K and V): stored there and found again."""
    KV, hd, page, H = 8, 128, 64, 16
    per = KV * page * hd
    n_pages = 2 ** 32 // per + 9
    p = Paged(hip, 97, L.F16, H, KV, hd, page, new, kv)
    kp, vp = (torch.empty(n_pages, per, dtype=torch.float16, device="cuda") for _ in range(2))
    far = [n_pages - 1 - i for i in range(p.n_pages)]  # where each page of the small pool goes
    for a, b in ((p.kp, kp), (p.vp, vp)):
        for i, f in enumerate(far):
            b[f] = a.t[i]
    p.table = np.where(p.table >= 0, np.array(far)[p.table.clip(0)], -1)
    pool = hip.PagePool(n_pages, page, KV, hd, L.F16, k=Dev(kp), v=Dev(vp))
    p.pool = pool
    check(p.run(), p.want(), f"far pages {new}")
    # and a store there
    x = torch.randn(1, (H + 2 * KV) * hd)
    dx, pos, slot = Dev(x), i32([0]), Dev(torch.tensor([(n_pages - 1) * page + 63]))
    cos, sin = Dev(torch.ones(1, hd // 2)), Dev(torch.zeros(1, hd // 2))
    torch.cuda.synchronize()
    base, w = dx.ptr, (H + 2 * KV) * hd
    hip.rope_append(base, w, base, w, H, base + 4 * H * hd, w, base + 4 * (H + KV) * hd, w, 1, pos, cos, sin, 1, slot, pool)
    hip.sync()
    got = kp[n_pages - 1].view(KV, page, hd)[:, 63].float().cpu()
    assert torch.equal(got, x[0, H * hd:(H + KV) * hd].view(KV, hd).half().float())


def test_repeated_calls_give_the_same_bits(hip):
    for new, kv in (([1] * 5, [900, 3, 77, 2000, 512]), ([1, 90, 1], [900, 400, 33])):
        p = Paged(hip, 60, L.F16, 32, 4, 64, 16, new, kv)
        a = p.run()
        for _ in range(3):
            p.launch()
            p.hip.sync()
            assert np.array_equal(p.fetch(), a)


def test_two_calls_at_once_on_two_streams(hip):
    s1, s2 = hip.Stream(), hip.Stream()
    a = Paged(hip, 61, L.BF16, 32, 4, 64, 16, [1] * 9, [1500 + 7 * i for i in range(9)])
    b = Paged(hip, 62, L.F32, 8, 2, 128, 32, [100, 1], [700, 900])
    ra, rb = a.run(), b.run()
    for _ in range(4):
        a.dev[1].t.fill_(5.0)
        b.dev[1].t.fill_(5.0)
        torch.cuda.synchronize()
        a.launch(s1)
        b.launch(s2)
        s1.sync()
        s2.sync()
        assert np.array_equal(a.fetch(), ra) and np.array_equal(b.fetch(), rb)


def test_too_small_a_workspace_is_refused(hip):
    p = Paged(hip, 63, L.F16, 32, 4, 64, 16, [1], [4000])
    p.run()
    dq, out, dt, ds, dk, ws, args, ldq = p.dev
    need = hip.paged_attention_workspace_bytes(32, p.pool, *args)
    if need:
        small = Dev(torch.zeros(need - 1, dtype=torch.uint8))
        with pytest.raises(L.HipError, match="workspace"):
            hip.paged_attention(dq, ldq, out, ldq, 32, p.pool, dt, p.ld, ds, dk, *args, 0.125, ws=small)
        with pytest.raises(L.HipError, match="workspace"):
            hip.paged_attention(dq, ldq, out, ldq, 32, p.pool, dt, p.ld, ds, dk, *args, 0.125, ws=None)


# ---- packed prompts --------------------------------------------------------------------------------------
class Packed:
    def __init__(self, hip, seed, qtype, H, KV, hd, lens, pad=0):
        g = D.rng(seed)
        self.hip, self.qtype, self.H, self.KV, self.hd, self.lens = hip, qtype, H, KV, hd, lens
        self.rows = sum(lens)
        self.start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.q = g.standard_normal((self.rows, H, hd), dtype=np.float32)
        self.k, self.v = (torch.from_numpy(g.standard_normal((self.rows, KV, hd), dtype=np.float32)).to(TORCH[qtype]) for _ in range(2))
        self.pad = pad

    def run(self, behind=3, stream=None):
        H, KV, hd, n = self.H, self.KV, self.hd, self.rows + behind
        ldq, ldk, ldv = H * hd + self.pad, KV * hd + self.pad, KV * hd + 2 * self.pad
        q = torch.full((n, ldq), float("nan"))
        q[:self.rows, :H * hd] = torch.from_numpy(self.q).view(self.rows, -1)
        k, v = (torch.full((n, ld), float("nan"), dtype=TORCH[self.qtype]) for ld in (ldk, ldv))
        k[:self.rows, :KV * hd], v[:self.rows, :KV * hd] = self.k.view(self.rows, -1), self.v.view(self.rows, -1)
        need = self.hip.packed_attention_workspace_bytes(H, KV, hd, self.qtype, len(self.lens), n)
        self.dev = (Dev(q), Dev(k), Dev(v), Dev(torch.full((n, ldq), 5.0)), i32(self.start), Dev(torch.full((max(need, 16),), 0xFF, dtype=torch.uint8)),
                    (ldq, ldk, ldv, n))
        torch.cuda.synchronize()
        self.launch(stream)
        self.hip.sync(stream)
        return self.fetch()

    def launch(self, stream=None):
        q, k, v, out, start, ws, (ldq, ldk, ldv, n) = self.dev
        self.hip.packed_attention(q, ldq, k, ldk, v, ldv, self.qtype, out, ldq, self.H, self.KV, self.hd, start, len(self.lens), n,
                                  float(1.0 / np.sqrt(self.hd)), ws=ws, stream=stream)

    def fetch(self):
        o = self.dev[3].np()
        assert (o[self.rows:] == 5.0).all() and (o[:, self.H * self.hd:] == 5.0).all()
        return o[:self.rows, :self.H * self.hd].reshape(self.rows, self.H, self.hd)

    def want(self):
        out, k, v = np.zeros((self.rows, self.H, self.hd)), self.k.double().numpy(), self.v.double().numpy()
        for r, n in enumerate(self.lens):
            a = self.start[r]
            for i in range(n):
                out[a + i] = softmax_ref(self.q[a + i].astype(np.float64), k[a:a + i + 1], v[a:a + i + 1], 1.0 / np.sqrt(self.hd))
        return out


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("H,KV,hd", SHAPES)
@pytest.mark.parametrize("lens", [[1], [0, 5, 0, 1, 64, 65, 0], [33, 200, 16, 15, 17], [300]])
def test_packed(hip, qtype, H, KV, hd, lens):
    print(f"[case] packed {qtype} H={H} KV={KV} hd={hd} {lens}", flush=True)
    p = Packed(hip, hd + len(lens), qtype, H, KV, hd, lens, pad=8)
    check(p.run(), p.want(), f"packed {qtype} {H}/{KV}/{hd} {lens}")


@pytest.mark.parametrize("qtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("which", ["k", "v"])
def test_packed_infinities(hip, qtype, value, which):
    """An infinite value or key row: prompts beside it and rows before it do not see it."""
    p = Packed(hip, 9, qtype, 8, 2, 64, [50, 150, 40])
    (p.k if which == "k" else p.v)[50 + 100, 1, 7] = value
    got, seen = p.run(), np.zeros((p.rows, 8), bool)
    seen[150:200, 4:] = True
    with np.errstate(all="ignore"):
        want = p.want()
    assert np.isfinite(got[~seen]).all()
    check(np.where(seen[..., None], 0, got), np.where(seen[..., None], 0, want), f"packed {which} {value}")
    if which == "v":
        assert np.array_equal(got[150:200, 4:, 7], np.full((50, 4), value, np.float32), equal_nan=True)
        rest = [d for d in range(64) if d != 7]
        assert np.abs(got[150:200, 4:][..., rest] - want[150:200, 4:][..., rest]).max() < 64 * U
    else:
        assert np.array_equal(np.isnan(got[seen]), np.isnan(want[seen]))


# FP32 and BF16 keys and values prepared as FP16 tiles, as they are where there is enough work.
# Either way FP32 tiles are scaled and split, before the kernel or in it.
@pytest.fixture(params=["prepared", "rows"])
def prepared(request, monkeypatch):
    monkeypatch.setenv("EF_HIP_PACKED_ATTENTION", request.param)
    return request.param == "prepared"


@pytest.mark.parametrize("qtype", [L.F32, L.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [(4, 2, 64), (2, 1, 128), (3, 1, 80), (2, 1, 256), (2, 2, 8)])
@pytest.mark.parametrize("lens", [[1024], [0, 300, 1, 63, 64, 65, 0, 700, 31, 32, 33, 0]])
def test_packed_prepared(hip, prepared, qtype, H, KV, hd, lens):
    print(f"[case] prepared {qtype} H={H} KV={KV} hd={hd} {lens}", flush=True)
    p = Packed(hip, hd + len(lens), qtype, H, KV, hd, lens, pad=8)
    assert (hip.packed_attention_workspace_bytes(H, KV, hd, qtype, len(lens), p.rows + 3) > 0) == prepared
    check(p.run(), p.want(), f"prepared {qtype} {H}/{KV}/{hd} {lens}")


@pytest.mark.parametrize("qtype", [L.F32, L.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("how", ["tiles", "jumps", "rows", "zeros", "huge", "tiny"])
def test_packed_prepared_scales(hip, prepared, qtype, hd, how):
    """Keys and values of very different sizes: from tile to tile, past what the sums' scale can follow, from row to row
    of a tile, tiles and rows of zeros, and whole inputs far from 1 (queries the other way, so that scores stay)."""
    p = Packed(hip, 71, qtype, 2, 1, hd, [1000, 90])
    f = torch.ones(p.rows, 1, 1)
    i = torch.arange(p.rows)
    if how == "tiles":
        f = (2.0 ** ((i // 64 * 5) % 23 - 11).double()).float().view(-1, 1, 1)
    elif how == "jumps":
        f = (2.0 ** torch.where(i // 64 % 3 == 1, 60.0, torch.where(i // 64 % 3 == 2, -40.0, 0.0)).double()).float().view(-1, 1, 1)
    elif how == "rows":
        f = torch.where(i % 37 == 5, 2.0 ** 20, torch.where(i % 41 == 7, 2.0 ** -20, 1.0)).view(-1, 1, 1)
    elif how == "zeros":
        f = torch.where((i // 64 % 3 == 0) | (i % 5 == 1), 0.0, 1.0).view(-1, 1, 1)
    big = {"huge": 2.0 ** 50, "tiny": 2.0 ** -50}.get(how, 1.0)
    p.k = (p.k.float() * big).to(TORCH[qtype])
    p.q = p.q * np.float32(1.0 / big)
    p.v = (p.v.float() * f * big).to(TORCH[qtype])
    if how == "zeros":
        p.k = (p.k.float() * f).to(TORCH[qtype])
    if how == "rows":  # keys of uneven sizes as well, none so large that one position takes all the weight
        p.k = (p.k.float() * torch.where(i % 29 == 3, 2.0 ** -30, 1.0).view(-1, 1, 1)).to(TORCH[qtype])
    got, want = p.run(), p.want()
    assert np.isfinite(got).all()
    # Where one value row outweighs the others by its size, its weight's own error is the output's: nothing averages it, and
    # with a small weight nothing cancels it against the sum.  The exponent c2 s - sub of a weight of e^-10 is about -14:
    # its rounding (half an ulp of 8 .. 16) is 8 u, c2's two roundings (1.5 u relative) make 21 u of it at 14, together
    # ln 2 (8 + 21) = 20 u; the score's sums and parts are 12 u, exp2 2 u, the sum's and the output's own sums 8 u:
    # below 48 u.
    check(got, want, f"scales {how} {qtype} {hd}", worst=48 * U if how in ("tiles", "jumps", "rows") else WORST)


@pytest.mark.parametrize("qtype", [L.F32, L.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("which", ["k", "v"])
def test_packed_prepared_infinities(hip, prepared, qtype, value, which):
    p = Packed(hip, 10, qtype, 8, 2, 64, [80, 900, 60])
    at = 80 + 500
    (p.k if which == "k" else p.v)[at, 1, 7] = value
    got, seen = p.run(), np.zeros((p.rows, 8), bool)
    seen[at:980, 4:] = True
    with np.errstate(all="ignore"):
        want = p.want()
    assert np.isfinite(got[~seen]).all()
    check(np.where(seen[..., None], 0, got), np.where(seen[..., None], 0, want), f"prepared {which} {value}")
    if which == "v":
        assert np.array_equal(got[at:980, 4:, 7], np.full((400, 4), value, np.float32), equal_nan=True)
        rest = [d for d in range(64) if d != 7]
        assert np.abs(got[at:980, 4:][..., rest] - want[at:980, 4:][..., rest]).max() < 64 * U
    else:
        assert np.array_equal(np.isnan(got[seen]), np.isnan(want[seen]))
        fine = seen[..., None] & np.isfinite(want)
        assert np.abs(got[fine] - want[fine]).max(initial=0) < 64 * U


@pytest.mark.parametrize("qtype", [L.F32, L.BF16], ids=["f32", "bf16"])
def test_packed_rows_and_prepared_agree(hip, monkeypatch, qtype):
    """Either way of a packed call, on sides of the rule that chooses: the same within both tolerances."""
    p = Packed(hip, 12, qtype, 4, 2, 64, [500, 30])
    monkeypatch.setenv("EF_HIP_PACKED_ATTENTION", "rows")
    assert hip.packed_attention_workspace_bytes(4, 2, 64, qtype, 2, p.rows + 3) == 0
    a, want = p.run(), p.want()
    monkeypatch.setenv("EF_HIP_PACKED_ATTENTION", "prepared")
    b = p.run()
    check(a, want, f"rows {qtype}")
    check(b, want, f"prepared {qtype}")


@pytest.mark.parametrize("hd", [64, 96, 256])
@pytest.mark.parametrize("how", ["tiles", "jumps", "rows", "zeros"])
def test_chunk_scales(hip, hd, how):
    """FP32 pages whose values' sizes differ from tile to tile, by more than the sums' scale can follow, from row to row,
    and rows of zeros, with a page lost among them."""
    p = Paged(hip, 95, L.F32, 4, 2, hd, 16, [90, 1], [420, 200])
    for r in range(2):
        for j in range(p.kv[r]):
            f = {"tiles": 2.0 ** (j // 64 * 5 % 23 - 11), "jumps": (1.0, 2.0 ** 60, 2.0 ** -40)[j // 64 % 3],
                 "rows": 2.0 ** 20 if j % 37 == 5 else 2.0 ** -20 if j % 41 == 7 else 1.0,
                 "zeros": 0.0 if j // 64 % 3 == 0 or j % 5 == 1 else 1.0}[how]
            pg, off = p.place(r, j)
            for pool, host in ((p.vp, p.v),) + (((p.kp, p.k),) if how == "zeros" else ()):
                view = pool.t[pg].view(2, 16, hd)
                view[:, off] *= f
                host[r][j] *= f
    lost = {(0, 3)}
    table = p.table.copy()
    table[0, 3] = -1
    check(p.run(table=table), p.want(lost), f"chunk scales {how} {hd}", worst=48 * U if how != "zeros" else WORST)


def test_long_context_of_one_request(hip):
    """One request whose positions are cut into more ranges than one wave adds (65 and more), and a few rows of it."""
    for new, kv, qtype in ((1, 30001, L.F32), (3, 20011, L.F16), (1, 64 * 128 + 1, L.BF16)):
        p = Paged(hip, 90, qtype, 8, 1, 128, 32, [new], [kv])
        check(p.run(), p.want(), f"long context {kv} {qtype}")


def test_packed_workspace_is_checked(hip):
    p = Packed(hip, 11, L.F32, 4, 2, 64, [1100])
    p.run()
    q, k, v, out, start, ws, (ldq, ldk, ldv, n) = p.dev
    need = hip.packed_attention_workspace_bytes(4, 2, 64, L.F32, 1, n)
    for small in (Dev(torch.zeros(need - 1, dtype=torch.uint8)), None):
        with pytest.raises(L.HipError, match="workspace"):
            hip.packed_attention(q, ldq, k, ldk, v, ldv, L.F32, out, ldq, 4, 2, 64, start, 1, n, 0.125, ws=small)


# ---- captured ------------------------------------------------------------------------------------------
def test_captured_step_replays_with_other_lengths(hip):
    """plan, append and attention captured once over fixed bounds, replayed while requests grow, end and start: every
    replay against the same calls made eagerly, with eager work in between."""
    H, KV, hd, page, n, ld, n_pages, max_rows, n_pos = 8, 2, 64, 8, 6, 16, 70, 24, 128
    g = torch.Generator().manual_seed(3)
    cos, sin = hip.rope_tables(10000.0, hd, n_pos)
    width = (H + 2 * KV) * hd

    def state():
        z = lambda *s, dt=torch.int32: Dev(torch.zeros(*s, dtype=dt))  # noqa: E731
        s = dict(len=z(n), new=z(n), table=Dev(torch.full((n, ld), -1, dtype=torch.int32)), free=i32(np.arange(n_pages)), n_free=i32([n_pages]),
                 start=z(n + 1), pos=z(max_rows), slot=z(max_rows, dt=torch.int64), status=z(4), qkv=Dev(torch.zeros(max_rows, width)),
                 out=Dev(torch.zeros(max_rows, H * hd)), kp=Dev(torch.zeros(n_pages, KV * page * hd, dtype=torch.float16)),
                 vp=Dev(torch.zeros(n_pages, KV * page * hd, dtype=torch.float16)))
        s["pool"] = hip.PagePool(n_pages, page, KV, hd, L.F16, k=s["kp"], v=s["vp"])
        need = hip.paged_attention_workspace_bytes(H, s["pool"], n, max_rows, 12, ld * page)
        s["ws"] = Dev(torch.zeros(max(need, 16), dtype=torch.uint8))
        return s

    def step(s, stream):
        hip.page_plan(s["len"], s["new"], n, page, n_pages, s["table"], ld, s["free"], s["n_free"], s["n_free"], s["len"], s["start"], s["pos"],
                      s["slot"], max_rows, s["status"], stream=stream)
        b = s["qkv"].ptr
        hip.rope_append(b, width, b, width, H, b + 4 * H * hd, width, b + 4 * (H + KV) * hd, width, max_rows, s["pos"], cos, sin, n_pos, s["slot"],
                        s["pool"], stream=stream)
        hip.paged_attention(b, width, s["out"], H * hd, H, s["pool"], s["table"], ld, s["start"], s["len"], n, max_rows, 12, ld * page,
                            0.125, ws=s["ws"], stream=stream)

    eager, held = state(), state()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(held, torch.cuda.current_stream().cuda_stream)
    own = hip.Stream()
    r = D.rng(17)
    lens = np.zeros(n, int)
    for it in range(30):
        new = r.integers(0, 4, n)
        new[r.integers(0, n)] = r.integers(5, 10)
        if it % 4 == 3:
            new[r.integers(0, n)] = -1
        new = np.where(lens + new > ld * page, -1, new)
        lens = np.where(new < 0, 0, lens + new)
        qkv = torch.randn(max_rows, width, generator=g)
        for s in (eager, held):
            s["new"].t.copy_(torch.from_numpy(new.astype(np.int32)))
            s["qkv"].t.copy_(qkv)
            s["out"].t.fill_(3.0)
        torch.cuda.synchronize()
        step(eager, own.ptr)
        own.sync()
        graph.replay()
        torch.cuda.synchronize()
        for k in ("len", "table", "free", "n_free", "start", "pos", "slot", "status", "qkv", "out", "kp", "vp"):
            assert torch.equal(eager[k].t, held[k].t), (it, k)
        assert eager["status"].t.sum().item() == 0 and eager["len"].np().tolist() == lens.tolist()
        assert torch.isfinite(eager["out"].t).all()
