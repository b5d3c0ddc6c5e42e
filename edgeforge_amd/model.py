"""Synthetic TinyLlama-shaped models on the device and the decode engine over them.

The model mirrors the reference's quantized file layout (src/model.cpp:66-111): every layer
matrix Q4_0 except the TinyLlama policy's six Q8_0 overrides (src/quantizer.cpp:75-80), a Q8_0
lm_head, a BF16 embedding and F32 norms.  Weights are random-init N(0, 0.02) and norms
1 + 0.1 N(0, 1) (tools/make_synthetic_checkpoint.py:92-95), generated on the device and packed by
the device quantizer, which is byte-identical to the reference's quantize_row.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field

import numpy as np

from . import _lib as EL
from . import hip as H

LAYER_MATS = ("wq", "wk", "wv", "wo", "w_gate", "w_up", "w_down")
# model.layers.{l}.self_attn.{k,v}_proj stored Q8_0 by the tinyllama-1.1b-chat-v1.0 policy
TINYLLAMA_Q8 = frozenset({(0, "wk"), (0, "wv"), (1, "wv"), (2, "wv"), (17, "wv"), (18, "wv")})


def _packed_row_bytes(qtype: int, cols: int) -> int:  # src/quant.cpp:136-149
    return cols // 32 * (34 if qtype == EL.Q8_0 else 18)


@dataclass
class Config:
    D: int = 2048
    F: int = 5632
    H: int = 32
    KV: int = 4
    hd: int = 64
    V: int = 32000
    L: int = 22
    max_pos: int = 2048
    eps: float = 1e-5
    rope_theta: float = 10000.0

    def shape(self, name: str) -> tuple[int, int]:
        kvd = self.KV * self.hd
        return {"wq": (self.D, self.D), "wk": (kvd, self.D), "wv": (kvd, self.D), "wo": (self.D, self.D),
                "w_gate": (self.F, self.D), "w_up": (self.F, self.D), "w_down": (self.D, self.F)}[name]

    def c_struct(self) -> EL.ef_hip_model_config:
        return EL.ef_hip_model_config(self.D, self.F, self.H, self.KV, self.hd, self.V, self.L, self.max_pos,
                                     self.eps, self.rope_theta)

    def weight_bytes_per_token(self, q8=TINYLLAMA_Q8, lm_type=EL.Q8_0) -> int:
        """Bytes streamed per decoded token: layer matrices + norms + lm_head (QuantFile::bytes_per_token)."""
        total = 0
        for l in range(self.L):
            for m in LAYER_MATS:
                r, c = self.shape(m)
                total += r * _packed_row_bytes(EL.Q8_0 if (l, m) in q8 else EL.Q4_0, c)
            total += 2 * self.D * 4
        total += self.D * 4 + self.V * _packed_row_bytes(lm_type, self.D)
        return total


TINYLLAMA = Config()


@dataclass
class DeviceModel:
    cfg: Config
    seed: int
    q8: frozenset = TINYLLAMA_Q8
    weights: dict = field(default_factory=dict)  # (layer, name) -> H.Weight ; ("embed"|"lm_head") -> H.Weight
    packed: dict = field(default_factory=dict)   # same keys -> DeviceArray of packed bytes
    norms: dict = field(default_factory=dict)    # (layer, "attn"|"ffn") | "final" -> DeviceArray

    @classmethod
    def synthetic(cls, cfg: Config, seed: int = 1234, q8=TINYLLAMA_Q8, layer_type: int = EL.Q4_0,
                  lm_type: int = EL.Q8_0, embed_type: int = EL.BF16, std: float = 0.02) -> "DeviceModel":
        H.init()
        m = cls(cfg, seed, frozenset(q8))
        biggest = max(cfg.V, cfg.F, cfg.D) * cfg.D  # embedding and head, feed-forward, q and o
        scratch = H.DeviceArray((biggest,), np.float32)
        tid = 0

        def gen(n, mean, scale):
            nonlocal tid
            EL.call("ef_hip_fill_normal", scratch.ptr, n, seed, tid, mean, scale, None)
            tid += 1

        def pack(key, qtype, rows, cols):
            gen(rows * cols, 0.0, std)
            buf = H.quantize(qtype, scratch, rows, cols, search=True)
            m.packed[key] = buf
            m.weights[key] = H.Weight(qtype, rows, cols, device=buf)

        pack("embed", embed_type, cfg.V, cfg.D)
        for l in range(cfg.L):
            for name in LAYER_MATS:
                r, c = cfg.shape(name)
                pack((l, name), EL.Q8_0 if (l, name) in m.q8 else layer_type, r, c)
            for nn in ("attn", "ffn"):
                gen(cfg.D, 1.0, 0.1)
                d = H.DeviceArray((cfg.D,), np.float32)
                EL.call("ef_hip_memcpy_d2d", d.ptr, scratch.ptr, cfg.D * 4, None)
                m.norms[(l, nn)] = d
        gen(cfg.D, 1.0, 0.1)
        d = H.DeviceArray((cfg.D,), np.float32)
        EL.call("ef_hip_memcpy_d2d", d.ptr, scratch.ptr, cfg.D * 4, None)
        m.norms["final"] = d
        pack("lm_head", lm_type, cfg.V, cfg.D)
        H.sync()
        scratch.free()
        return m

    def host_bytes(self, key) -> np.ndarray:
        w = self.weights[key]
        return self.packed[key].numpy().reshape(w.rows, w.row_bytes)

    def host_norm(self, key) -> np.ndarray:
        return self.norms[key].numpy()


class Engine:
    """ef_hip_engine: Transformer::forward on the device for `batch` sequences."""

    def __init__(self, model, max_seq: int, batch: int = 1):
        """model: a DeviceModel, or a device model handle holder with .h (qfile.EfqModel)."""
        self.model, self.max_seq, self.batch = model, max_seq, batch
        cfg = model.cfg
        if not isinstance(model, DeviceModel):
            h = C.c_void_p()
            EL.call("ef_hip_model_engine_create", model.h, max_seq, batch, C.byref(h))
            self.h = h.value
            return
        layers = (EL.ef_hip_layer * cfg.L)()
        for l in range(cfg.L):
            layers[l] = EL.ef_hip_layer(*[model.weights[(l, n)].handle for n in LAYER_MATS],
                                       model.norms[(l, "attn")].ptr, model.norms[(l, "ffn")].ptr)
        self._cfg = cfg.c_struct()
        h = C.c_void_p()
        EL.call("ef_hip_engine_create", C.byref(self._cfg), layers, model.weights["embed"].handle,
               model.weights["lm_head"].handle, model.norms["final"].ptr, max_seq, batch, C.byref(h))
        self.h = h.value

    def forward(self, tokens, pos: int, compute_logits: bool = True) -> None:
        t = np.ascontiguousarray(np.asarray(tokens, dtype=np.int32).reshape(self.batch))
        EL.call("ef_hip_engine_forward", self.h, t.ctypes.data_as(EL._i32p), pos, int(compute_logits))

    def prefill(self, tokens, pos: int, compute_logits: bool = True) -> None:
        """tokens [batch][n] at positions pos .. pos+n-1, all rows at once (ef_hip_engine_prefill)."""
        t = np.ascontiguousarray(np.asarray(tokens, dtype=np.int32).reshape(self.batch, -1))
        EL.call("ef_hip_engine_prefill", self.h, t.ctypes.data_as(EL._i32p), t.shape[1], pos, int(compute_logits))

    def _fetch(self, fn: str, n: int) -> np.ndarray:
        p = C.c_void_p()
        EL.call(fn, self.h, C.byref(p))
        out = np.empty((self.batch, n), np.float32)
        EL.call("ef_hip_memcpy_d2h", out.ctypes.data, p.value, out.nbytes, None)
        return out

    def logits(self) -> np.ndarray:
        return self._fetch("ef_hip_engine_logits", self.model.cfg.V)

    def hidden(self) -> np.ndarray:
        return self._fetch("ef_hip_engine_hidden", self.model.cfg.D)

    def generate(self, prompt, n: int, sampler: dict | None = None, rng: H.RngStates | None = None):
        """prompt [batch][n_prompt] -> (tokens [batch][n], prefill_s, decode_s)."""
        p = np.ascontiguousarray(np.asarray(prompt, dtype=np.int32).reshape(self.batch, -1))
        out = np.empty((self.batch, n), np.int32)
        pre, dec = C.c_double(), C.c_double()
        cfg = None
        if sampler is not None:
            cfg = EL.ef_hip_sampler_config(sampler.get("temperature", 0.0), sampler.get("top_k", 0),
                                          sampler.get("top_p", 1.0), sampler.get("repetition_penalty", 1.0),
                                          sampler.get("seed", 0))
        EL.call("ef_hip_engine_generate", self.h, p.ctypes.data_as(EL._i32p), p.shape[1], n,
               C.byref(cfg) if cfg is not None else None, rng.buf.ptr if rng else None,
               out.ctypes.data_as(EL._i32p), C.byref(pre), C.byref(dec))
        return out, pre.value, dec.value

    def reply(self, ids, max_new: int, sampler: dict | None = None, rng: H.RngStates | None = None,
              eos_id: int = -1, eos_min_p: float = 0.0, steps_per_check: int = 8):
        """ChatSession::reply at the token level (batch 1): (reply ids, P(EOS) per step, stats)."""
        ids = np.ascontiguousarray(np.asarray(ids, dtype=np.int32).reshape(-1))
        sampler = sampler or {}
        cfg = EL.ef_hip_sampler_config(sampler.get("temperature", 0.0), sampler.get("top_k", 0),
                                      sampler.get("top_p", 1.0), sampler.get("repetition_penalty", 1.0),
                                      sampler.get("seed", 0))
        opts = EL.ef_hip_reply_options(max_new, eos_id, eos_min_p, steps_per_check)
        out = np.empty(max_new, np.int32)
        peos = np.empty(max_new, np.float64)
        st = EL.ef_hip_reply_stats()
        EL.call("ef_hip_engine_reply", self.h, ids.ctypes.data_as(EL._i32p), ids.size, C.byref(cfg),
               rng.buf.ptr if rng else None, C.byref(opts), out.ctypes.data_as(EL._i32p),
               peos.ctypes.data_as(C.POINTER(C.c_double)), C.byref(st))
        return out[:st.generated].copy(), peos[:st.steps].copy(), st

    PROFILE_GROUPS = ("embed", "qkv", "attention", "o_proj", "gate_up", "down", "lm_head", "pick")

    def staged_tables(self) -> tuple[bool, str]:
        """Whether several-sequence steps run over producer-staged product inputs, and why not
        (ef_hip_engine_tables)."""
        on, why = C.c_int(0), C.c_char_p()
        EL.call("ef_hip_engine_tables", self.h, C.byref(on), C.byref(why))
        return bool(on.value), (why.value or b"").decode()

    def profile(self, reps: int = 20, sampler: dict | None = None, rng: H.RngStates | None = None) -> dict:
        """Milliseconds per step of each kernel group of a decode step (ef_hip_engine_profile)."""
        out = (C.c_double * len(self.PROFILE_GROUPS))()
        cfg = None
        if sampler is not None:
            cfg = EL.ef_hip_sampler_config(sampler.get("temperature", 0.0), sampler.get("top_k", 0),
                                          sampler.get("top_p", 1.0), sampler.get("repetition_penalty", 1.0),
                                          sampler.get("seed", 0))
        EL.call("ef_hip_engine_profile", self.h, C.byref(cfg) if cfg is not None else None,
               rng.buf.ptr if rng else None, reps, out)
        return {g: float(out[i]) for i, g in enumerate(self.PROFILE_GROUPS)}

    def reset(self) -> None:
        EL.call("ef_hip_engine_reset", self.h)

    def score(self, ids, first: int = 0, logits: H.DeviceArray | None = None) -> np.ndarray:
        """Teacher-forced NLL of ids[p+1] at positions p in [first, n-1) (batch 1); logits, when given,
        receives those positions' logits [(n-1-first)][V] on the device."""
        ids = np.ascontiguousarray(np.asarray(ids, dtype=np.int32).reshape(-1))
        nll = np.empty(ids.size - 1 - first, np.float64)
        EL.call("ef_hip_engine_score", self.h, ids.ctypes.data_as(EL._i32p), ids.size, first,
               nll.ctypes.data_as(C.POINTER(C.c_double)), logits.ptr if logits is not None else None)
        return nll

    def close(self) -> None:
        if getattr(self, "h", None):
            EL.call("ef_hip_engine_destroy", self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


MOST_ROWS = 65535  # rows that one product (and ef_hip_rows_f32) takes


class PagesShort(RuntimeError):
    """A step needs more free pages than there are; nothing was changed."""


class PagedEngine:
    """Transformer::forward for requests of different lengths that come and go: a pool of KV pages per
    layer, block tables and slots planned on the device, and each step's new tokens (one for a request
    that decodes, a chunk for one whose prompt is brought in) through every product together.

    `seqs` slots hold one request each; step() takes the new tokens of any of them, release() gives a
    slot's pages back.  After a step, `logits` holds row i's logits [V] on the device for the i-th slot
    that got tokens (in order of slots): hip.sample and hip.argmax take it from there.  step() returns without
    waiting: what reads `logits` runs on the same `stream` (`stream=` of those calls, `logits.numpy(stream)`) or
    waits for it.  score() takes `logits` for its own.  `kv_type` is what
    the pages hold (F32 as the engine's cache, F16 or BF16 for half the memory and traffic)."""

    def __init__(self, model, pages: int, page_size: int = 16, seqs: int = 64, rows: int = 512, max_seq: int | None = None,
                 kv_type: int = EL.F32, stream=None):
        """model: a DeviceModel or an EfqModel (which has to outlive this).  rows: new tokens of one step;
        max_seq: positions of one request."""
        self.model, self.cfg, self.stream = model, model.cfg, stream
        c = self.cfg
        if c.hd % 8 or not 8 <= c.hd <= 256:
            raise ValueError("paged attention needs a head size that is a multiple of 8 up to 256")
        if not 1 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two up to 1024")
        if pages < 1:
            raise ValueError("pages must be at least 1")
        H.init()
        self.seqs, self.rows, self.page_size, self.pages = seqs, rows, page_size, pages
        self.max_seq = min(max_seq or c.max_pos, c.max_pos)
        self.table_ld = -(-self.max_seq // page_size)
        self.kvd, self.width = c.KV * c.hd, c.D + 2 * c.KV * c.hd
        if isinstance(model, DeviceModel):
            w, nrm = model.weights, model.norms
            self._layers = [({n: w[(l, n)].handle for n in LAYER_MATS}, nrm[(l, "attn")].ptr, nrm[(l, "ffn")].ptr)
                            for l in range(c.L)]
            self._embed, self._head, self._final = w["embed"].handle, w["lm_head"].handle, nrm["final"].ptr
        else:
            self._layers = []
            for l in range(c.L):
                h = model.layer_handles(l)
                self._layers.append(({n: getattr(h, n) for n in LAYER_MATS}, h.attn_norm_dev, h.ffn_norm_dev))
            e, m, f = C.c_void_p(), C.c_void_p(), C.c_void_p()
            EL.call("ef_hip_model_tensors", model.h, C.byref(e), C.byref(m), C.byref(f))
            self._embed, self._head, self._final = e.value, m.value, f.value
        self.pools = [H.PagePool(pages, page_size, c.KV, c.hd, kv_type) for _ in range(c.L)]
        self.cos, self.sin = H.rope_tables(c.rope_theta, c.hd, self.max_seq)
        i32 = np.int32
        self.lens = np.zeros(seqs, i32)  # positions of each slot, as on the device
        self._len, self._new = H.DeviceArray.from_host(self.lens), H.DeviceArray((seqs,), i32)
        self._table = H.DeviceArray.from_host(np.full((seqs, self.table_ld), -1, i32))
        self._free = H.DeviceArray.from_host(np.arange(pages, dtype=i32))
        self._n_free = H.DeviceArray.from_host(np.array([pages], i32))
        self._start, self._status = H.DeviceArray((seqs + 1,), i32), H.DeviceArray((4,), i32)
        self._pos, self._slot = H.DeviceArray((rows,), i32), H.DeviceArray((rows,), np.int64)
        self._ids, self._last = H.DeviceArray((rows,), i32), H.DeviceArray((max(seqs, rows),), i32)
        self._x, self._qkv = H.DeviceArray((rows, c.D)), H.DeviceArray((rows, self.width))
        self._ctx, self._act = H.DeviceArray((rows, c.D)), H.DeviceArray((rows, c.F))
        self._hidden, self.logits = H.DeviceArray((seqs, c.D)), H.DeviceArray((seqs, c.V))
        self._x_rows = H.Weight(EL.F32, rows, c.D, device=self._x)  # rows of x, to pick some of them
        self._ws, self._scale = None, float(np.float32(1.0) / np.sqrt(np.float32(c.hd)))

    # ---- one step -------------------------------------------------------------------------------------
    def step(self, tokens: dict) -> list[int]:
        """tokens: {slot: new ids}.  Runs them all; returns the slots in the order of `logits`' rows.  Raises
        PagesShort, with nothing changed, when the pages do not suffice (release some, or wait).  A step that
        raises anything else leaves the requests as they were before it, too."""
        slots = sorted(tokens)
        new = np.zeros(self.seqs, np.int32)
        ids = [self._ids_of(tokens[s]) for s in slots]
        for s, t in zip(slots, ids):
            if not 0 <= s < self.seqs or t.size == 0:
                raise ValueError(f"slot {s}: no such slot, or no tokens")
            if self.lens[s] + t.size > self.max_seq:
                raise ValueError(f"slot {s}: {self.lens[s] + t.size} positions, max_seq is {self.max_seq}")
            new[s] = t.size
        n = int(new.sum())
        if n == 0:
            return []
        if n > min(self.rows, MOST_ROWS):
            raise ValueError(f"{n} new tokens, {min(self.rows, MOST_ROWS)} rows")
        c, s, lens = self.cfg, self.stream, self.lens
        max_new, max_kv = int(new.max()), int((lens + new).max())
        self._workspace(H.paged_attention_workspace_bytes(c.H, self.pools[0], self.seqs, n, max_new, max_kv))
        flat = np.concatenate(ids)
        EL.call("ef_hip_memcpy_h2d", self._ids.ptr, flat.ctypes.data, flat.nbytes, H._s(s))

        def attend(l):
            b = self._qkv.ptr
            H.rope_append(b, self.width, b, self.width, c.H, b + 4 * c.D, self.width, b + 4 * (c.D + self.kvd), self.width, n, self._pos,
                          self.cos, self.sin, self.max_seq, self._slot, self.pools[l], stream=s)
            H.paged_attention(b, self.width, self._ctx, c.D, c.H, self.pools[l], self._table, self.table_ld, self._start, self._len,
                              self.seqs, n, max_new, max_kv, self._scale, ws=self._ws, stream=s)

        try:
            self._plan(new)
            self._layers_of(n, attend)
            self._head_of(np.cumsum([t.size for t in ids]).astype(np.int32) - 1, self.logits)
        except BaseException:
            self._take_back(lens)
            raise
        return slots

    def release(self, *slots: int) -> None:
        """The slots' pages back to the pool; the slots are free for other requests."""
        if any(not 0 <= s < self.seqs for s in slots):
            raise ValueError(f"{slots}: no such slot")
        new = np.zeros(self.seqs, np.int32)
        new[list(slots)] = -1
        self._plan(new)

    def free_pages(self) -> int:
        return int(self._n_free.numpy(self.stream)[0])

    def score(self, windows) -> list[np.ndarray]:
        """Teacher-forced NLL of ids[p + 1] at every position p of each window (Engine.score, several windows of
        different lengths in one pass, without pages)."""
        c, s = self.cfg, self.stream
        out, at = [None] * len(windows), 0
        windows = [self._ids_of(w) for w in windows]
        lens = [len(w) - 1 for w in windows]
        rows = min(self.rows, MOST_ROWS)
        if any(n < 1 or n > min(rows, self.max_seq) for n in lens):
            raise ValueError(f"windows of 2 to {min(rows, self.max_seq) + 1} ids")
        while at < len(windows):  # as many windows as fit the rows
            group, n = [], 0
            while at + len(group) < len(windows) and n + lens[at + len(group)] <= rows and len(group) < self.seqs:
                n += lens[at + len(group)]
                group.append(at + len(group))
            up = {self._ids: np.concatenate([windows[i][:-1] for i in group]),
                  self._last: np.concatenate([windows[i][1:] for i in group]),
                  self._pos: np.concatenate([np.arange(lens[i], dtype=np.int32) for i in group]),
                  self._slot: np.full(n, -1, np.int64),
                  self._start: np.concatenate([[0], np.cumsum([lens[i] for i in group])]).astype(np.int32)}
            for dev, host in up.items():
                EL.call("ef_hip_memcpy_h2d", dev.ptr, host.ctypes.data, host.nbytes, H._s(s))
            self._workspace(H.packed_attention_workspace_bytes(c.H, c.KV, c.hd, EL.F32, len(group), n))

            def attend(l):
                q = self._qkv.ptr
                k, v = q + 4 * c.D, q + 4 * (c.D + self.kvd)
                H.rope_append(q, self.width, q, self.width, c.H, k, self.width, v, self.width, n, self._pos, self.cos, self.sin, self.max_seq,
                              self._slot, self.pools[0], k_out=k, ldko=self.width, stream=s)
                H.packed_attention(q, self.width, k, self.width, v, self.width, EL.F32, self._ctx, c.D, c.H, c.KV, c.hd, self._start,
                                   len(group), n, self._scale, ws=self._ws, stream=s)

            self._layers_of(n, attend)
            nll = H.DeviceArray((n,), np.float64)
            for r0 in range(0, n, self.seqs):  # the logits' buffer holds `seqs` rows at a time
                m = min(self.seqs, n - r0)
                job = (EL.ef_hip_job * 1)(EL.ef_hip_job(self.logits.ptr, self._head, self._x.at(r0 * c.D)))
                EL.call("ef_hip_matvec_jobs_rmsnorm", job, 1, self._final, c.eps, m, c.D, c.V, H._s(s))
                EL.call("ef_hip_neg_log_prob", self.logits.ptr, c.V, m, c.V, self._last.at(r0), nll.at(r0), H._s(s))
            got, r0 = nll.numpy(s), 0
            for i in group:
                out[i] = got[r0:r0 + lens[i]].copy()
                r0 += lens[i]
            at += len(group)
        return out

    def _ids_of(self, tokens) -> np.ndarray:
        t = np.asarray(tokens).reshape(-1)
        if t.size and (t.dtype.kind not in "iu" or t.min() < 0 or t.max() >= self.cfg.V):
            raise ValueError(f"token ids are integers in the vocabulary, 0 to {self.cfg.V - 1}")
        return t.astype(np.int32)

    # ---- parts ---------------------------------------------------------------------------------------
    def _plan(self, new: np.ndarray) -> None:
        s = self.stream
        EL.call("ef_hip_memcpy_h2d", self._new.ptr, new.ctypes.data, new.nbytes, H._s(s))
        H.page_plan(self._len, self._new, self.seqs, self.page_size, self.pages, self._table, self.table_ld, self._free, self._n_free,
                    self._n_free, self._len, self._start, self._pos, self._slot, self.rows, self._status, stream=s)
        status = self._status.numpy(s)
        if status[0]:
            raise PagesShort(f"{status[0]} pages are missing")
        if status.any():
            raise RuntimeError(f"page plan refused: {status.tolist()}")
        self.lens = np.where(new < 0, 0, self.lens + new).astype(np.int32)

    def _take_back(self, lens: np.ndarray) -> None:
        """The lengths and free pages of before a step, which only takes pages: the free ones' list still holds
        them above its count, and what the table has behind a request's length is not read."""
        s = self.stream
        self.lens = lens
        self._len.upload(lens, s)
        self._n_free.upload(np.array([self.pages - int((-(-lens // self.page_size)).sum())], np.int32), s)

    def _workspace(self, need: int) -> None:
        if need and (self._ws is None or self._ws.nbytes < need):
            H.sync(self.stream)  # what uses the smaller one is done
            self._ws = H.DeviceArray((need,), np.uint8)

    def _layers_of(self, n: int, attend) -> None:
        """The embedding rows of _ids[:n] and every layer over them, in _x."""
        c, s = self.cfg, H._s(self.stream)
        x, qkv, ctx, act = self._x.ptr, self._qkv.ptr, self._ctx.ptr, self._act.ptr
        EL.call("ef_hip_rows_f32", self._embed, self._ids.ptr, n, x, c.D, s)
        for l, (w, attn_norm, ffn_norm) in enumerate(self._layers):
            jobs = (EL.ef_hip_job * 3)(EL.ef_hip_job(qkv, w["wq"], x), EL.ef_hip_job(qkv + 4 * c.D, w["wk"], x),
                                       EL.ef_hip_job(qkv + 4 * (c.D + self.kvd), w["wv"], x))
            EL.call("ef_hip_matvec_jobs_rmsnorm", jobs, 3, attn_norm, c.eps, n, c.D, self.width, s)
            attend(l)
            EL.call("ef_hip_matvec_residual", w["wo"], ctx, x, n, c.D, c.D, s)
            EL.call("ef_hip_matvec_swiglu", w["w_gate"], w["w_up"], x, ffn_norm, c.eps, act, n, c.D, c.F, s)
            EL.call("ef_hip_matvec_residual", w["w_down"], act, x, n, c.F, c.D, s)

    def _head_of(self, rows: np.ndarray, logits: H.DeviceArray) -> None:
        """Final norm and lm_head of the given rows of _x."""
        c, s = self.cfg, H._s(self.stream)
        EL.call("ef_hip_memcpy_h2d", self._last.ptr, rows.ctypes.data, rows.nbytes, s)
        EL.call("ef_hip_rows_f32", self._x_rows.handle, self._last.ptr, rows.size, self._hidden.ptr, c.D, s)
        job = (EL.ef_hip_job * 1)(EL.ef_hip_job(logits.ptr, self._head, self._hidden.ptr))
        EL.call("ef_hip_matvec_jobs_rmsnorm", job, 1, self._final, c.eps, rows.size, c.D, c.V, s)
