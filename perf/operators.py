"""What serving many requests over a paged cache is timed on: the operators through the Python view of
the C-ABI (edgeforge_amd.hip), beside the same mathematics in elementary torch operations.

Kinds of work (a case's "kind"):
  plan     one step's block tables and slot maps from the requests' lengths: pages given back by the
           requests that ended, pages taken by those that grow, each new token's position and slot
           (page_plan).
  append   RoPE on the new tokens' queries and keys, and their keys and values stored into the pages
           (rope_append).
  paged    attention of each request's new tokens over its pages, from one token (decode) to a long
           chunk, and both in one call (paged_attention).
  packed   causal attention over whole prompts of different lengths packed one after another
           (packed_attention).

Head layouts are TinyLlama-1.1B's (32 query heads over 4 KV heads of 64), the repository's own
workload, and common ones (32 over 8 of 128, as many KV heads as query heads, heads of 80, 96 and 256).
Queries and keys are N(0, 1) with a common part along some dims, as trained models' have, so that scores
spread over several units; values are N(0, 1).  Pages are handed out in random order, as they are
after a while of serving.
"""
import math
import random

import numpy as np
import torch

own = False

#: the storage types: their numbers in the library (include/ef_hip.h), torch types and bytes
TYPES = {"f32": (0, torch.float32, 4), "f16": (1, torch.float16, 2), "bf16": (2, torch.bfloat16, 2)}


# ---- the cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # a serving batch's decode step: one new token each (latency bound, before every step)
        {"name": "plan_decode_64", "kind": "plan", "seqs": 64, "new": 1, "chunks": 0, "ended": 3, "ctx": 1900, "page": 16, "mix": 1},
        # a busy step: many requests, prompts arriving, others ending
        {"name": "plan_mixed_700", "kind": "plan", "seqs": 700, "new": 400, "chunks": 70, "ended": 25, "ctx": 4000, "page": 32, "mix": 2},
        # the decode step's new tokens into a 16-bit cache
        {"name": "append_decode_64", "kind": "append", "rows": 64, "H": 32, "KV": 4, "hd": 64, "page": 16, "type": "f16", "mix": 3},
        # the rows of a long prompt
        {"name": "append_rows_7777", "kind": "append", "rows": 7777, "H": 32, "KV": 8, "hd": 128, "page": 64, "type": "bf16", "mix": 4},
        # interactive decode: one request, TinyLlama's whole context, FP32 cache as the engine's
        {"name": "decode_b1_f32", "kind": "paged", "seqs": 1, "new": 1, "chunks": 0, "ctx": 2047, "H": 32, "KV": 4, "hd": 64, "page": 16, "type": "f32", "mix": 5},
        # a serving batch of TinyLlama requests of different lengths
        {"name": "decode_b64_f16", "kind": "paged", "seqs": 64, "new": 1, "chunks": 0, "ctx": 2047, "H": 32, "KV": 4, "hd": 64, "page": 16, "type": "f16", "mix": 6},
        # a few requests with very long contexts
        {"name": "decode_long_bf16", "kind": "paged", "seqs": 12, "new": 1, "chunks": 0, "ctx": 32750, "H": 32, "KV": 8, "hd": 128, "page": 64, "type": "bf16", "mix": 7},
        # one chunk of a long prompt after what was prefilled before it
        {"name": "chunk_500_f16", "kind": "paged", "seqs": 1, "new": 500, "chunks": 1, "ctx": 8111, "H": 32, "KV": 8, "hd": 128, "page": 32, "type": "f16", "mix": 8},
        # a step that mixes decode with two prompts' chunks
        {"name": "mixed_41_bf16", "kind": "paged", "seqs": 41, "new": 300, "chunks": 2, "ctx": 1700, "H": 32, "KV": 4, "hd": 64, "page": 16, "type": "bf16", "mix": 9},
        # short prompts that arrive together
        {"name": "packed_short_f32", "kind": "packed", "seqs": 9, "rows": 333, "H": 32, "KV": 4, "hd": 64, "type": "f32", "mix": 10},
        # a few prompts of TinyLlama's context, straight from the FP32 projections
        {"name": "packed_f32", "kind": "packed", "seqs": 5, "rows": 6001, "H": 32, "KV": 4, "hd": 64, "type": "f32", "mix": 11},
        # one long prompt beside a short one
        {"name": "packed_long_f16", "kind": "packed", "seqs": 2, "rows": 9001, "H": 32, "KV": 8, "hd": 128, "type": "f16", "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "paged", "paged", "paged", "packed", "packed"])
    mix = rng.randrange(1, 1 << 20)
    page = rng.choice([1, 8, 16, 32, 64, 128])
    H, KV, hd = rng.choice([(32, 4, 64), (32, 8, 128), (16, 16, 64), (8, 1, 128), (12, 4, 80), (10, 2, 96), (8, 4, 256), (7, 1, 64)])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "plan":
        seqs = _log_int(rng, 1, 700)
        return {"kind": kind, "seqs": seqs, "new": _log_int(rng, 1, 400), "chunks": rng.randrange(0, 1 + seqs // 8),
                "ended": rng.randrange(0, 1 + seqs // 8), "ctx": _log_int(rng, 16, 4000), "page": max(8, page), "mix": mix}
    if kind == "append":
        return {"kind": kind, "rows": _log_int(rng, 1, 7777), "H": H, "KV": KV, "hd": hd, "page": page, "type": dtype, "mix": mix}
    if kind == "packed":
        rows = _log_int(rng, 30, 6000)
        return {"kind": kind, "seqs": min(rows, _log_int(rng, 1, 40)), "rows": rows, "H": H, "KV": KV, "hd": hd, "type": dtype, "mix": mix}
    shape = rng.choice(["decode", "decode", "few", "chunk", "mixed"])
    if shape in ("decode", "few"):
        seqs = _log_int(rng, 1, 128)
        new = 1 if shape == "decode" else rng.randrange(2, 9)
        ctx = _log_int(rng, 16, max(64, 120000 // seqs))
        return {"kind": kind, "seqs": seqs, "new": new, "chunks": 0 if new == 1 else seqs, "ctx": ctx, "H": H, "KV": KV, "hd": hd,
                "page": page, "type": dtype, "mix": mix}
    seqs = 1 if shape == "chunk" else _log_int(rng, 2, 41)
    return {"kind": kind, "seqs": seqs, "new": _log_int(rng, 16, 500 if seqs == 1 else 300), "chunks": 1 if seqs == 1 else rng.randrange(1, 3),
            "ctx": _log_int(rng, 16, 8111 if seqs == 1 else 1700), "H": H, "KV": KV, "hd": hd, "page": page, "type": dtype, "mix": mix}


# ---- lengths: a part of the case, so that its work is known -----------------------------------------------
def _requests(case):
    """(cached tokens, new tokens) of each request."""
    r = random.Random(case["mix"])
    n, ctx = case["seqs"], case["ctx"]
    cached = [ctx if i == 0 else r.randint(ctx // 2, ctx) for i in range(n)]
    new = [r.randint(max(1, case["new"] // 2), case["new"]) if i < case["chunks"] else 1 for i in range(n)]
    if case["chunks"]:
        new[0] = case["new"]
    if case["chunks"] > 1:
        cached[1] = 0  # a prompt that has just arrived
    for i in range(case.get("ended", 0)):
        new[n - 1 - 2 * i] = -1  # requests that ended
    order = list(range(n))
    r.shuffle(order)
    return [cached[i] for i in order], [new[i] for i in order]


def _prompts(case):
    """The packed prompts' lengths: a long one, a single token, and what lies between."""
    r = random.Random(case["mix"])
    n, rows = case["seqs"], case["rows"]
    cuts = sorted(r.randint(0, rows) for _ in range(n - 1))
    if n > 2:
        cuts[0] = min(cuts[0], 1)
        cuts.sort()
    return [b - a for a, b in zip([0] + cuts, cuts + [rows])]


def _pages(tokens, page):
    return -(-tokens // page)


# ---- inputs ------------------------------------------------------------------------------------------
class Buffer:
    """Device memory of a torch tensor, as the hip module's calls take it."""

    def __init__(self, t):
        self.t = t.contiguous()
        self.ptr = self.t.data_ptr()
        self.nbytes = self.t.numel() * self.t.element_size()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 29)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _common(hd):
    """What queries and keys share along the first dims: about 3 in every score."""
    c = torch.zeros(hd, device="cuda")
    c[:4] = math.sqrt(3.0 * math.sqrt(hd) / 4.0)
    return c


def _plan_inputs(case, seed):
    cached, new = _requests(case)
    page = case["page"]
    held = [_pages(c, page) for c in cached]
    need = [max(0, _pages(c + x, page) - h) if x >= 0 else 0 for c, x, h in zip(cached, new, held)]
    n_pages = sum(held) + sum(need) + 37
    ld = max(h + t for h, t in zip(held, need)) + 2
    ids = np.random.default_rng(seed * 31 + 7).permutation(n_pages).astype(np.int32)
    table = np.full((len(cached), ld), -1, np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = ids[at:at + h]
        at += h
    free = np.full(n_pages, -1, np.int32)
    free[:n_pages - at] = ids[at:]
    rows = sum(max(0, x) for x in new)
    max_rows = rows + 13  # a padded step
    return {"cached": _ints(cached), "new": _ints(new), "table": torch.from_numpy(table).cuda(), "free": torch.from_numpy(free).cuda(),
            "n_free": _ints([n_pages - at]), "n_pages": n_pages, "ld": ld, "max_rows": max_rows, "seqs": len(cached)}


def _append_inputs(case, seed):
    g, rows, H, KV, hd, page = _gen(seed), case["rows"], case["H"], case["KV"], case["hd"], case["page"]
    n_pages = _pages(rows, page) + 5
    qkv = _randn(g, rows, (H + 2 * KV) * hd)  # the projections' output, one row per token
    dtype = TYPES[case["type"]][1]
    pools = [_randn(g, n_pages, KV, page, hd).to(dtype) for _ in range(2)]
    perm = torch.randperm(n_pages * page, generator=g, device="cuda")[:rows]
    slot = perm.sort()[0][torch.randperm(rows, generator=g, device="cuda")] if case["mix"] % 2 else perm
    n_pos = 8192
    pos = torch.randint(0, n_pos, (rows,), generator=g, device="cuda", dtype=torch.int32)
    inv = 10000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    ang = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * inv
    return {"qkv": qkv, "k_pool": pools[0], "v_pool": pools[1], "slot": slot.to(torch.int64), "pos": pos, "cos": ang.cos().float(),
            "sin": ang.sin().float(), "n_pos": n_pos, "n_pages": n_pages}


def _paged_inputs(case, seed):
    g, H, KV, hd, page = _gen(seed), case["H"], case["KV"], case["hd"], case["page"]
    cached, new = _requests(case)
    kv = [c + x for c, x in zip(cached, new)]
    held = [_pages(n, page) for n in kv]
    n_pages, ld = sum(held) + 3, max(held) + 1
    ids = np.random.default_rng(seed * 31 + 11).permutation(n_pages).astype(np.int32)
    table = np.full((len(kv), ld), -1, np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = ids[at:at + h]
        at += h
    dtype = TYPES[case["type"]][1]
    q = _randn(g, sum(new), H * hd).view(-1, H, hd) + _common(hd)
    k = torch.empty(n_pages, KV, page, hd, device="cuda", dtype=dtype)
    v = torch.empty(n_pages, KV, page, hd, device="cuda", dtype=dtype)
    k.copy_(_randn(g, n_pages, KV, page, hd) + _common(hd))
    v.copy_(_randn(g, n_pages, KV, page, hd))
    start = np.concatenate([[0], np.cumsum(new)])
    return {"q": q.reshape(-1, H * hd), "k_pool": k, "v_pool": v, "table": torch.from_numpy(table).cuda(), "kv_len": _ints(kv),
            "row_start": _ints(start.tolist()), "seqs": len(kv), "rows": sum(new), "max_new": max(new), "max_kv": max(kv),
            "ld": ld, "n_pages": n_pages}


def _packed_inputs(case, seed):
    g, H, KV, hd, rows = _gen(seed), case["H"], case["KV"], case["hd"], case["rows"]
    lens = _prompts(case)
    dtype = TYPES[case["type"]][1]
    q = (_randn(g, rows, H, hd) + _common(hd)).view(rows, H * hd)
    k = (_randn(g, rows, KV, hd) + _common(hd)).to(dtype).view(rows, KV * hd)
    v = _randn(g, rows, KV * hd).to(dtype)
    start = np.concatenate([[0], np.cumsum(lens)])
    return {"q": q, "k": k, "v": v, "row_start": _ints(start.tolist()), "seqs": len(lens), "rows": rows}


def prepare(case, seed):
    kind = case["kind"]
    s = {"plan": _plan_inputs, "append": _append_inputs, "paged": _paged_inputs, "packed": _packed_inputs}[kind](case, seed)
    s["case"] = case
    if kind == "plan":
        n = s["seqs"]
        s["n_free_out"], s["kv_len"], s["row_start"] = (torch.zeros(m, dtype=torch.int32, device="cuda") for m in (1, n, n + 1))
        s["pos"] = torch.zeros(s["max_rows"], dtype=torch.int32, device="cuda")
        s["slot"] = torch.zeros(s["max_rows"], dtype=torch.int64, device="cuda")
        s["status"] = torch.zeros(4, dtype=torch.int32, device="cuda")
    elif kind == "append":
        s["q_out"] = torch.zeros(case["rows"], case["H"] * case["hd"], device="cuda")
    else:
        s["out"] = torch.zeros(s["rows"], case["H"] * case["hd"], device="cuda")
    if own:  # the handles and the workspace that a serving program keeps
        from edgeforge_amd import hip as H
        H.init()
        s["buf"] = {k: Buffer(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        if kind in ("append", "paged"):
            s["pool"] = H.PagePool(s["n_pages"], case["page"], case["KV"], case["hd"], TYPES[case["type"]][0],
                                   k=s["buf"]["k_pool"], v=s["buf"]["v_pool"])
        if kind == "paged":
            need = H.paged_attention_workspace_bytes(case["H"], s["pool"], s["seqs"], s["rows"], s["max_new"], s["max_kv"])
            s["ws"] = Buffer(torch.empty(max(need, 16), dtype=torch.uint8, device="cuda"))
        if kind == "packed":
            need = H.packed_attention_workspace_bytes(case["H"], case["KV"], case["hd"], TYPES[case["type"]][0], s["seqs"], s["rows"])
            s["ws"] = Buffer(torch.empty(max(need, 16), dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "paged": _own_paged, "packed": _own_packed}[kind](s)
    return {"plan": _plain_plan, "append": _plain_append, "paged": _plain_paged, "packed": _plain_packed}[kind](s)


PLAN_OUT = ("table", "free", "n_free_out", "kv_len", "row_start", "pos", "slot", "status")


def _own_plan(s):
    from edgeforge_amd import hip as H
    b = s["buf"]
    H.page_plan(b["cached"], b["new"], s["seqs"], s["case"]["page"], s["n_pages"], b["table"], s["ld"], b["free"], b["n_free"],
                b["n_free_out"], b["kv_len"], b["row_start"], b["pos"], b["slot"], s["max_rows"], b["status"])
    return [s[k] for k in PLAN_OUT]


def _own_append(s):
    from edgeforge_amd import hip as H
    c, b = s["case"], s["buf"]
    nq, nk = c["H"] * c["hd"], c["KV"] * c["hd"]
    ld, base = nq + 2 * nk, b["qkv"].ptr
    H.rope_append(base, ld, b["q_out"], nq, c["H"], base + 4 * nq, ld, base + 4 * (nq + nk), ld, c["rows"], b["pos"], b["cos"], b["sin"],
                  s["n_pos"], slot=b["slot"], pool=s["pool"])
    return [s["q_out"], s["k_pool"], s["v_pool"]]


def _own_paged(s):
    from edgeforge_amd import hip as H
    c, b = s["case"], s["buf"]
    nq = c["H"] * c["hd"]
    H.paged_attention(b["q"], nq, b["out"], nq, c["H"], s["pool"], b["table"], s["ld"], b["row_start"], b["kv_len"], s["seqs"], s["rows"],
                      s["max_new"], s["max_kv"], 1.0 / math.sqrt(c["hd"]), ws=s["ws"])
    return s["out"]


def _own_packed(s):
    from edgeforge_amd import hip as H
    c, b = s["case"], s["buf"]
    nq, nk = c["H"] * c["hd"], c["KV"] * c["hd"]
    H.packed_attention(b["q"], nq, b["k"], nk, b["v"], nk, TYPES[c["type"]][0], b["out"], nq, c["H"], c["KV"], c["hd"], b["row_start"],
                       s["seqs"], s["rows"], 1.0 / math.sqrt(c["hd"]), ws=s["ws"])
    return s["out"]


# ---- the plain forms -----------------------------------------------------------------------------------
def _plain_plan(s):
    page, cached, new, table, free = s["case"]["page"], s["cached"].long(), s["new"].long(), s["table"], s["free"]
    ended = new < 0
    rows_of = new.clamp(min=0)
    held = (cached + page - 1) // page
    total = torch.where(ended, 0, cached + rows_of)
    take = torch.where(ended, 0, (total + page - 1) // page - held)
    give = torch.where(ended, held, 0)
    n0 = s["n_free"].long()[0]
    n1 = n0 + give.sum()
    missing = (take.sum() - n1).clamp(min=0)
    # the ended requests' pages, request by request, go on top of the free pages
    col = torch.arange(table.shape[1], device=table.device)
    given = ended[:, None] & (col < held[:, None])
    free[n0 + torch.arange(int(given.sum()), device=free.device)] = table[given]
    # the growing requests take from the top
    taken = (col >= held[:, None]) & (col < (held + take)[:, None])
    table[taken] = free[n1 - 1 - torch.arange(int(taken.sum()), device=free.device)]
    ends = torch.cumsum(rows_of, 0)
    s["row_start"].copy_(torch.cat([torch.zeros(1, dtype=torch.long, device=ends.device), ends]))
    s["kv_len"].copy_(total)
    s["n_free_out"].copy_(n1 - take.sum())
    row = torch.arange(s["max_rows"], device=ends.device)
    real = row < ends[-1]
    who = torch.searchsorted(ends, row, right=True).clamp(max=len(ends) - 1)
    pos = torch.where(real, cached[who] + row - (ends - rows_of)[who], 0)
    s["pos"].copy_(pos)
    s["slot"].copy_(torch.where(real, table[who, pos // page].long() * page + pos % page, -1))
    s["status"].copy_(torch.stack([missing, (cached < 0).sum(), (ends[-1] - s["max_rows"]).clamp(min=0), torch.zeros_like(missing)]))
    return [s[k] for k in PLAN_OUT]


def _turn(x, c, s):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _plain_append(s):
    c = s["case"]
    nq, nk, page = c["H"] * c["hd"], c["KV"] * c["hd"], c["page"]
    q, k, v = s["qkv"].split([nq, nk, nk], -1)
    cos, sin = (s[n][s["pos"].long()][:, None, :] for n in ("cos", "sin"))
    s["q_out"].copy_(_turn(q.view(-1, c["H"], c["hd"]), cos, sin).view(-1, nq))
    at, off = s["slot"] // page, s["slot"] % page
    s["k_pool"][at, :, off] = _turn(k.view(-1, c["KV"], c["hd"]), cos, sin).to(s["k_pool"].dtype)
    s["v_pool"][at, :, off] = v.view(-1, c["KV"], c["hd"]).to(s["v_pool"].dtype)
    return [s["q_out"], s["k_pool"], s["v_pool"]]


def _attend(q, k, v, mask, scale):
    """q [..., G, n, hd], k / v [..., m, hd], mask [..., n, m] of what is seen: softmax(q k^T scale) v, zero where nothing is seen."""
    G, n, hd = q.shape[-3:]
    sc = torch.matmul(q.reshape(*q.shape[:-3], G * n, hd), k.transpose(-1, -2).contiguous()).view(*q.shape[:-1], k.shape[-2])
    sc *= scale
    sc.masked_fill_(~mask.unsqueeze(-3), -math.inf)
    top = sc.amax(-1, keepdim=True)
    sc -= torch.where(torch.isinf(top), 0.0, top)
    sc.exp_()
    total = sc.sum(-1, keepdim=True)
    out = torch.matmul(sc.view(*q.shape[:-3], G * n, -1), v).view(*q.shape[:-1], hd)
    return out / torch.where(total == 0, 1.0, total)


def _plain_paged(s):
    c = s["case"]
    H, KV, hd, page = c["H"], c["KV"], c["hd"], c["page"]
    G, n_new, n_kv = H // KV, s["max_new"], s["max_kv"]
    start, kv = s["row_start"].long(), s["kv_len"].long()
    new = start[1:] - start[:-1]
    dev = kv.device
    j = torch.arange(n_kv, device=dev)
    at = s["table"][:, j // page].clamp(min=0).long()  # [seqs, n_kv]
    k, v = (s[p][at, :, j % page].float().permute(0, 2, 1, 3).contiguous() for p in ("k_pool", "v_pool"))
    i = torch.arange(n_new, device=dev)
    row = (start[:-1, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"][row].view(-1, n_new, KV, G, hd).permute(0, 2, 3, 1, 4).contiguous()
    seen = j <= (kv - new)[:, None, None] + i[:, None]
    o = _attend(q, k, v, seen[:, None], 1.0 / math.sqrt(hd))  # [seqs, KV, G, n_new, hd]
    real = i < new[:, None]
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(-1, n_new, H * hd)[real])
    return s["out"]


def _plain_packed(s):
    c = s["case"]
    H, KV, hd, n = c["H"], c["KV"], c["hd"], s["rows"]
    row = torch.arange(n, device="cuda")
    who = torch.searchsorted(s["row_start"][1:].long(), row, right=True)
    seen = (who[:, None] == who) & (row <= row[:, None])
    q = s["q"].view(n, KV, H // KV, hd).permute(1, 2, 0, 3).contiguous()
    k, v = (s[p].view(n, KV, hd).float().permute(1, 0, 2).contiguous() for p in ("k", "v"))
    s["out"].copy_(_attend(q, k, v, seen, 1.0 / math.sqrt(hd)).permute(2, 0, 1, 3).reshape(n, H * hd))
    return s["out"]


# ---- what a pass cannot do without ---------------------------------------------------------------------
def _pairs(cached, new):
    """How many (new token, position that it sees) pairs there are."""
    return sum(x * c + x * (x + 1) // 2 for c, x in zip(cached, new))


def work(case):
    kind = case["kind"]
    if kind == "plan":
        cached, new = _requests(case)
        page, n, rows = case["page"], case["seqs"], sum(max(0, x) for x in new)
        moved = sum(_pages(c, page) if x < 0 else _pages(c + x, page) - _pages(c, page) for c, x in zip(cached, new))
        return {"bytes": 4 * (2 * n + 2 * n + 1) + 8 * moved + 4 * n + 12 * rows + 8, "flops": 8 * n + 6 * rows}
    H, KV, hd, size = case["H"], case["KV"], case["hd"], TYPES[case["type"]][2]
    if kind == "append":
        rows = case["rows"]
        return {"bytes": rows * (4 * hd * (2 * H + 2 * KV) + 2 * KV * hd * size + 4 * hd + 12), "flops": 3 * rows * (H + KV) * hd}
    if kind == "paged":
        cached, new = _requests(case)
        kv, rows = sum(c + x for c, x in zip(cached, new)), sum(new)
        return {"bytes": 2 * kv * KV * hd * size + 8 * rows * H * hd + 4 * _pages(kv, case["page"]), "flops": 4 * H * hd * _pairs(cached, new)}
    lens = _prompts(case)
    return {"bytes": case["rows"] * (8 * H * hd + 2 * KV * hd * size), "flops": 4 * H * hd * _pairs([0] * len(lens), lens)}


# ---- the same in 64 bits -------------------------------------------------------------------------------
def _softmax_rows(q, k, v, first, scale):
    """One head: row i of q sees k / v up to first + i.  Rows in blocks, to bound the scores' memory."""
    out = torch.empty_like(q)
    m = torch.arange(k.shape[0], device=q.device)
    for at in range(0, q.shape[0], 2048):
        part = q[at:at + 2048]
        sc = (part @ k.t()) * scale
        sc[m > first + at + torch.arange(part.shape[0], device=q.device)[:, None]] = -math.inf
        out[at:at + 2048] = torch.softmax(sc, -1) @ v
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None  # whole numbers
    H, KV, hd = case["H"], case["KV"], case["hd"]
    G, scale = H // KV, 1.0 / math.sqrt(hd)
    if kind == "append":
        s = _append_inputs(case, seed)
        rows, page, nq, nk = case["rows"], case["page"], H * hd, KV * hd
        z = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]  # a turn is a complex product
        x = s["qkv"].double()

        def turned(part, heads):
            p = part.reshape(rows, heads, 2, hd // 2)
            w = torch.complex(p[:, :, 0], p[:, :, 1]) * z
            return torch.stack([w.real, w.imag], 2).reshape(rows, heads, hd)

        out = [turned(x[:, :nq], H).reshape(rows, nq)]
        for pool, val in ((s["k_pool"], turned(x[:, nq:nq + nk], KV)), (s["v_pool"], x[:, nq + nk:].reshape(rows, KV, hd))):
            p = pool.double().permute(0, 2, 1, 3).reshape(-1, KV, hd)
            p[s["slot"]] = val
            out.append(p.view(-1, page, KV, hd).permute(0, 2, 1, 3).contiguous())
        return out
    if kind == "paged":
        s = _paged_inputs(case, seed)
        cached, new = _requests(case)
        out = torch.empty(s["rows"], H, hd, dtype=torch.float64, device="cuda")
        at = 0
        for b, (c, x) in enumerate(zip(cached, new)):
            pages = s["table"][b, :_pages(c + x, case["page"])].long()
            for h in range(KV):
                k, v = (s[p][pages, h].reshape(-1, hd)[:c + x].double() for p in ("k_pool", "v_pool"))
                for g in range(h * G, h * G + G):
                    out[at:at + x, g] = _softmax_rows(s["q"][at:at + x, g * hd:(g + 1) * hd].double(), k, v, c, scale)
            at += x
        return out.view(-1, H * hd)
    s = _packed_inputs(case, seed)
    out = torch.empty(case["rows"], H, hd, dtype=torch.float64, device="cuda")
    at = 0
    for x in _prompts(case):
        for h in range(KV):
            k, v = (s[p][at:at + x, h * hd:(h + 1) * hd].double() for p in ("k", "v"))
            for g in range(h * G, h * G + G):
                out[at:at + x, g] = _softmax_rows(s["q"][at:at + x, g * hd:(g + 1) * hd].double(), k, v, 0, scale)
        at += x
    return out.view(-1, H * hd)
