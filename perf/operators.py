"""Decoding many continuations of shared prompts: the operators a server needs beside its decode step.

Three operators, as the provider's users call them:

  prefix   attention of a batch whose sequences share the pages of a long prefix
           (forked sessions, one system prompt for many): every shared page is read
           once for all of the sequences' query rows, the rest of each window by itself
  verify   drafted tokens checked against the target's logits: accepted while
           u q(x) < p(x), then one token of the remaining distribution
  copy     pool pages copied in every layer: a fork's first write into a shared
           page, and the moves of a compaction

Where `own` is false `run` computes them in elementary torch operations, else it
makes the provider's calls on the same data.  Shapes: 32 q / 8 kv heads of 128
(Llama-3-8B), 16 / 4 of 128 (its tensor-parallel shard), 32 / 4 of 64
(TinyLlama-1.1B), vocabularies of 32000 and 128256.
"""
from __future__ import annotations

import ctypes as C
import math
import random

import numpy as np
import torch

own = False

PAGE = 16


def listed():
    return [
        # one prompt sampled a few times: the smallest shared batch, where latency counts
        {"name": "prefix_samples_b4", "op": "prefix", "heads": 32, "kv_heads": 4, "head_dim": 64, "kv": "bf16",
         "groups": 1, "sessions": 4, "rows": 1, "prefix": 517, "median": 40, "spread": 0.5, "limit": 256},
        # best-of-n over a long document
        {"name": "prefix_document_b16", "op": "prefix", "heads": 32, "kv_heads": 8, "head_dim": 128, "kv": "bf16",
         "groups": 1, "sessions": 16, "rows": 1, "prefix": 8000, "median": 150, "spread": 0.8, "limit": 1024},
        # a serving batch behind four system prompts, ragged conversations
        {"name": "prefix_system_b256", "op": "prefix", "heads": 32, "kv_heads": 8, "head_dim": 128, "kv": "bf16",
         "groups": 4, "sessions": 256, "rows": 1, "prefix": 2040, "median": 300, "spread": 1.0, "limit": 2048},
        # a verification step: the last token and four drafts of each session, on one worker of two
        {"name": "prefix_drafts_b48", "op": "prefix", "heads": 16, "kv_heads": 4, "head_dim": 128, "kv": "bf16",
         "groups": 1, "sessions": 48, "rows": 5, "prefix": 4011, "median": 200, "spread": 0.8, "limit": 1024},
        # pages in the reference's own precision
        {"name": "prefix_f32_b32", "op": "prefix", "heads": 32, "kv_heads": 4, "head_dim": 64, "kv": "f32",
         "groups": 1, "sessions": 32, "rows": 1, "prefix": 3001, "median": 200, "spread": 0.8, "limit": 1024},
        # one stream that drafts for itself
        {"name": "verify_one", "op": "verify", "sequences": 1, "drafts": 4, "ragged": False, "vocab": 32000,
         "temperature": 0.7, "certain": False, "greedy": 0},
        # a batch whose sessions drafted differently far, some of them greedy, with an odd vocabulary
        {"name": "verify_ragged_b33", "op": "verify", "sequences": 33, "drafts": 7, "ragged": True, "vocab": 50021,
         "temperature": 1.0, "certain": False, "greedy": 4},
        # a large batch with a draft model's probabilities
        {"name": "verify_b64", "op": "verify", "sequences": 64, "drafts": 4, "ragged": False, "vocab": 128256,
         "temperature": 0.8, "certain": False, "greedy": 0},
        # drafts looked up in the prompt: no probabilities, the draft was certain
        {"name": "verify_lookup_b48", "op": "verify", "sequences": 48, "drafts": 5, "ragged": True, "vocab": 128256,
         "temperature": 1.0, "certain": True, "greedy": 0},
        # the first step after a 16-way fork: every new session's last page
        {"name": "copy_fork_15", "op": "copy", "layers": 22, "kv_heads": 4, "head_dim": 64, "kv": "bf16", "pages": 15,
         "pool": 400},
        # compaction of a pool after many sessions have left
        {"name": "copy_compact_1025", "op": "copy", "layers": 32, "kv_heads": 8, "head_dim": 128, "kv": "bf16",
         "pages": 1025, "pool": 2300},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["prefix", "prefix", "verify", "copy"])
    if op == "prefix":
        d, heads, kv_heads = rng.choice([(128, 32, 8), (64, 32, 4), (128, 16, 4)])
        groups = rng.choice([1, 1, 2, 4])
        rows = rng.choice([1, 1, 1, 2, 5])
        sessions = groups * _log_int(rng, 2, 240 // rows // groups)
        return {"op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": d, "kv": rng.choice(["bf16", "bf16", "f32"]),
                "groups": groups, "sessions": sessions, "rows": rows, "prefix": _log_int(rng, 150, 6000 // groups),
                "median": _log_int(rng, 10, 300), "spread": round(rng.uniform(0.2, 1.0), 2), "limit": 1024}
    if op == "verify":
        drafts = rng.randint(1, 7)
        return {"op": op, "sequences": _log_int(rng, 1, 300 // (drafts + 1)), "drafts": drafts,
                "ragged": rng.random() < 0.5, "vocab": rng.choice([32000, 128256, _log_int(rng, 1000, 120000)]),
                "temperature": round(rng.uniform(0.5, 1.2), 2), "certain": rng.random() < 0.3,
                "greedy": rng.choice([0, 0, 1, 3])}
    d, kv_heads = rng.choice([(128, 8), (64, 4), (128, 4), (80, 4)])
    pages = _log_int(rng, 1, 600)
    return {"op": op, "layers": rng.randint(1, 32), "kv_heads": kv_heads, "head_dim": d,
            "kv": rng.choice(["bf16", "bf16", "f32"]), "pages": pages, "pool": 2 * pages + rng.randint(1, 100)}


# ------------------------------------------------------------------ inputs
def _gen(seed, *salt):
    x = int(seed) & 0xFFFFFFFF
    for s in salt:
        x = (x * 1000003 + int(s) + 0x9E3779B9) & 0x7FFFFFFFFFFF
    return torch.Generator(device="cuda").manual_seed(x)


def _rng(seed, salt):
    return np.random.default_rng([int(seed) & 0xFFFFFFFF, salt])


def _dtype(case):
    return torch.bfloat16 if case["kv"] == "bf16" else torch.float32


class State:
    """What a program has in hand: tensors, the pages' tables, and where the provider runs its context and plan."""

    ctx = staged = None

    def close(self):
        if self.ctx is not None and self.ctx.h:
            if self.staged:
                self.ctx.lib.zr_staged_destroy(self.staged)
            self.staged = None
            self.ctx.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PoolView:
    """A context's page pool as a tensor (the context lives as long as the view does)."""

    def __init__(self, state, shape, itemsize):
        self.state = state
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<i%d" % itemsize, "version": 2,
                                         "data": (state.ctx.lib.zr_kv_pool_data(state.ctx.h), False)}


def _lengths(case, seed):
    """Rows after the prefix of every sequence, this step's included."""
    z = _rng(seed, 5).standard_normal(case["sessions"])
    own_rows = np.round(case["median"] * np.exp(case["spread"] * z)).astype(np.int64)
    return np.clip(own_rows, case["rows"], case["limit"])


def _window(case, seed):
    """The pages of a prefix batch: (full shared pages, tables [sessions, pages] int32, rows past the shared pages [sessions])."""
    lens = _lengths(case, seed)
    n, g = case["sessions"], case["groups"]
    shared = case["prefix"] // PAGE
    tail = lens + case["prefix"] % PAGE  # a fork has its own copy of the prefix's last, partial page
    tail_pages = -(-tail // PAGE)
    total = g * shared + int(tail_pages.sum())
    # a pool that has served a while hands out its pages in no order
    order = _rng(seed, 9).permutation(total).astype(np.int32)
    tables = np.zeros((n, shared + int(tail_pages.max())), np.int32)
    tables[:, :shared] = np.repeat(order[:g * shared].reshape(g, shared), n // g, 0)
    at = g * shared + np.concatenate([[0], np.cumsum(tail_pages)[:-1]])
    for i in range(n):
        tables[i, shared:shared + tail_pages[i]] = order[at[i]:at[i] + tail_pages[i]]
    return shared, tables, tail, total


def _pages(case, seed, total):
    """K and V of every page, [2, pages, 16, kv_heads, head_dim] in the pool's type."""
    shape = (2, total, PAGE, case["kv_heads"], case["head_dim"])
    return torch.randn(shape, generator=_gen(seed, 23), device="cuda").to(_dtype(case))


def _queries(case, seed):
    shape = (case["sessions"] * case["rows"], case["heads"] * case["head_dim"])
    return torch.randn(shape, generator=_gen(seed, 31), device="cuda") * 1.3


def _context(case, layers, pages, seqs, rows, table):
    from mesh_amd import DeviceContext, ModelGeometry

    heads = case.get("heads", case["kv_heads"])
    g = ModelGeometry(hidden=heads * case["head_dim"], num_heads=heads, num_kv_heads=case["kv_heads"],
                      num_layers=layers, vocab=32, ffn=64)
    ctx = DeviceContext(g, kv_dtype=case["kv"], max_tokens=rows, max_seqs=seqs, max_pages_per_seq=table,
                        split_activations=True)
    ctx.create_kv_pool(pages)
    return ctx


def _prepare_prefix(case, seed):
    s = State()
    shared, tables, tail, total = _window(case, seed)
    n, r = case["sessions"], case["rows"]
    pages = _pages(case, seed, total)
    s.q = _queries(case, seed)
    s.groups, s.n, s.r, s.shared = case["groups"], n, r, shared
    s.heads, s.kvh, s.d = case["heads"], case["kv_heads"], case["head_dim"]
    if own:
        from mesh_amd import _lib

        s.ctx = ctx = _context(case, 1, total, n, n * r, tables.shape[1])
        # the pages' rows through the snapshot scatter, one window over the whole pool
        whole = np.arange(total, dtype=np.int32)
        rows = pages.float().reshape(2, total * PAGE, -1).contiguous()
        torch.cuda.synchronize()
        ctx.check(ctx.lib.zr_kv_scatter(ctx.h, whole.ctypes.data_as(_lib.c_int_p), total, 0, 0, total * PAGE,
                                        C.cast(rows[0].data_ptr(), _lib.c_f32_p),
                                        C.cast(rows[1].data_ptr(), _lib.c_f32_p)))
        ints = [np.full(n, r, np.int32), (shared * PAGE + tail - r).astype(np.int32),
                (shared * PAGE + tail - r).astype(np.int32), np.zeros(n, np.int32), np.ascontiguousarray(tables)]
        ip = [a.ctypes.data_as(_lib.c_int_p) for a in ints]
        mb = _lib.Microbatch(n, ip[0], ip[1], ip[2], ip[3], ip[4], tables.shape[1], None)
        st = C.c_void_p()
        ctx.check(ctx.lib.zr_stage(ctx.h, C.byref(mb), C.byref(st)))
        s.staged = st.value
        s.out = torch.zeros_like(s.q)
    else:
        s.pages = pages
        s.prefix_table = torch.from_numpy(tables[::n // case["groups"], :shared].astype(np.int64)).cuda()
        s.tail_table = torch.from_numpy(tables[:, shared:].astype(np.int64)).cuda()
        s.tail = torch.from_numpy(tail).cuda()
    torch.cuda.synchronize()
    return s


def _draft_lengths(case, seed):
    n, k = case["sequences"], case["drafts"]
    return _rng(seed, 13).integers(0, k + 1, n).astype(np.int32) if case["ragged"] else np.full(n, k, np.int32)


def _prepare_verify(case, seed):
    s = State()
    n, k, vocab = case["sequences"], case["drafts"], case["vocab"]
    lens = _draft_lengths(case, seed)
    nd, rows = int(lens.sum()), int(lens.sum()) + n
    s.n, s.k, s.vocab, s.certain = n, k, vocab, case["certain"]
    s.temps = np.full(n, case["temperature"], np.float32)
    if case["greedy"]:
        s.temps[::case["greedy"]] = 0.0
    s.lens = lens
    s.logits = torch.randn((rows, vocab), generator=_gen(seed, 41), device="cuda") * 3.0
    first = np.concatenate([[0], np.cumsum(lens + 1)[:-1]])
    at = np.concatenate([[0], np.cumsum(lens)[:-1]])
    # a draft model's logits are near the target's; drafts are sampled from its probabilities
    draft_rows = torch.from_numpy(np.concatenate([f + np.arange(m) for f, m in zip(first, lens)]).astype(np.int64)).cuda()
    t = torch.from_numpy(np.repeat(np.maximum(s.temps, 0.05), lens)).cuda()
    noise = torch.randn((nd, vocab), generator=_gen(seed, 43), device="cuda")
    probs = torch.softmax((s.logits[draft_rows] + noise * 0.7) / t[:, None], -1)
    race = torch.empty((nd, vocab), device="cuda").exponential_(generator=_gen(seed, 47))
    s.drafts = (probs / race).argmax(-1).to(torch.int32) if nd else torch.zeros(0, dtype=torch.int32, device="cuda")
    s.probs = None if case["certain"] else probs.contiguous()
    s.u = torch.rand(rows, generator=_gen(seed, 53), device="cuda")
    if own:
        from mesh_amd import DeviceContext, ModelGeometry

        s.ctx = DeviceContext(ModelGeometry(64, 1, 1, 1, 32, 64), max_tokens=1, max_seqs=1, max_pages_per_seq=1)
        s.tokens = torch.zeros((n, k + 1), dtype=torch.int32, device="cuda")
        s.accepted = torch.zeros(n, dtype=torch.int32, device="cuda")
    else:
        dev = lambda a: torch.from_numpy(np.asarray(a, np.int64)).cuda()  # noqa: E731
        s.t_rows = torch.from_numpy(np.repeat(s.temps, lens + 1).astype(np.float64)).cuda()
        s.greedy = torch.from_numpy(s.temps <= 0).cuda()
        s.len_d, s.first_d, s.at_d = dev(lens), dev(first), dev(at)
    torch.cuda.synchronize()
    return s


def _prepare_copy(case, seed):
    s = State()
    item = 2 if case["kv"] == "bf16" else 4
    shape = (case["layers"], case["pool"], 2 * case["kv_heads"] * case["head_dim"] * PAGE)
    kind = torch.int16 if item == 2 else torch.int32
    pool = torch.randint(-(1 << 15), 1 << 15, shape, generator=_gen(seed, 61), device="cuda", dtype=kind)
    n = case["pages"]
    # the lowest pages are free and take pages from all over the rest
    s.dst = _rng(seed, 17).permutation(n).astype(np.int32)
    s.src = (n + _rng(seed, 19).permutation(case["pool"] - n)[:n]).astype(np.int32)
    s.pages = n
    if own:
        s.ctx = _context(case, case["layers"], case["pool"], 1, 1, 1)
        # (no reference back to the state on the state: the view alone keeps it)
        torch.as_tensor(PoolView(s, shape, item), device="cuda").copy_(pool)
        s.shape, s.item = shape, item
    else:
        s.pool = pool
        s.dst_d, s.src_d = (torch.from_numpy(a.astype(np.int64)).cuda() for a in (s.dst, s.src))
    torch.cuda.synchronize()
    return s


def prepare(case, seed):
    s = {"prefix": _prepare_prefix, "verify": _prepare_verify, "copy": _prepare_copy}[case["op"]](case, seed)
    s.op = case["op"]
    return s


# ------------------------------------------------------------- one pass
def _plain_prefix(s):
    g, n, r, d, kvh = s.groups, s.n, s.r, s.d, s.kvh
    m, gq = n // g, s.heads // s.kvh
    rows = s.shared * PAGE
    q = s.q.view(n, r, kvh, gq, d) * (1.0 / math.sqrt(d))
    # the prefix once for all of a group's rows: [g, kvh, m r gq, d] x [g, kvh, d, rows]
    kv = s.pages[:, s.prefix_table].float().view(2, g, rows, kvh, d)
    qp = q.view(g, m * r, kvh, gq, d).permute(0, 2, 1, 3, 4).reshape(g, kvh, m * r * gq, d)
    sp = torch.matmul(qp, kv[0].permute(0, 2, 3, 1).contiguous())
    # each sequence's own rows
    tmax = s.tail_table.shape[1] * PAGE
    kt = s.pages[:, s.tail_table].float().view(2, n, tmax, kvh, d)
    qt = q.permute(0, 2, 1, 3, 4).reshape(n, kvh, r * gq, d)
    stail = torch.matmul(qt, kt[0].permute(0, 2, 3, 1).contiguous()).view(n, kvh, r, gq, tmax)
    seen = s.tail[:, None] - r + 1 + torch.arange(r, device="cuda")
    hidden = torch.arange(tmax, device="cuda")[None, None, :] >= seen[:, :, None]
    stail = stail.masked_fill(hidden[:, None, :, None, :], -math.inf)
    sp = sp.view(g, kvh, m, r, gq, rows).permute(0, 2, 1, 3, 4, 5).reshape(n, kvh, r, gq, rows)
    top = torch.maximum(sp.amax(-1), stail.amax(-1))[..., None] if rows else stail.amax(-1)[..., None]
    pp, pt = torch.exp(sp - top), torch.exp(stail - top)
    total = pp.sum(-1) + pt.sum(-1)
    pg = pp.view(g, m, kvh, r, gq, rows).permute(0, 2, 1, 3, 4, 5).reshape(g, kvh, m * r * gq, rows)
    op = torch.matmul(pg, kv[1].permute(0, 2, 1, 3).contiguous())
    op = op.view(g, kvh, m, r, gq, d).permute(0, 2, 1, 3, 4, 5).reshape(n, kvh, r, gq, d)
    ot = torch.matmul(pt.view(n, kvh, r * gq, tmax), kt[1].permute(0, 2, 1, 3).contiguous()).view(n, kvh, r, gq, d)
    return ((op + ot) / total[..., None]).permute(0, 2, 1, 3, 4).reshape(n * r, s.heads * d)


def _plain_verify(s):
    n, k = s.n, s.k
    # in 64 bits: a token changes where two cumulative sums of a vocabulary's probabilities change places
    x = s.logits.double() / torch.where(s.t_rows > 0, s.t_rows, 1.0)[:, None]
    best = s.logits.argmax(-1)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    step = torch.arange(k, device="cuda")
    valid = step[None, :] < s.len_d[:, None]
    row = torch.where(valid, s.first_d[:, None] + step, 0)
    if s.drafts.numel():
        at = torch.where(valid, s.at_d[:, None] + step, 0)
        x_d = s.drafts.long()[at]
        q_x = 1.0 if s.certain else s.probs[at, x_d].double()
        ok = torch.where(s.greedy[:, None], best[row] == x_d, s.u[row].double() * q_x < p[row, x_d])
    else:
        x_d, ok = torch.zeros_like(row), torch.zeros_like(valid)
    accepted = torch.cumprod((ok & valid).long(), 1).sum(1)
    erow = s.first_d + accepted
    pe, left = p[erow], accepted < s.len_d
    rest = pe
    if s.drafts.numel():
        eat = torch.where(left, s.at_d + accepted, 0)
        qe = torch.nn.functional.one_hot(s.drafts.long()[eat], s.vocab).double() if s.certain else s.probs[eat].double()
        rest = torch.where(left[:, None], (pe - qe).clamp_min(0.0), pe)
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, pe)
    cum = torch.cumsum(rest, -1)
    target = s.u[s.first_d + s.len_d].double() * cum[:, -1]
    token = (cum <= target[:, None]).sum(-1).clamp_max(s.vocab - 1)
    token = torch.where(s.greedy, best[erow], token)
    place = torch.arange(k + 1, device="cuda")[None, :]
    padded = torch.cat([x_d, x_d.new_zeros((n, 1))], 1)
    out = torch.where(place < accepted[:, None], padded, torch.where(place == accepted[:, None], token[:, None], -1))
    return {"tokens": out.to(torch.int32), "accepted": accepted.to(torch.int32)}


def run(s):
    if own:
        from mesh_amd import _lib

        lib, ctx = s.ctx.lib, s.ctx
        if s.op == "prefix":
            ctx.check(lib.zr_attention_async(ctx.h, s.staged, 0, s.q.data_ptr(), s.out.data_ptr()))
            return s.out
        if s.op == "verify":
            vb = _lib.VerifyBatch(s.n, s.lens.ctypes.data_as(_lib.c_int_p), s.drafts.data_ptr(),
                                  None if s.probs is None else s.probs.data_ptr(),
                                  s.temps.ctypes.data_as(_lib.c_f32_p), s.u.data_ptr())
            ctx.check(lib.zr_verify_async(ctx.h, s.logits.data_ptr(), s.vocab, C.byref(vb), s.tokens.data_ptr(),
                                          s.k + 1, s.accepted.data_ptr()))
            return {"tokens": s.tokens, "accepted": s.accepted}
        ctx.check(lib.zr_kv_copy_pages_async(ctx.h, s.src.ctypes.data_as(_lib.c_int_p),
                                             s.dst.ctypes.data_as(_lib.c_int_p), s.pages))
        return torch.as_tensor(PoolView(s, s.shape, s.item), device="cuda")[:, :s.pages]
    if s.op == "prefix":
        return _plain_prefix(s)
    if s.op == "verify":
        return _plain_verify(s)
    s.pool[:, s.dst_d] = s.pool[:, s.src_d]
    return s.pool[:, :s.pages]


# ------------------------------------------------------------- what it needs
def work(case):
    if case["op"] == "copy":
        item = 2 if case["kv"] == "bf16" else 4
        page = 2 * case["kv_heads"] * case["head_dim"] * PAGE * item
        return {"bytes": 2.0 * case["layers"] * case["pages"] * page, "flops": 0.0}
    if case["op"] == "verify":
        lens = _draft_lengths(case, 1)
        rows = float(lens.sum() + len(lens))
        # every row's logits; of the draft's probabilities one row per sequence (the first rejected draft's)
        q_rows = 0.0 if case["certain"] else float((lens > 0).sum())
        return {"bytes": 4.0 * case["vocab"] * (rows + q_rows), "flops": 0.0}
    lens = _lengths(case, 1).astype(np.float64)
    r, width = case["rows"], case["kv_heads"] * case["head_dim"]
    item = 2 if case["kv"] == "bf16" else 4
    kv = (case["groups"] * case["prefix"] + lens.sum()) * 2.0 * width * item
    io = 2.0 * 4.0 * case["sessions"] * r * case["heads"] * case["head_dim"]
    seen = (r * (case["prefix"] + lens) - r * (r - 1) / 2.0).sum()
    return {"bytes": kv + io, "flops": 4.0 * case["heads"] * case["head_dim"] * float(seen)}


# ----------------------------------------------------------- 64-bit restatement
def exact(case, seed):
    if case["op"] != "prefix":
        return None  # tokens and copied bits
    _, tables, tail, total = _window(case, seed)
    pages, q = _pages(case, seed, total), _queries(case, seed)
    d, kvh, r = case["head_dim"], case["kv_heads"], case["rows"]
    gq = case["heads"] // kvh
    out = []
    for i in range(case["sessions"]):
        rows = case["prefix"] // PAGE * PAGE + int(tail[i])
        table = torch.from_numpy(tables[i, :-(-rows // PAGE)].astype(np.int64)).cuda()
        k, v = (pages[j, table].reshape(-1, kvh, d)[:rows].double().repeat_interleave(gq, 1) for j in (0, 1))
        qi = q[i * r:(i + 1) * r].double().view(r, kvh * gq, d)
        w = torch.matmul(qi.transpose(0, 1).contiguous(), k.permute(1, 2, 0).contiguous()) / math.sqrt(d)
        for j in range(r):
            w[:, j, rows - r + 1 + j:] = -math.inf
        w = torch.softmax(w, -1)
        out.append(torch.matmul(w, v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(r, -1))
    return torch.cat(out)
