"""Forked sessions that decode with drafts: one prompt, forks of it, verified steps
over their shared pages, rejected rows dropped, and ordinary steps after them."""
import ctypes as C

import numpy as np
import pytest

from mesh_amd import BackendMicrobatchExecutor, DecodeMicrobatchRequest, DeviceBuffer, DeviceContext, ModelGeometry
from mesh_amd import VerifyMicrobatchRequest as Request
from mesh_amd._lib import Microbatch, ZrError
from tests.gpu_util import i32p
from tests.test_gpu_fork_pages import model_context
from tests.test_gpu_verify import expect

pytestmark = pytest.mark.gpu
VOCAB = 512


def verify(requests, **kw):
    return [(o.tokens, o.accepted) for o in BackendMicrobatchExecutor.verify_batch(requests, **kw)]


def greedy(b, token, steps):
    """The tokens that follow `token`, one step each, with the logits of every step."""
    tokens, logits = [], []
    for _ in range(steps):
        x = b.decode_step(token)
        token = int(np.argmax(x))
        tokens.append(token)
        logits.append(x)
    return tokens, logits


def margin(logits):
    two = np.sort(np.asarray(logits), axis=-1)[..., -2:]
    return float((two[..., 1] - two[..., 0]).min())


# A step of several rows and one of one row sum in other orders; a bf16 pool adds a tie of a new
# key or value (2^-8 of one element of one of 40 keys and more).  Greedy paths whose two largest
# logits are apart by more than that, 2e-3, have to be the same.
TIE = 2e-3


def distinct_start(ctx, prompt, steps, first=0):
    """A first token whose greedy continuation has no near tie (chosen on the one-row path alone)."""
    for token in range(first, VOCAB):
        b = ctx.new_backend()
        b.prefill(prompt)
        tokens, logits = greedy(b, token, steps)
        ok = margin(logits) > TIE
        b.close()
        if ok:
            return token, tokens
    raise AssertionError("no path without a tie")


@pytest.mark.parametrize("kv,heads,kv_heads,d", [("bf16", 4, 2, 64), ("f32", 4, 1, 64), ("bf16", 2, 2, 80),
                                                 ("bf16", 8, 2, 128)])
@pytest.mark.parametrize("rows", [40, 128, 300])
def test_forks_with_drafts_emit_the_greedy_path(kv, heads, kv_heads, d, rows):
    ctx = model_context(kv, heads, kv_heads, d, pages=400)
    rng = np.random.default_rng(rows + d)
    prompt = rng.integers(0, VOCAB, rows).tolist()
    parent = ctx.new_backend()
    parent.prefill(prompt)
    token, path = distinct_start(ctx, prompt, 24)
    forks = [parent] + [parent.fork() for _ in range(5)]
    done = [0] * 6
    last = [token] * 6
    for step in range(4):
        reqs, want = [], []
        for i, f in enumerate(forks):
            k = (i + step) % 4
            right = (2 * i + step) % 5  # this many drafts are right, the next one is not
            drafts = path[done[i]:done[i] + k]
            if right < k:
                drafts[right] = (drafts[right] + 1) % VOCAB
            a = min(right, k)
            reqs.append(Request(str(i), last[i], drafts, f))
            want.append((path[done[i]:done[i] + a + 1], a))
        assert verify(reqs) == want
        for i, (t, a) in enumerate(want):
            done[i] += a + 1
            last[i] = t[-1]
            assert forks[i].sequence_position() == rows + done[i] == forks[i].cache_seq_len()
    # ordinary steps go on from there, in eager and replayed microbatches
    for step in range(5):
        out = BackendMicrobatchExecutor.decode_step_batch(
            [DecodeMicrobatchRequest(str(i), last[i], f) for i, f in enumerate(forks)])
        for i, o in enumerate(out):
            assert o.sampled_token == path[done[i]]
            done[i] += 1
            last[i] = o.sampled_token
    # and every window holds the path's keys and values: those of a session that only ever stepped
    b = ctx.new_backend()
    b.prefill(prompt)
    greedy(b, token, 24)
    k0 = b.export_kv_cache()
    for i, f in enumerate(forks):
        k = f.export_kv_cache()
        n = rows + done[i]
        assert k.keys.shape[1] == n
        np.testing.assert_array_equal(k.keys[:, :rows], k0.keys[:, :rows])
        np.testing.assert_allclose(k.keys, k0.keys[:, :n], rtol=2.0 ** -7, atol=1e-3)
        np.testing.assert_allclose(k.values, k0.values[:, :n], rtol=2.0 ** -7, atol=1e-3)
    ctx.close()


@pytest.mark.parametrize("certain", [False, True])
def test_drawn_tokens_are_the_definitions_on_the_stepped_logits(certain):
    ctx = model_context("f32", 4, 2, 64)
    rng = np.random.default_rng(4)
    prompt = rng.integers(0, VOCAB, 70).tolist()
    parent = ctx.new_backend()
    parent.prefill(prompt)
    lens = [3, 0, 5, 1, 2]
    temps = [0.7, 1.0, 1.3, 0.0, 0.4]
    token = int(rng.integers(0, VOCAB))
    drafts, logits = [], []
    for k, t in zip(lens, temps):
        b = parent.fork()
        seq = [token]
        for i in range(k + 1):
            x = b.decode_step(seq[-1])
            logits.append(x)
            seq.append(int(np.argsort(-x)[rng.integers(0, 3)]))
        drafts.append(seq[1:k + 1])
        b.close()
    logits = np.array(logits)
    q = None
    if not certain:
        rows = [r for s in range(5) for r in range(sum(lens[:s]) + s, sum(lens[:s]) + s + lens[s])]
        x = logits[rows].astype(np.float64) * 1.5
        q = np.exp(x - x.max(1, keepdims=True))
        q = (q / q.sum(1, keepdims=True)).astype(np.float32)
    u = rng.random(len(logits)).astype(np.float32)
    want = expect(logits, drafts, temps, u, q)
    row = 0
    reqs = []
    for i, y in enumerate(drafts):
        reqs.append(Request(str(i), token, y, parent.fork(), temperature=temps[i], uniforms=u[row:row + len(y) + 1]))
        row += len(y) + 1
    assert verify(reqs, draft_probs=q) == list(zip(*want))
    # ... and the same from device memory, on other forks
    for r in reqs:
        r.backend = parent.fork()
    if q is not None:
        assert verify(reqs, draft_probs=DeviceBuffer.from_numpy(ctx, q)) == list(zip(*want))
    ctx.close()


def state(backends):
    return [(b.sequence_position(), b.cache_seq_len(), b.block_table()) for b in backends]


def test_refused_steps_change_nothing():
    ctx = model_context("bf16", 4, 2, 64, pages=16)
    rng = np.random.default_rng(2)
    a = ctx.new_backend()
    a.prefill(rng.integers(0, VOCAB, 47).tolist())
    small = ctx.new_backend(max_seq_len=50)
    small.prefill(rng.integers(0, VOCAB, 48).tolist())
    fresh = ctx.new_backend()
    both = [a, small]
    before, free = state(both), ctx.free_pages

    def refused(*requests, **kw):
        with pytest.raises(ZrError):
            verify(list(requests), **kw)
        assert state(both) == before and ctx.free_pages == free

    refused()
    refused(Request("w", 1, [2, 3], small))                         # the window would slide
    refused(Request("a", 1, [2, 3], a), Request("w", 1, [2, 3], small))
    refused(Request("a", 1, [2, 3], a), Request("f", 1, [2], fresh))  # not prefilled
    refused(Request("a", 1, [2, 3], a), Request("a", 1, [2], a))    # twice
    refused(Request("a", 1, [2] * 256, a))
    refused(Request("a", 1, [2] * 130, a))                          # more rows than the context takes
    refused(Request("a", 1, [VOCAB], a))                            # a token outside the vocabulary
    refused(Request("a", 1, [2, 3], a, temperature=0.5))            # no uniforms
    refused(Request("a", 1, [2, 3], a, temperature=0.5, uniforms=[0.1] * 2))
    refused(Request("a", 1, [2, 3], a, temperature=float("nan"), uniforms=[0.1] * 3))
    refused(Request("a", 1, [2, 3], a), draft_probs=np.zeros((1, VOCAB), np.float32))
    refused(Request("a", 1, [2, 3], a), draft_probs=np.zeros((3, VOCAB), np.float32))
    lens, toks = np.array([2], np.int32), np.array([1, 2, 3], np.uint32)
    t, u = np.zeros(1, np.float32), np.zeros(3, np.float32)
    out, acc = np.zeros(3, np.uint32), np.zeros(1, np.int32)
    arr = (C.c_void_p * 1)(a.h)

    def raw(p=arr, n=1, k=lens, y=toks, tt=t, uu=u, o=out, stride=3, c=acc):
        def at(x, ty):
            return None if x is None else x.ctypes.data_as(C.POINTER(ty))
        return ctx.lib.zrh_verify_batch(C.cast(p, C.POINTER(C.c_void_p)) if p else None, n, at(k, C.c_int),
                                        at(y, C.c_uint32), at(tt, C.c_float), at(uu, C.c_float), None,
                                        at(o, C.c_uint32), stride, at(c, C.c_int))

    for bad in (dict(p=None), dict(n=0), dict(n=-1), dict(k=None), dict(y=None), dict(tt=None), dict(uu=None),
                dict(o=None), dict(c=None), dict(stride=2), dict(k=np.array([-1], np.int32)),
                dict(p=(C.c_void_p * 1)(None))):
        assert raw(**bad) == -1
        assert state(both) == before and ctx.free_pages == free
    # the pool's last pages: a step that needs more of them than there are
    filler = ctx.new_backend()
    filler.prefill(rng.integers(0, VOCAB, 16 * free).tolist())
    assert ctx.free_pages == 0
    with pytest.raises(ZrError):
        verify([Request("w", 1, [], small), Request("a", 1, [2, 3], a)])
    assert state(both) == before
    assert raw(k=np.array([0], np.int32)) == 0 and acc[0] == 0  # one row: the last one of the page
    ctx.close()


def test_a_window_that_slides_takes_a_step_without_drafts():
    ctx = model_context("bf16", 4, 2, 64)
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, VOCAB, 50).tolist()
    a, b = ctx.new_backend(max_seq_len=50), ctx.new_backend(max_seq_len=50)
    a.prefill(prompt)
    b.prefill(prompt)
    for t in (3, 5, 7):
        want = int(np.argmax(b.decode_step(t)))
        assert verify([Request("a", t, [], a)]) == [([want], 0)]
    assert (a.cache_seq_len(), a.base_position(), a.sequence_position()) == (50, 3, 53)
    ctx.close()


def test_sampling_after_a_verification_needs_a_forward():
    ctx = model_context("bf16", 4, 2, 64)
    b = ctx.new_backend()
    b.prefill([1, 2, 3])
    one, seed, out = np.ones(1, np.float32), np.zeros(1, np.uint64), np.zeros(1, np.uint32)

    def sample():
        return ctx.lib.zr_sample_last_logits(ctx.h, 1, one.ctypes.data_as(C.POINTER(C.c_float)),
                                             one.ctypes.data_as(C.POINTER(C.c_float)),
                                             seed.ctypes.data_as(C.POINTER(C.c_uint64)),
                                             out.ctypes.data_as(C.POINTER(C.c_uint32)))
    for _ in range(12):  # eager, then replayed steps between the verified ones
        verify([Request("b", 4, [5, 6], b)])
        assert sample() == -1
        for _ in range(3):
            BackendMicrobatchExecutor.decode_step_batch([DecodeMicrobatchRequest("b", 4, b)])
            assert sample() == 0
    ctx.close()


def test_forward_refusals():
    """The device entry by itself; a vocabulary of 2^22: 128 rows are 2^29 logits, 129 too many."""
    g = ModelGeometry(64, 1, 1, 1, 1 << 22, 64)
    ctx = DeviceContext(g, max_tokens=256, max_seqs=2, max_pages_per_seq=16)
    ctx.create_kv_pool(16)
    f32, u32 = C.POINTER(C.c_float), C.POINTER(C.c_uint32)
    t, u = np.zeros(2, np.float32), np.zeros(256, np.float32)
    out, acc = np.zeros(2 * 256, np.uint32), np.zeros(2, np.int32)

    def call(rows, n=1, mb=True, temps=t, stride=256, tables=np.arange(16, dtype=np.int32)):
        ql, zero = np.array([rows] * n, np.int32), np.zeros(n, np.int32)
        toks = np.zeros(max(rows, 1) * n, np.uint32)
        m = Microbatch(n, i32p(ql), i32p(zero), i32p(zero), i32p(zero), i32p(tables), 16, toks.ctypes.data_as(u32))
        rc = ctx.lib.zr_forward_verify(ctx.h, C.byref(m) if mb else None, temps.ctypes.data_as(f32) if temps is not None
                                       else None, u.ctypes.data_as(f32), None, out.ctypes.data_as(u32), stride, i32p(acc))
        return rc, ctx.lib.zr_last_error(ctx.h).decode()

    assert call(129) == (-1, "verification of 129 rows of 4194304 logits: at most 2^29 logits a call")
    rc, why = call(128)
    assert rc != 0 and "weights not uploaded" in why
    assert call(0)[0] != 0 and call(257)[0] != 0 and call(1, n=0)[0] != 0 and call(1, n=3)[0] != 0
    assert call(4, temps=None)[0] == -1
    assert ctx.lib.zr_forward_verify(ctx.h, None, None, None, None, None, 1, None) == -1
    assert ctx.lib.zr_forward_verify(None, None, None, None, None, None, 1, None) == -1
    ctx.close()


@pytest.mark.parametrize("kv,kv_heads,d", [("f32", 1, 64), ("bf16", 2, 128)])
@pytest.mark.parametrize("seed", [0, 1])
def test_any_program_of_forks_steps_drafts_and_compactions(kv, kv_heads, d, seed):
    """Random calls; in the end every window holds the keys and values of its own tokens, as a session
    that was prefilled with them has them."""
    ctx = model_context(kv, 4, kv_heads, d, pages=220)
    rng = np.random.default_rng(seed)
    live = []  # [session, its tokens]

    def some(n=None):
        n = int(rng.integers(1, min(len(live), 12) + 1)) if n is None else n
        return [live[i] for i in rng.permutation(len(live))[:n]]

    for step in range(150):
        what = rng.choice(["new", "fork", "fork", "step", "step", "step", "verify", "verify", "chunk", "truncate", "close",
                           "compact"])
        if what == "new" or not live:
            if len(live) < 14:
                tokens = rng.integers(0, VOCAB, int(rng.integers(1, 120))).tolist()
                b = ctx.new_backend()
                b.prefill(tokens)
                live.append([b, tokens])
        elif what == "fork" and len(live) < 14:
            b, tokens = some(1)[0]
            live.append([b.fork(), list(tokens)])
        elif what == "step":
            part = some()
            for _ in range(int(rng.integers(1, 7))):  # (as many as replay)
                toks = rng.integers(0, VOCAB, len(part)).tolist()
                BackendMicrobatchExecutor.decode_step_batch(
                    [DecodeMicrobatchRequest("", t, s[0]) for t, s in zip(toks, part)])
                for t, s in zip(toks, part):
                    s[1].append(t)
        elif what == "verify":
            part = some(min(len(live), 10))
            reqs = []
            for s in part:
                k = int(rng.integers(0, 6))
                reqs.append(Request("", int(rng.integers(0, VOCAB)), rng.integers(0, VOCAB, k).tolist(), s[0],
                                    temperature=8.0, uniforms=(rng.random(k + 1) * 1e-3).tolist()))
            for s, r, (tokens, a) in zip(part, reqs, verify(reqs)):
                assert tokens[:a] == r.drafts[:a] and len(tokens) == a + 1
                s[1] += [r.token] + r.drafts[:a]
        elif what == "chunk":
            part = some(min(len(live), 4))
            chunks = [rng.integers(0, VOCAB, int(rng.integers(1, 32))).tolist() for _ in part]
            BackendMicrobatchExecutor.forward_mixed([s[0] for s in part], chunks, want_logits=False)
            for c, s in zip(chunks, part):
                s[1] += c
        elif what == "truncate":
            s = some(1)[0]
            n = int(rng.integers(0, min(len(s[1]), 40)))
            s[0].truncate(n)
            del s[1][len(s[1]) - n:]
        elif what == "close" and len(live) > 3:
            s = some(1)[0]
            live.remove(s)
            s[0].close()
        elif what == "compact":
            ctx.compact_pages()
        while ctx.free_pages < 60:
            live.pop(int(rng.integers(0, len(live))))[0].close()
        for b, tokens in live:
            assert b.sequence_position() == b.cache_seq_len() == len(tokens)
    for b, tokens in live:
        got = b.export_kv_cache()
        own = ctx.new_backend()
        own.prefill(tokens)
        want = own.export_kv_cache()
        own.close()
        # Other batches form their sums in other orders.  Activations enter the products as hi + lo
        # bf16, 16 bits: where the last f32 bits differ, lo may fall a step apart, 2^-16 of x.  A key
        # of layer 1 sums 256 of them (x of order 1, w of 0.05: 16 * 0.05 * 2^-16 = 1.2e-5 in the
        # mean square if all did), and what reached x through layer 0's three products is of the same
        # size, so six deviations are 1e-4 and a little.  A bf16 pool adds a step of a value on a tie,
        # 2^-7 of it at most, and its weight in the layer above.  A wrong row is off by order 1.
        rtol, atol = (2.0 ** -7, 2e-3) if kv == "bf16" else (0, 2e-4)
        np.testing.assert_allclose(got.keys, want.keys, rtol=rtol, atol=atol)
        np.testing.assert_allclose(got.values, want.values, rtol=rtol, atol=atol)
    ctx.close()
