"""Draft verification against a restatement of its definition in 64 bits, row by
row.  Tokens and counts are whole numbers and have to be equal: the drawn row's
weights and sums are held in f64 on both sides, so a random uniform meets a border
between two tokens with a chance of about 1e-9; a draft's test has one border, and
sums Z in f32 (a few 2^-24 of themselves) move it by 1e-6 of a probability at most."""
import ctypes as C

import numpy as np
import pytest

from mesh_amd import DeviceBuffer, DeviceContext, ModelGeometry, _lib, verify_device
from mesh_amd._lib import ZrError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = DeviceContext(ModelGeometry(64, 1, 1, 1, 32, 64), max_tokens=1, max_seqs=1, max_pages_per_seq=1)
    yield c
    c.close()


def weights(x, t):
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    m = x.max()
    if m == -np.inf:
        return np.zeros(x.size)
    with np.errstate(all="ignore"):
        w = np.exp((x - m) / np.float64(t))
    return np.where(x == m, 1.0, np.where(np.isnan(w), 0.0, w))


def expect(logits, drafts, temps, u, probs=None):
    tokens, accepted, row, d = [], [], 0, 0
    cols = logits.shape[1]
    for y, t in zip(drafts, np.asarray(temps, np.float32)):
        k, out = len(y), []
        for i in range(k):
            x = logits[row + i]
            if t <= 0:
                ok = y[i] == np.argmax(np.where(np.isnan(x), -np.inf, x))
            else:
                w = weights(x, t)
                q = 1.0 if probs is None else (max(float(probs[d + i, y[i]]), 0.0) if y[i] < cols else 0.0)
                ok = y[i] < cols and np.float64(u[row + i]) * q * w.sum() < w[y[i]]
            if not ok:
                break
            out.append(int(y[i]))
        a = len(out)
        x = logits[row + a]
        w = weights(x, t if t > 0 else 1.0)
        if t <= 0 or w.sum() == 0:
            token = int(np.argmax(np.where(np.isnan(x), -np.inf, x)))
        else:
            rest = w
            if a < k and probs is not None:
                rest = np.maximum(w - np.maximum(probs[d + a].astype(np.float64), 0.0) * w.sum(), 0.0)
            elif a < k and y[a] < cols:
                rest = w.copy()
                rest[y[a]] = 0.0
            if rest.sum() <= 0:
                rest = w
            cum = np.cumsum(rest)
            hit = np.flatnonzero((rest > 0) & (cum > np.float64(u[row + k]) * cum[-1]))
            token = int(hit[0]) if hit.size else int(np.flatnonzero(rest > 0)[-1])
        tokens.append(out + [token])
        accepted.append(a)
        row += k + 1
        d += k
    return tokens, accepted


def problem(rng, cols, lens, temps, certain, spread=2.0, near=0.5):
    rows = sum(lens) + len(lens)
    logits = (rng.standard_normal((rows, cols)) * spread).astype(np.float32)
    drafts, probs, row = [], [], 0
    for k, t in zip(lens, temps):
        y = []
        for i in range(k):
            x = logits[row + i].astype(np.float64) + near * rng.standard_normal(cols)
            q = weights(x, max(t, 0.05))
            q = (q / q.sum()).astype(np.float32)
            y.append(int(rng.choice(cols, p=q.astype(np.float64) / q.astype(np.float64).sum())))
            probs.append(q)
        drafts.append(y)
        row += k + 1
    u = rng.random(rows, dtype=np.float32)
    q = None if certain else np.array(probs, np.float32).reshape(-1, cols)
    return logits, drafts, u, q


# a chunk is 1024 to 8192 columns; rows whose width is no multiple of four are read by single words
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("cols", [1, 2, 3, 64, 1000, 1023, 1024, 1025, 5000, 32000, 50021])
def test_matches_the_definition(ctx, cols, certain):
    rng = np.random.default_rng(cols)
    for lens in ([4], [0], [0, 3, 1, 7, 2], [1] * 9):
        temps = rng.choice([0.0, 0.5, 1.0, 1.3], len(lens)).astype(np.float32)
        logits, drafts, u, q = problem(rng, cols, lens, temps, certain)
        assert verify_device(ctx, logits, drafts, temps, u, q) == expect(logits, drafts, temps, u, q)


def test_many_sequences_go_in_several_launches(ctx):
    rng = np.random.default_rng(7)
    lens = rng.integers(0, 4, 600).tolist()
    temps = rng.choice([0.0, 0.8], 600).astype(np.float32)
    for certain in (False, True):
        logits, drafts, u, q = problem(rng, 37, lens, temps, certain)
        assert verify_device(ctx, logits, drafts, temps, u, q) == expect(logits, drafts, temps, u, q)


def test_largest_draft_and_large_chunks(ctx):
    rng = np.random.default_rng(8)
    # 256 rows and more fill the chip: chunks of 8192 columns
    logits, drafts, u, q = problem(rng, 9001, [255, 3], [0.3, 0.3], False, near=0.02)
    got = verify_device(ctx, logits, drafts, [0.3, 0.3], u, q)
    assert got == expect(logits, drafts, [0.3, 0.3], u, q)
    # every draft accepted: u = 0
    got = verify_device(ctx, logits, drafts, [0.3, 0.3], np.zeros_like(u), q)
    assert got[1] == [255, 3] and got == expect(logits, drafts, [0.3, 0.3], np.zeros_like(u), q)


@pytest.mark.parametrize("u_last", [0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1.0, 7.0, -1.0])
@pytest.mark.parametrize("certain", [False, True])
def test_uniforms_at_and_beyond_their_ends(ctx, u_last, certain):
    rng = np.random.default_rng(11)
    logits, drafts, u, q = problem(rng, 3000, [2, 0, 3], [1.0, 1.0, 1.0], certain)
    logits[:, :50] = -np.inf  # the first columns weigh nothing
    logits[:, -50:] = -np.inf
    for fill in (u_last, np.nan):
        u[[2, 3, 7]] = fill
        got = verify_device(ctx, logits, drafts, [1.0] * 3, u, q)
        assert got == expect(logits, drafts, [1.0] * 3, u, q)
        assert all(50 <= t[-1] < 2950 for t in got[0])


def test_logits_that_are_not_finite(ctx):
    rng = np.random.default_rng(12)
    cols = 2500
    logits, drafts, u, q = problem(rng, cols, [1, 1, 1, 1, 0, 2], [1.0, 1.0, 0.0, 1.0, 1.0, 0.5], False)
    logits[0, ::3] = np.nan
    logits[1, ::2] = -np.inf
    logits[2, :] = -np.inf       # no finite logit: the draft is refused, token 0
    logits[4, [7, 1900]] = np.inf  # (greedy) the first of two
    logits[6, [5, 2200]] = np.inf  # all weight on two columns
    logits[8, :] = np.nan
    logits[9, :] = -np.inf
    temps = [1.0, 1.0, 0.0, 1.0, 1.0, 0.5]
    got = verify_device(ctx, logits, drafts, temps, u, q)
    assert got == expect(logits, drafts, temps, u, q)
    assert got[0][1][-1:] == [0] and got[0][4] == [0]


def test_drafts_and_probabilities_out_of_range(ctx):
    rng = np.random.default_rng(13)
    logits, drafts, u, q = problem(rng, 400, [2, 2, 2], [1.0, 1.0, 0.0], False)
    drafts[0][0] = 400           # outside the columns: refused, the rest is p less q
    drafts[1][1] = 0xffffffff
    drafts[2][0] = 400
    u[3] = 0.0                   # ... after an accepted one
    for probs in (q, None):
        got = verify_device(ctx, logits, drafts, [1.0, 1.0, 0.0], u, probs)
        assert got == expect(logits, drafts, [1.0, 1.0, 0.0], u, probs)
        assert got[1][0] == 0 and got[1][2] == 0
    q[:, ::2] = -1.0             # below 0 and not a number: probability 0
    q[:, 1::5] = np.nan
    clean = np.where(np.isnan(q), 0.0, q)
    drafts[0][0] = 3
    assert verify_device(ctx, logits, drafts, [1.0, 1.0, 0.0], u, q) == expect(logits, drafts, [1.0, 1.0, 0.0], u, clean)


@pytest.mark.parametrize("t", [1e-30, 1e-3, 1e30, np.inf])
def test_extreme_temperatures(ctx, t):
    rng = np.random.default_rng(14)
    logits, drafts, u, q = problem(rng, 1500, [2, 2], [1.0, 1.0], False)
    logits[3, 10] = -np.inf
    assert verify_device(ctx, logits, drafts, [t, t], u, q) == expect(logits, drafts, [t, t], u, q)


def test_draft_equal_to_target_is_always_accepted_and_a_spent_rest_falls_back(ctx):
    # q covers p: nothing is left of max(p - q, 0), so the refused draft's place is drawn from p
    logits = np.zeros((2, 8), np.float32)
    q = np.full((1, 8), 0.5, np.float32)
    u = np.array([0.9, 0.3], np.float32)
    got = verify_device(ctx, logits, [[1]], [1.0], u, q)
    assert got == ([[2]], [0]) == expect(logits, [[1]], [1.0], u, q)
    rng = np.random.default_rng(15)
    logits = rng.standard_normal((2, 700)).astype(np.float32)
    w = weights(logits[0], 1.0)
    q = (w / w.sum()).astype(np.float32)[None]
    y = int(np.argmax(q))
    got = verify_device(ctx, logits, [[y]], [1.0], np.array([0.999, 0.2], np.float32), q)
    assert got[1] == [1] and got[0][0][0] == y


def test_emitted_tokens_have_the_targets_distribution(ctx):
    # 40000 sequences of one draft: the first token's counts against p, whatever q
    rng = np.random.default_rng(16)
    n, cols = 40000, 6
    x = np.array([0.3, -1.0, 1.1, 0.0, -0.4, 0.8], np.float32)
    p = weights(x, 0.9)
    p /= p.sum()
    q = np.array([0.1, 0.3, 0.05, 0.25, 0.2, 0.1])
    y = rng.choice(cols, n, p=q)
    logits = np.broadcast_to(x, (2 * n, cols)).astype(np.float32)
    tokens, _ = verify_device(ctx, logits, [[int(t)] for t in y], [0.9] * n, rng.random(2 * n, dtype=np.float32),
                              np.broadcast_to(q.astype(np.float32), (n, cols)))
    count = np.bincount([t[0] for t in tokens], minlength=cols)
    # six standard deviations of a binomial count: once in 10^8 runs
    assert np.all(np.abs(count - n * p) < 6 * np.sqrt(n * p * (1 - p)))


def test_calls_in_flight_share_a_workspace_in_order(ctx):
    # a large call, a small one and the large one again, nothing waited for between them
    rng = np.random.default_rng(17)
    lib = ctx.lib
    sets = []
    for lens, cols in (([4] * 40, 20000), ([1], 777)):
        logits, drafts, u, q = problem(rng, cols, lens, [0.7] * len(lens), True, near=0.2)
        temps, ln = np.full(len(lens), 0.7, np.float32), np.array(lens, np.int32)
        dev = [DeviceBuffer.from_numpy(ctx, a) for a in (logits, np.array([t for d in drafts for t in d], np.uint32), u)]
        out = [DeviceBuffer(ctx, 4 * len(lens) * 5) for _ in range(2)]
        acc = [DeviceBuffer(ctx, 4 * len(lens)) for _ in range(2)]
        vb = _lib.VerifyBatch(len(lens), ln.ctypes.data_as(_lib.c_int_p), dev[1].ptr, None,
                              temps.ctypes.data_as(_lib.c_f32_p), dev[2].ptr)
        sets.append((cols, vb, dev, out, acc, (temps, ln), expect(logits, drafts, temps, u)))
    for r, i in ((0, 0), (0, 1), (1, 0), (1, 1)):
        cols, vb, dev, out, acc, _, _ = sets[i]
        ctx.check(lib.zr_verify_async(ctx.h, dev[0].ptr, cols, C.byref(vb), out[r].ptr, 5, acc[r].ptr))
    ctx.check(lib.zr_synchronize(ctx.h))
    for cols, vb, dev, out, acc, _, want in sets:
        for r in range(2):
            a = acc[r].download(np.int32, (vb.num_seqs,))
            t = out[r].download(np.uint32, (vb.num_seqs, 5))
            assert a.tolist() == want[1]
            for s in range(vb.num_seqs):
                assert t[s, :a[s] + 1].tolist() == want[0][s] and np.all(t[s, a[s] + 1:] == 0xffffffff)


def test_refusals(ctx):
    lib = ctx.lib
    x, u, o, a = (DeviceBuffer(ctx, 4096) for _ in range(4))
    lens, temps = np.array([2, 0], np.int32), np.array([1.0, 0.0], np.float32)

    def call(n=2, lens=lens, temps=temps, y=x.ptr, u_=u.ptr, cols=8, logits=x.ptr, out=o.ptr, stride=3, acc=a.ptr):
        vb = _lib.VerifyBatch(n, None if lens is None else lens.ctypes.data_as(_lib.c_int_p), y, None,
                              None if temps is None else temps.ctypes.data_as(_lib.c_f32_p), u_)
        return lib.zr_verify(ctx.h, logits, cols, C.byref(vb), out, stride, acc)

    for kw in (dict(n=0), dict(n=-1), dict(lens=None), dict(temps=None), dict(y=None), dict(u_=None), dict(logits=None),
               dict(out=None), dict(acc=None), dict(cols=0), dict(cols=(1 << 24) + 1), dict(stride=2), dict(stride=0),
               dict(lens=np.array([2, -1], np.int32)), dict(lens=np.array([256, 0], np.int32), stride=300),
               dict(temps=np.array([1.0, np.nan], np.float32))):
        assert call(**kw) == -1, kw
    assert lib.zr_verify(ctx.h, x.ptr, 8, None, o.ptr, 3, a.ptr) == -1
    assert lib.zr_verify(None, x.ptr, 8, C.byref(_lib.VerifyBatch()), o.ptr, 3, a.ptr) == -1
    with pytest.raises(ZrError):
        verify_device(ctx, np.zeros((2, 4), np.float32), [[1], []], [1.0, 1.0], np.zeros(2))
    with pytest.raises(ZrError):
        verify_device(ctx, np.zeros((2, 4), np.float32), [[1]], [1.0], np.zeros(2), np.zeros((1, 5)))


@pytest.mark.parametrize("cols", [2048, 5001])
@pytest.mark.parametrize("x_off,q_off", [(4, 0), (0, 4), (4, 8), (12, 12)])
def test_rows_at_any_alignment(ctx, cols, x_off, q_off):
    rng = np.random.default_rng(cols + x_off)
    lens = [3, 1, 2]
    temps = np.array([0.8, 1.0, 0.0], np.float32)
    logits, drafts, u, q = problem(rng, cols, lens, temps, False)
    ln = np.array(lens, np.int32)
    y, du = DeviceBuffer.from_numpy(ctx, np.array([t for d in drafts for t in d], np.uint32)), DeviceBuffer.from_numpy(ctx, u)
    pad = [DeviceBuffer.from_numpy(ctx, np.concatenate([np.full(o // 4, np.inf, np.float32), np.ravel(a)]))
           for o, a in ((x_off, logits), (q_off, q))]
    out, acc = DeviceBuffer(ctx, 4 * 3 * 9), DeviceBuffer(ctx, 12)
    out.upload(np.full(27, 7, np.uint32))
    vb = _lib.VerifyBatch(3, ln.ctypes.data_as(_lib.c_int_p), y.ptr, pad[1].ptr + q_off, temps.ctypes.data_as(_lib.c_f32_p),
                          du.ptr)
    ctx.check(ctx.lib.zr_verify(ctx.h, pad[0].ptr + x_off, cols, C.byref(vb), out.ptr, 9, acc.ptr))
    a, t = acc.download(np.int32, (3,)), out.download(np.uint32, (3, 9))
    want = expect(logits, drafts, temps, u, q)
    assert a.tolist() == want[1]
    for s in range(3):
        assert t[s, :a[s] + 1].tolist() == want[0][s] and np.all(t[s, a[s] + 1:] == 0xffffffff)


@pytest.mark.parametrize("certain", [False, True])
def test_small_calls_draw_in_two_launches_again_and_again(ctx, certain):
    """Calls of 1 to 64 workgroups over the emission rows, and one above, in turn: the count of a
    sequence's workgroups is back at 0 behind every call, also where a row is greedy."""
    rng = np.random.default_rng(31)
    sets = []
    for lens, cols in (([4], 32000), ([2], 2048), ([1, 3, 0], 40000), ([2] * 32, 4000), ([3, 1], 66000), ([4, 0, 2], 60000)):
        temps = np.where(rng.random(len(lens)) < 0.25, 0.0, 0.9).astype(np.float32)
        p = problem(rng, cols, lens, temps, certain)
        sets.append((p, temps, expect(p[0], p[1], temps, p[2], p[3])))
    for _ in range(3):
        for i in rng.permutation(len(sets)):
            (logits, drafts, u, q), temps, want = sets[i]
            assert verify_device(ctx, logits, drafts, temps, u, q) == want
