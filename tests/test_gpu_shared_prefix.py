"""Attention of sequences that share leading pages, against a 64-bit
restatement of the same softmax over each sequence's own window."""
import ctypes as C

import numpy as np
import pytest

from mesh_amd import DeviceBuffer, DeviceContext, ModelGeometry, _lib
from mesh_amd._lib import ZrError
from tests.gpu_util import f32p, i32p

pytestmark = pytest.mark.gpu


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16) & 0xFFFFFFFF).astype(np.uint32).view(np.float32)


class Batch:
    """Sequences given as page tables over a pool whose rows are known: (table, first_offset, kv_before, q_len) each."""

    def __init__(self, kv, heads, kv_heads, d, seqs, seed=0, pages=None, split=True, nan_rows=()):
        self.kv, self.heads, self.kv_heads, self.d, self.seqs = kv, heads, kv_heads, d, seqs
        rng = np.random.default_rng(seed)
        pages = pages or 1 + max(max(t) for t, *_ in seqs)
        total = sum(s[3] for s in seqs)
        stride = max(len(t) for t, *_ in seqs)
        g = ModelGeometry(hidden=heads * d, num_heads=heads, num_kv_heads=kv_heads, num_layers=2, vocab=32, ffn=64)
        self.ctx = ctx = DeviceContext(g, kv_dtype=kv, max_tokens=max(total, 16), max_seqs=len(seqs), max_pages_per_seq=stride,
                                       split_activations=split)
        ctx.create_kv_pool(pages)
        w = kv_heads * d
        self.k = rng.standard_normal((2, pages * 16, w), dtype=np.float32)
        self.v = rng.standard_normal((2, pages * 16, w), dtype=np.float32)
        if kv == "bf16":
            self.k, self.v = bf16(self.k), bf16(self.v)
        for r in nan_rows:  # rows outside every window
            self.k[:, r] = np.nan
            self.v[:, r] = np.inf
        whole = np.arange(pages, dtype=np.int32)
        ctx.check(ctx.lib.zr_kv_scatter(ctx.h, i32p(whole), pages, 0, 0, pages * 16, f32p(self.k), f32p(self.v)))
        self.q = (rng.standard_normal((total, heads * d)) * 1.3).astype(np.float32)
        self.stage(stride)

    def stage(self, stride):
        ctx, seqs = self.ctx, self.seqs
        n = len(seqs)
        tables = np.zeros((n, stride), np.int32)
        for i, (t, *_) in enumerate(seqs):
            tables[i, :len(t)] = t
        arr = [np.ascontiguousarray([s[j] for s in seqs], np.int32) for j in (3, 2, 1)]
        q_len, kv_before, first_offset = arr
        self.mb_keep = (q_len, kv_before, first_offset, tables)
        mb = _lib.Microbatch(n, i32p(q_len), i32p(kv_before), i32p(kv_before), i32p(first_offset), i32p(tables), stride,
                             None)
        st = C.c_void_p()
        ctx.check(ctx.lib.zr_stage(ctx.h, C.byref(mb), C.byref(st)))
        self.st = st.value

    def info(self):
        p = _lib.PrefixInfo()
        self.ctx.check(self.ctx.lib.zr_staged_prefix_info(self.st, C.byref(p)))
        return {n: getattr(p, n) for n, _ in _lib.PrefixInfo._fields_}

    def attend(self, layer=1, q=None):
        ctx = self.ctx
        q = self.q if q is None else q
        d_q = DeviceBuffer.from_numpy(ctx, q)
        d_o = DeviceBuffer.from_numpy(ctx, np.full_like(q, np.nan))
        ctx.check(ctx.lib.zr_attention(ctx.h, self.st, layer, d_q.ptr, d_o.ptr))
        out = d_o.download(np.float32, q.shape)
        d_q.free()
        d_o.free()
        return out

    def want(self, layer=1):
        """(values, bound on the error of each) in 64 bits."""
        out, tol = np.zeros(self.q.shape), np.zeros(self.q.shape)
        row = 0
        G = self.heads // self.kv_heads
        for table, fo, kb, ql in self.seqs:
            rows = np.concatenate([np.arange(p * 16, p * 16 + 16) for p in table])[fo:fo + kb + ql]
            k = self.k[layer, rows].astype(np.float64).reshape(-1, self.kv_heads, self.d)
            v = self.v[layer, rows].astype(np.float64).reshape(-1, self.kv_heads, self.d)
            for i in range(ql):
                n = kb + i + 1
                for h in range(self.heads):
                    q = self.q[row, h * self.d:(h + 1) * self.d].astype(np.float64)
                    kh, vh = k[:n, h // G], v[:n, h // G]
                    s = kh @ q / np.sqrt(self.d)
                    p = np.exp(s - s.max())
                    sl = slice(h * self.d, (h + 1) * self.d)
                    out[row, sl] = p @ vh / p.sum()
                    # Each operand enters as hi + lo bf16, off by at most 2^-18 of itself (half a step of
                    # lo, 2^-9, times the largest lo, 2^-9); the dropped lo x lo products are below that
                    # again; sums of up to d terms and the exponent's scale are off by d 2^-24 at most.
                    s_err = (4 * 2.0 ** -18 + self.d * 2.0 ** -24) * (np.abs(kh) @ np.abs(q)).max() / np.sqrt(self.d)
                    # o = sum p v / sum p: relative errors of p of e move it by 2 e max |v|; P and V are
                    # split too (f32 pools), exp2 and the f32 sums of n terms add their last bits
                    e = np.expm1(s_err) + 4 * 2.0 ** -18 + (n + 64) * 2.0 ** -24
                    tol[row, sl] = 2 * e * np.abs(vh).max()
                row += 1
        return out, tol

    def check(self, layer=1):
        want, tol = self.want(layer)
        got = self.attend(layer)
        assert np.all(np.isfinite(got))
        bad = np.abs(got - want) > tol
        assert not bad.any(), (int(bad.sum()), float(np.abs(got - want).max()), float(tol.min()))
        # far below the bound in the mean: a missed or doubled row shows
        assert np.linalg.norm(got - want) < 1e-4 * np.linalg.norm(want)
        return got

    def close(self):
        self.ctx.lib.zr_staged_destroy(self.st)
        self.ctx.close()


def forked(sessions, shared, tails, rows=1, fo=0, extra=(), order_seed=1):
    """Sessions behind `shared` common pages; tail i holds tails[i % len] rows, the new ones among them."""
    rng = np.random.default_rng(order_seed)
    need = shared + sum(-(-max(tails[i % len(tails)], rows) // 16) for i in range(sessions))
    order = rng.permutation(need + 3).tolist()
    prefix, at, out = order[:shared], shared, []
    for i in range(sessions):
        t = max(tails[i % len(tails)], rows)
        n = -(-t // 16)
        out.append((prefix + order[at:at + n], fo, shared * 16 - fo + t - rows, rows))
        at += n
    return out


GEOMETRIES = [("bf16", 8, 2, 128), ("bf16", 16, 2, 64), ("bf16", 4, 4, 128), ("bf16", 16, 1, 128), ("bf16", 4, 2, 64),
              ("f32", 16, 2, 64), ("f32", 8, 2, 128), ("f32", 2, 2, 64)]


@pytest.mark.parametrize("kv,heads,kv_heads,d", GEOMETRIES)
@pytest.mark.parametrize("sessions,shared,tails,rows", [
    (3, 9, [1, 7, 40], 1),          # the smallest batches, an odd number of pages
    (9, 4, [16, 17, 33], 1),        # the shortest run that is shared
    (5, 33, [5, 30], 5),            # the last token and four drafts each
    (40, 12, [3, 20], 2),           # more columns than a unit holds
])
def test_shared_prefix_matches_64_bit(kv, heads, kv_heads, d, sessions, shared, tails, rows):
    b = Batch(kv, heads, kv_heads, d, forked(sessions, shared, tails, rows), seed=sessions)
    info = b.info()
    assert info["segments"] == 1 and info["sequences"] == sessions and info["rows"] == sessions * rows
    assert info["pages_saved"] == (sessions - 1) * shared
    b.check(0)
    b.check(1)
    b.close()


@pytest.mark.parametrize("kv,d", [("bf16", 128), ("bf16", 64), ("f32", 64)])
@pytest.mark.parametrize("fo", [1, 15])
def test_trimmed_first_page_hides_what_it_holds(kv, d, fo):
    # the rows before the window are not finite, in the shared pages' first one
    seqs = forked(6, 10, [4, 19], 1, fo=fo)
    rows = [seqs[0][0][0] * 16 + r for r in range(fo)]
    b = Batch(kv, 8, 2, d, seqs, nan_rows=rows)
    assert b.info()["segments"] == 1
    b.check()
    b.close()


def test_windows_that_start_at_other_rows_are_not_shared():
    seqs = forked(4, 8, [9], 1)
    seqs[1] = (seqs[1][0], 3, seqs[1][2] - 3, 1)
    seqs[3] = (seqs[3][0], 3, seqs[3][2] - 3, 1)
    b = Batch("bf16", 8, 2, 128, seqs)
    assert b.info()["segments"] == 2 and b.info()["sequences"] == 4
    b.check()
    b.close()


@pytest.mark.parametrize("seqs,why", [
    (forked(1, 20, [5]), "one sequence"),
    (forked(8, 3, [5]), "a run below four pages"),
    (forked(2, 5, [5]), "a run that saves too little"),
    ([(list(range(10)), 0, 150, 1), (list(range(10, 20)), 0, 150, 1)], "nothing in common"),
    # the pages agree, but one sequence's new rows are in them (an unusual caller): only full pages before them count
    ([([0, 1, 2, 3, 4], 0, 40, 1), ([0, 1, 5, 6, 7], 0, 70, 1)], "two full pages in common"),
])
def test_what_is_not_shared(seqs, why):
    b = Batch("bf16", 8, 2, 64, seqs)
    assert b.info()["segments"] == 0, why
    b.check()
    b.close()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_prompts_with_forks_of_their_own(kv):
    # prompt A (12 pages) with two groups of forks that went on together (9 and 20 pages more), one
    # fork by itself; prompt B (30 pages); a session on its own; sequences in no order
    ids = iter(np.random.default_rng(3).permutation(400).tolist())
    take = lambda n: [next(ids) for _ in range(n)]  # noqa: E731
    a, b30 = take(12), take(30)
    a1, a2 = a + take(9), a + take(20)
    seqs = [(a1 + take(2), 0, 21 * 16 + 20, 1) for _ in range(3)] + [(a2 + take(1), 0, 32 * 16 + 3, 1) for _ in range(5)]
    seqs += [(a + take(3), 0, 12 * 16 + 40, 1), (take(7), 0, 100, 1)] + [(b30 + take(1), 0, 480 + i, 1) for i in range(4)]
    order = np.random.default_rng(4).permutation(len(seqs))
    b = Batch(kv, 8, 2, 128, [seqs[i] for i in order], pages=400)
    info = b.info()
    assert info["segments"] == 4 and info["sequences"] == 13
    assert info["pages_saved"] == 8 * 12 + 2 * 9 + 4 * 20 + 3 * 30
    b.check()
    b.close()


def test_short_common_start_is_read_with_the_longer_runs_behind_it():
    # two common pages (too few to share), then two groups with six more of their own each
    ids = iter(range(200))
    take = lambda n: [next(ids) for _ in range(n)]  # noqa: E731
    a = take(2)
    a1, a2 = a + take(6), a + take(6)
    seqs = [(t + take(1), 0, 8 * 16 + 5, 1) for t in (a1, a2) for _ in range(4)]
    b = Batch("bf16", 8, 2, 128, seqs)
    info = b.info()
    assert info["segments"] == 2 and info["pages_saved"] == 2 * 3 * 8
    b.check()
    b.close()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_beside_prompt_chunks_and_sequences_of_their_own(kv):
    # a prompt chunk on the same prefix runs as prefill blocks and is not shared; a short one is
    seqs = forked(6, 20, [3, 18], 1, order_seed=7)
    top = 1 + max(max(t) for t, *_ in seqs)
    chunk = seqs[0][0][:20] + list(range(top, top + 5))
    short = seqs[0][0][:20] + list(range(top + 5, top + 7))
    alone = list(range(top + 7, top + 30))
    seqs = [(chunk, 0, 20 * 16, 70)] + seqs[:3] + [(short, 0, 20 * 16 + 1, 7), (alone, 0, 300, 1)] + seqs[3:]
    b = Batch(kv, 8, 2, 128, seqs)
    info = b.info()
    shared = 7 if kv == "bf16" else info["sequences"]  # f32 chunks of little work run as decode tiles and are shared
    assert info["segments"] == 1 and info["sequences"] == shared
    b.check()
    b.close()


def test_long_prefix_in_many_splits():
    b = Batch("bf16", 4, 1, 64, forked(3, 300, [5, 100], 1))
    assert b.info()["segments"] == 1 and b.info()["units"] > 1
    b.check()
    b.close()


def test_switched_off_it_reads_every_window_by_itself(monkeypatch):
    seqs = forked(10, 24, [9, 30], 1)
    b = Batch("bf16", 8, 2, 128, seqs)
    on = b.check()
    monkeypatch.setenv("ZR_SHARED_PREFIX", "0")
    off = Batch("bf16", 8, 2, 128, seqs)
    assert off.info() == dict(segments=0, sequences=0, rows=0, units=0, pages_saved=0)
    got = off.check()
    assert np.abs(got - on).max() < 1e-3 and b.info()["segments"] == 1
    off.close()
    b.close()


@pytest.mark.parametrize("rope", [0, 1])
def test_rope_attention_of_a_shared_batch_is_its_two_stages(rope):
    b = Batch("bf16", 8, 2, 64, forked(7, 12, [4, 21], 1))
    ctx, w = b.ctx, 512 + 2 * 128
    qkv = np.random.default_rng(5).standard_normal((7, w), dtype=np.float32)
    d_qkv = DeviceBuffer.from_numpy(ctx, qkv)
    d_q, d_a, d_b = (DeviceBuffer(ctx, 4 * 7 * 512) for _ in range(3))
    ctx.check(ctx.lib.zr_rope_kv_write(ctx.h, b.st, 0, d_qkv.ptr, d_q.ptr, rope))
    ctx.check(ctx.lib.zr_attention(ctx.h, b.st, 0, d_q.ptr, d_a.ptr))
    ctx.check(ctx.lib.zr_rope_attention(ctx.h, b.st, 0, d_qkv.ptr, d_b.ptr, rope))
    np.testing.assert_array_equal(d_a.download(np.float32, (7, 512)), d_b.download(np.float32, (7, 512)))
    b.close()


def test_calls_in_flight_and_repeated_are_the_same():
    # four calls of two batches on two contexts, nothing waited for between them
    bs = [Batch("bf16", 8, 2, 128, forked(20, 40, [5, 60], 1), seed=1), Batch("f32", 8, 2, 64, forked(6, 9, [30], 1), seed=2)]
    want = [b.attend() for b in bs]
    d_q = [DeviceBuffer.from_numpy(b.ctx, b.q) for b in bs]
    outs = [[DeviceBuffer(b.ctx, b.q.nbytes) for _ in range(2)] for b in bs]
    for r in range(2):
        for b, q, o in zip(bs, d_q, outs):
            b.ctx.check(b.ctx.lib.zr_attention_async(b.ctx.h, b.st, 1, q.ptr, o[r].ptr))
    for b, w, o in zip(bs, want, outs):
        b.ctx.check(b.ctx.lib.zr_synchronize(b.ctx.h))
        for x in o:  # sums in a fixed order: the same bits every time
            np.testing.assert_array_equal(x.download(np.float32, b.q.shape), w)
        b.close()


def test_refusals():
    b = Batch("bf16", 8, 2, 64, forked(4, 8, [9]))
    lib, ctx = b.ctx.lib, b.ctx
    d = DeviceBuffer(ctx, b.q.nbytes)
    for args in [(None, b.st, 0, d.ptr, d.ptr), (ctx.h, None, 0, d.ptr, d.ptr), (ctx.h, b.st, 0, None, d.ptr),
                 (ctx.h, b.st, 0, d.ptr, None), (ctx.h, b.st, 2, d.ptr, d.ptr), (ctx.h, b.st, -1, d.ptr, d.ptr)]:
        assert lib.zr_attention_async(*args) == -1
    other = Batch("bf16", 8, 2, 64, forked(4, 8, [9]))
    assert lib.zr_attention_async(ctx.h, other.st, 0, d.ptr, d.ptr) == -1
    assert b"another context" in lib.zr_last_error(ctx.h)
    assert lib.zr_staged_prefix_info(None, C.byref(_lib.PrefixInfo())) == -1
    assert lib.zr_staged_prefix_info(b.st, None) == -1
    other.close()
    b.close()


@pytest.mark.parametrize("kv,kv_heads,pages", [("bf16", 8, 70000), ("f32", 8, 35000)])
def test_pages_past_4_gib(kv, kv_heads, pages):
    """A layer of more than 2^32 bytes: the same contents at its last pages and, copied, at its first."""
    ctx = DeviceContext(ModelGeometry(4 * 8 * 128, 32, kv_heads, 1, 32, 64), kv_dtype=kv, max_tokens=64, max_seqs=8,
                        max_pages_per_seq=128, split_activations=True)
    ctx.create_kv_pool(pages)
    assert ctx.kv_pool_bytes() > 1 << 32
    ctx.check(ctx.lib.zr_kv_pool_fill_normal(ctx.h, 3, 1.0))
    rng = np.random.default_rng(5)
    n, shared, own = 6, 90, 20
    low = rng.permutation(shared + n * own).astype(np.int32)
    high = (pages - 1 - rng.permutation(shared + n * own)).astype(np.int32)
    assert (int(high.min()) + 1) * (ctx.kv_pool_bytes() // pages) > 1 << 32
    ctx.copy_pages(high, low)
    q = (rng.standard_normal((n, 32 * 128)) * 1.3).astype(np.float32)
    d_q, d_o = DeviceBuffer.from_numpy(ctx, q), DeviceBuffer(ctx, q.nbytes)
    out = []
    for ids in (high, low):
        tables = np.array([np.concatenate([ids[:shared], ids[shared + i * own:shared + (i + 1) * own]]) for i in range(n)], np.int32)
        ones, before, zero = np.ones(n, np.int32), np.full(n, (shared + own) * 16 - 5, np.int32), np.zeros(n, np.int32)
        mb = _lib.Microbatch(n, i32p(ones), i32p(before), i32p(before), i32p(zero), i32p(tables), shared + own, None)
        st, info = C.c_void_p(), _lib.PrefixInfo()
        ctx.check(ctx.lib.zr_stage(ctx.h, C.byref(mb), C.byref(st)))
        ctx.check(ctx.lib.zr_staged_prefix_info(st.value, C.byref(info)))
        assert info.segments == 1 and info.sequences == n
        ctx.check(ctx.lib.zr_attention(ctx.h, st.value, 0, d_q.ptr, d_o.ptr))
        out.append(d_o.download(np.float32, q.shape))
        ctx.lib.zr_staged_destroy(st.value)
    assert np.isfinite(out[0]).all()
    np.testing.assert_array_equal(out[0], out[1])
    assert np.std(out[0]) > 1e-3
    ctx.close()


def test_a_smaller_pool_refuses_what_named_pages_it_has_not():
    p = Batch("bf16", 4, 2, 64, [(list(range(12)) + [12 + i], 0, 195, 1) for i in range(3)])
    p.attend()
    p.ctx.check(p.ctx.lib.zr_kv_pool_create(p.ctx.h, 14))
    with pytest.raises(ZrError, match="page 14 of another pool, this one has 14"):
        p.attend()
    p.ctx.check(p.ctx.lib.zr_kv_pool_create(p.ctx.h, 15))
    assert np.all(p.attend() == 0)  # (the same page ids, in the new pool)
    p.ctx.close()
