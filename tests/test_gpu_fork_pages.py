"""Page copies, forks, truncation and compaction on the device: raw page bits,
and sessions that decode as if each had its own window."""
import ctypes as C

import numpy as np
import pytest

from mesh_amd import BackendMicrobatchExecutor, DeviceContext, ModelGeometry
from mesh_amd._lib import ZrError
from tests.gpu_util import i32p
from tests.testmodels import geometry, random_weights

pytestmark = pytest.mark.gpu


def context(kv="bf16", layers=2, heads=4, kv_heads=2, d=64, pages=64, **kw):
    g = ModelGeometry(hidden=heads * d, num_heads=heads, num_kv_heads=kv_heads, num_layers=layers, vocab=128, ffn=256)
    ctx = DeviceContext(g, kv_dtype=kv, max_tokens=kw.pop("max_tokens", 256), max_seqs=16, max_pages_per_seq=32, **kw)
    ctx.create_kv_pool(pages)
    return ctx


def page_bits(ctx, pages):
    """Raw bytes of `pages` in every layer."""
    n = len(pages)
    per = ctx.kv_pool_bytes() // (ctx.lib.zr_kv_pool_pages(ctx.h) * ctx.geo.num_layers)
    out = np.zeros((ctx.geo.num_layers, n, per), np.uint8)
    p = np.ascontiguousarray(pages, np.int32)
    for l in range(ctx.geo.num_layers):
        ctx.check(ctx.lib.zr_kv_read_pages(ctx.h, l, i32p(p), n, out[l].ctypes.data))
    return out


# head sizes of both page layouts; 448 pairs go in one launch
@pytest.mark.parametrize("kv,kv_heads,d,n", [("bf16", 2, 64, 1), ("f32", 2, 64, 7), ("bf16", 4, 128, 30),
                                             ("f32", 1, 80, 16), ("bf16", 1, 6 * 16, 449), ("bf16", 2, 64, 1000)])
def test_copied_pages_hold_the_source_bits_and_others_stay(kv, kv_heads, d, n):
    pages = 3 * n + 5
    ctx = context(kv, 3, 4 * kv_heads, kv_heads, d, pages)
    ctx.check(ctx.lib.zr_kv_pool_fill_normal(ctx.h, 5, 1.0))
    rng = np.random.default_rng(n)
    order = rng.permutation(pages)
    dst = order[:n]
    src = rng.choice(order[n:], n)  # a page may be the source of several
    before = page_bits(ctx, np.arange(pages))
    ctx.copy_pages(src, dst)
    after = page_bits(ctx, np.arange(pages))
    want = before.copy()
    want[:, dst] = before[:, src]
    np.testing.assert_array_equal(after, want)
    assert ctx.lib.zr_kv_pool_data(ctx.h)
    ctx.close()


def test_page_copy_refusals_copy_nothing():
    ctx = context(pages=8)
    ctx.check(ctx.lib.zr_kv_pool_fill_normal(ctx.h, 5, 1.0))
    before = page_bits(ctx, np.arange(8))
    for src, dst, status in [([0, 1], [2, 2], -1), ([0, 1], [1, 2], -1), ([3], [3], -1), ([0], [8], -4), ([-1], [0], -4)]:
        with pytest.raises(ZrError) as e:
            ctx.copy_pages(src, dst)
        assert e.value.status == status
    one = np.zeros(1, np.int32)
    assert ctx.lib.zr_kv_copy_pages(ctx.h, None, i32p(one), 1) == -1
    assert ctx.lib.zr_kv_copy_pages(ctx.h, i32p(one), i32p(one), -1) == -1
    assert ctx.lib.zr_kv_copy_pages(None, i32p(one), i32p(one), 1) == -1
    ctx.copy_pages([], [])
    np.testing.assert_array_equal(page_bits(ctx, np.arange(8)), before)
    ctx.close()
    bare = DeviceContext(ModelGeometry(64, 1, 1, 1, 32, 64), max_tokens=1, max_seqs=1, max_pages_per_seq=1)
    assert bare.lib.zr_kv_copy_pages(bare.h, i32p(one), i32p(one), 1) == -1
    assert not bare.lib.zr_kv_pool_data(bare.h)
    bare.close()


def model_context(kv, heads, kv_heads, d, layers=2, pages=200):
    cfg = dict(hidden=heads * d, num_heads=heads, num_kv_heads=kv_heads, num_layers=layers, vocab=512, ffn=256,
               rms_norm_eps=1e-5, rope_base=10000.0)
    ctx = DeviceContext(ModelGeometry(cfg["hidden"], heads, kv_heads, layers, 512, 256), kv_dtype=kv, max_tokens=128,
                        max_seqs=16, max_pages_per_seq=32, split_activations=True)
    ctx.upload_f32_model(random_weights(cfg, geometry(cfg), seed=3, std=0.05))
    ctx.create_kv_pool(pages)
    return ctx


def decode(backends, tokens):
    """One eager mixed microbatch of one row each, with logits."""
    return BackendMicrobatchExecutor.forward_mixed(backends, [[t] for t in tokens])[1]


# every page layout; prompts whose last page is full, has one row, and is the only one
@pytest.mark.parametrize("kv,heads,kv_heads,d", [("bf16", 4, 2, 64), ("f32", 4, 1, 64), ("bf16", 2, 2, 80)])
@pytest.mark.parametrize("rows", [5, 32, 33, 100])
def test_forks_decode_like_sessions_of_their_own(kv, heads, kv_heads, d, rows):
    ctx = model_context(kv, heads, kv_heads, d)
    rng = np.random.default_rng(rows)
    prompt = rng.integers(0, 512, rows).tolist()
    parent = ctx.new_backend()
    parent.prefill(prompt)
    forks = [parent.fork() for _ in range(3)]
    assert [f.sequence_position() for f in forks] == [rows] * 3
    own = []
    for _ in range(4):
        b = ctx.new_backend()
        b.prefill(prompt)
        own.append(b)
    shared = [parent] + forks
    for step in range(20):  # over a page border
        tokens = rng.integers(0, 512, 4).tolist()
        got, want = decode(shared, tokens), decode(own, tokens)
        # The same rows through other pages: the order of f32 sums may differ, and with it a new K / V
        # value on a bf16 tie (2^-8 of one element of one of at least 6 keys: under 2^-8 of an output
        # of order 1 spread over them, 7e-4).  A wrong row moves the logits by their own size, order 1.
        np.testing.assert_allclose(got, want, rtol=0, atol=1e-3)
    # every session's keys and values: the prompt's bit for bit, the others to a bf16 step
    for s, o in zip(shared, own):
        a, b = s.export_kv_cache(), o.export_kv_cache()
        assert a.keys.shape == b.keys.shape and a.next_position == b.next_position
        np.testing.assert_allclose(a.keys, b.keys, rtol=2.0 ** -7, atol=1e-3)
        np.testing.assert_allclose(a.values, b.values, rtol=2.0 ** -7, atol=1e-3)
        np.testing.assert_array_equal(a.keys[:, :rows], b.keys[:, :rows])
        np.testing.assert_array_equal(a.values[:, :rows], b.values[:, :rows])
    ctx.close()


def test_truncated_session_decodes_as_if_the_rows_had_never_been():
    ctx = model_context("bf16", 4, 2, 64)
    rng = np.random.default_rng(1)
    prompt = rng.integers(0, 512, 30).tolist()
    a, b = ctx.new_backend(), ctx.new_backend()
    a.prefill(prompt)
    b.prefill(prompt)
    keep = a.fork()
    BackendMicrobatchExecutor.forward_mixed([a], [[1, 2, 3, 4, 5]])
    a.truncate(5)
    assert a.sequence_position() == 30 and a.cache_seq_len() == 30
    for t in [7, 8, 9]:
        np.testing.assert_array_equal(decode([a], [t]), decode([b], [t]))
    np.testing.assert_array_equal(keep.export_kv_cache().keys, a.export_kv_cache().keys[:, :30])
    ctx.close()


def test_compaction_keeps_windows_and_refuses_what_was_staged():
    ctx = model_context("bf16", 4, 2, 64, pages=60)
    rng = np.random.default_rng(2)
    bs = [ctx.new_backend() for _ in range(6)]
    for b in bs:
        b.prefill(rng.integers(0, 512, int(rng.integers(20, 90))).tolist())
    fork = bs[5].fork()
    for b in bs[:4:2]:
        b.release_pages()
    live = [bs[1], bs[3], bs[4], bs[5], fork]
    before = [b.export_kv_cache() for b in live]
    logits = decode(live, [5] * 5)
    for b in live:
        b.truncate(1)
    one = np.ones(5, np.int32)
    arr = (C.c_void_p * 5)(*[b.h for b in live])
    st, g = C.c_void_p(), C.c_void_p()
    ctx.check(ctx.lib.zrh_stage_mixed(C.cast(arr, C.POINTER(C.c_void_p)), 5, i32p(one),
                                      np.full(5, 5, np.uint32).ctypes.data_as(C.POINTER(C.c_uint32)), C.byref(st)))
    ctx.check(ctx.lib.zr_graph_capture_staged(ctx.h, st.value, None, None, None, C.byref(g)))
    for b in live:
        b.truncate(1)
    moved = ctx.compact_pages()
    assert moved > 0
    for rc in (ctx.lib.zr_graph_launch(ctx.h, g.value), ctx.lib.zr_forward_staged_async(ctx.h, st.value, None, None, None)):
        assert rc == -1 and b"compacted" in ctx.lib.zr_last_error(ctx.h)
    ctx.lib.zr_graph_destroy(g.value)
    ctx.lib.zr_staged_destroy(st.value)
    used = {g for b in live for _, _, _, g in b.block_table()}
    assert max(used) < 60 - ctx.free_pages
    for b, s in zip(live, before):
        after = b.export_kv_cache()
        np.testing.assert_array_equal(after.keys, s.keys)
        np.testing.assert_array_equal(after.values, s.values)
    np.testing.assert_allclose(decode(live, [5] * 5), logits, rtol=0, atol=2e-4)
    ctx.close()
