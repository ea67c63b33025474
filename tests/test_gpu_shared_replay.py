"""Replayed decode steps of sessions that share their leading pages: the same
kernels and metadata as the eager steps, so the same ids, keys and values bit for
bit, through a step graph, through a pipeline, and with buckets that change between
shared and unshared batches."""
import ctypes as C

import numpy as np
import pytest

from mesh_amd import BackendMicrobatchExecutor, DecodeMicrobatchRequest, DecodePipeline, DeviceBuffer
from mesh_amd._lib import PrefixInfo
from tests.test_gpu_fork_pages import model_context

pytestmark = pytest.mark.gpu


def steps(backends, tokens, n, want_logits):
    """n greedy steps of one row each; eager where the logits are asked for."""
    out = []
    for _ in range(n):
        got = BackendMicrobatchExecutor.decode_step_batch(
            [DecodeMicrobatchRequest(str(i), t, b) for i, (t, b) in enumerate(zip(tokens, backends))], want_logits=want_logits)
        tokens = [o.sampled_token for o in got]
        out.append(tokens)
    return out


def same_cache(a, b):
    for x, y in zip(a, b):
        x, y = x.export_kv_cache(), y.export_kv_cache()
        np.testing.assert_array_equal(x.keys, y.keys)
        np.testing.assert_array_equal(x.values, y.values)


def prompt_of(ctx, rows, seed=0):
    p = ctx.new_backend()
    p.prefill(np.random.default_rng(rows + seed).integers(0, 512, rows).tolist())
    return p


@pytest.mark.parametrize("kv,heads,kv_heads,d", [("bf16", 4, 2, 64), ("f32", 4, 1, 64), ("bf16", 8, 2, 128), ("bf16", 2, 2, 64)])
@pytest.mark.parametrize("rows,forks", [(300, 6), (130, 16), (480, 2)])
def test_replayed_steps_are_the_eager_ones(kv, heads, kv_heads, d, rows, forks):
    ctx = model_context(kv, heads, kv_heads, d, pages=500)
    parent = prompt_of(ctx, rows)
    first = np.random.default_rng(1).integers(0, 512, forks).tolist()
    eager = [parent.fork() for _ in range(forks)]
    replayed = [parent.fork() for _ in range(forks)]
    assert ctx.shared_pages > 0
    want = steps(eager, first, 28, True)
    before = ctx.forward_replay_info()["launches"]
    assert steps(replayed, first, 28, False) == want
    info = ctx.forward_replay_info()
    assert info["launches"] - before >= 20
    same_cache(eager, replayed)
    ctx.close()


def test_pipelined_steps_are_the_eager_ones():
    ctx = model_context("bf16", 8, 2, 64, pages=500)
    parent = prompt_of(ctx, 200)
    first = np.random.default_rng(2).integers(0, 512, 5).tolist()
    eager, piped = ([parent.fork() for _ in range(5)] for _ in range(2))
    want = steps(eager, first, 24, True)
    p = DecodePipeline(piped, first)
    got = []
    for _ in range(24):
        t = p.step()
        if t is not None:
            got.append(list(t))
    got.append(list(p.finish()))
    p.close()
    assert got == want
    same_cache(eager, piped)
    ctx.close()


def test_buckets_follow_batches_that_share_and_batches_that_do_not():
    ctx = model_context("bf16", 4, 2, 64, pages=600)
    rng = np.random.default_rng(3)
    parents = [prompt_of(ctx, 150, s) for s in range(3)]
    other = [prompt_of(ctx, 90, s) for s in range(4)]
    shared = [parents[0].fork() for _ in range(4)]
    mixed = [parents[1].fork(), parents[1].fork(), parents[2].fork(), parents[2].fork()]
    twins = ([b.fork() for b in other], [b.fork() for b in shared], [b.fork() for b in mixed])
    groups = (other, shared, mixed)
    tokens = [rng.integers(0, 512, 4).tolist() for _ in groups]
    also = [list(t) for t in tokens]
    for n in (5, 1, 4, 2, 6):
        for i, (g, twin) in enumerate(zip(groups, twins)):
            # (a twin shares every page with its own original only: the batch of twins has the
            # original batch's structure, whatever that is)
            got, want = steps(g, tokens[i], n, False), steps(twin, also[i], n, True)
            assert got == want
            tokens[i], also[i] = got[-1], want[-1]
    for g, twin in zip(groups, twins):
        same_cache(g, twin)
    ctx.close()


def test_sessions_that_leave_the_shared_start_go_on_by_themselves(monkeypatch):
    """A window that trims its first pages stops sharing them; switched off, nothing is shared."""
    ctx = model_context("bf16", 4, 2, 64, pages=600)
    parent = ctx.new_backend(max_seq_len=160)
    parent.prefill(np.random.default_rng(9).integers(0, 512, 150).tolist())
    first = [1, 2, 3, 4]
    eager, replayed = ([parent.fork() for _ in range(4)] for _ in range(2))
    want = steps(eager, first, 40, True)  # slides from the 11th step on
    assert steps(replayed, first, 40, False) == want
    same_cache(eager, replayed)
    monkeypatch.setenv("ZR_SHARED_PREFIX", "0")
    alone = [parent.fork() for _ in range(4)]
    again = [parent.fork() for _ in range(4)]
    want = steps(alone, first, 12, True)
    assert steps(again, first, 12, False) == want
    same_cache(alone, again)
    ctx.close()


def test_a_captured_shared_step_replays_its_logits():
    ctx = model_context("bf16", 8, 2, 128, pages=300)
    lib, n = ctx.lib, 6
    parent = prompt_of(ctx, 260)
    forks = [parent.fork() for _ in range(n)]
    other = prompt_of(ctx, 40, 7)
    arr = (C.c_void_p * n)(*[b.h for b in forks])
    st, g = C.c_void_p(), C.c_void_p()
    tokens = np.arange(3, 3 + n, dtype=np.uint32)
    ones = np.ones(n, np.int32)
    ctx.check(lib.zrh_stage_mixed(C.cast(arr, C.POINTER(C.c_void_p)), n, ones.ctypes.data_as(C.POINTER(C.c_int)),
                                  tokens.ctypes.data_as(C.POINTER(C.c_uint32)), C.byref(st)))
    info = PrefixInfo()
    ctx.check(lib.zr_staged_prefix_info(st.value, C.byref(info)))
    assert (info.segments, info.sequences, info.rows) == (1, n, n)
    logits = DeviceBuffer(ctx, 4 * n * 512)
    other.decode_step(1)  # (grows what it needs before the capture)
    ctx.check(lib.zr_forward_staged_async(ctx.h, st.value, None, None, logits.ptr))
    ctx.check(lib.zr_synchronize(ctx.h))
    want = logits.download(np.float32, (n, 512))
    assert np.isfinite(want).all()
    ctx.check(lib.zr_graph_capture_staged(ctx.h, st.value, None, None, logits.ptr, C.byref(g)))
    for _ in range(4):
        logits.upload(np.full((n, 512), np.nan, np.float32))
        ctx.check(lib.zr_graph_launch(ctx.h, g.value))
        ctx.check(lib.zr_synchronize(ctx.h))
        np.testing.assert_array_equal(logits.download(np.float32, (n, 512)), want)
        other.decode_step(2)  # the program's own eager work between replays
    lib.zr_graph_destroy(g.value)
    lib.zr_staged_destroy(st.value)
    ctx.close()


def test_two_contexts_at_once():
    """Each context has its own stream and workspaces: interleaved steps are those of each alone."""
    rng = np.random.default_rng(11)
    ctxs = [model_context(kv, 4, 2, 64, pages=300) for kv in ("bf16", "f32")]
    parents = [prompt_of(c, 150 + 30 * i) for i, c in enumerate(ctxs)]
    first = rng.integers(0, 512, 4).tolist()
    alone = []
    for p in parents:
        forks = [p.fork() for _ in range(4)]
        alone.append(steps(forks, first, 10, False))
    forks = [[p.fork() for _ in range(4)] for p in parents]
    pipes = [DecodePipeline(f, first) for f in forks]  # (both streams run while the host goes on)
    got = [[], []]
    for _ in range(10):
        for out, p in zip(got, pipes):
            t = p.step()
            if t is not None:
                out.append(list(t))
    for out, p in zip(got, pipes):
        out.append(list(p.finish()))
        p.close()
    assert got == alone
    for c in ctxs:
        c.close()


@pytest.mark.parametrize("rows", [77, 80, 95])
def test_a_session_forked_inside_a_pipeline(rows):
    ctx = model_context("bf16", 4, 2, 64, pages=300)
    parent = prompt_of(ctx, rows)
    first = [4, 5, 6]
    eager, piped = ([parent.fork() for _ in range(3)] for _ in range(2))
    want = steps(eager, first, 20, True)
    p = DecodePipeline(piped, first)
    got, children = [], []
    for i in range(20):
        t = p.step()
        if t is not None:
            got.append(list(t))
        if i % 6 == 2:  # with this step in flight
            children.append((piped[1].fork(), i + 1))
            assert children[-1][0].cache_seq_len() == rows + i + 1
        if i % 6 == 4:  # a child writes beside the pipeline's own writes
            children[-1][0].decode_step(9)
    got.append(list(p.finish()))
    p.close()
    assert got == want
    same_cache(eager, piped)
    whole = eager[1].export_kv_cache()
    for child, n in children:
        c = child.export_kv_cache()
        np.testing.assert_array_equal(c.keys[:, :rows + n], whole.keys[:, :rows + n])
        np.testing.assert_array_equal(c.values[:, :rows + n], whole.values[:, :rows + n])
    ctx.close()
