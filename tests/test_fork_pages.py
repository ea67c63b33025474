"""Forked sessions' page tables on the CPU: sharing, copy on write, truncation,
idle pages and compaction, checked against a model of the pool's contents."""
import ctypes as C

import numpy as np
import pytest

from mesh_amd import _lib
from tests.test_cabi_host import HostBackend, _decode_batch, host_pool

LIB = _lib.load()


def fork(parent, child):
    return LIB.zrh_fork(parent.h, child.h)


def idle(b):
    n = C.c_int()
    _lib.check(LIB.zrh_release_idle_pages(b.h, C.byref(n)))
    return n.value


def compact(pool):
    n = C.c_int()
    _lib.check(LIB.zrh_pool_compact(pool, C.byref(n)))
    return n.value


class Model:
    """Pool contents as row ids: a row is written once, and every session must read back what it appended."""

    def __init__(self, pages, max_seq=4096):
        self.pages = pages
        self.pool = host_pool(pages)
        self.mem = {g: [None] * 16 for g in range(pages)}
        self.sessions, self.rows = [], []
        self.next = 0
        self.max_seq = max_seq

    def new(self, max_seq=None):
        self.sessions.append(HostBackend(self.pool, self.max_seq if max_seq is None else max_seq))
        self.rows.append([])
        return len(self.sessions) - 1

    def places(self, i):
        table, globals_ = self.sessions[i].table()
        return [(g, r) for (_, start, count), g in zip(table, globals_) for r in range(start, start + count)]

    def reserve(self, i, n):
        b = self.sessions[i]
        before = self.places(i)
        rc = LIB.zrh_kv_reserve(b.h, n)
        if rc:
            assert rc == -2 and self.places(i) == before
            return False
        self.next += n
        self.rows[i] = (self.rows[i] + list(range(self.next - n, self.next)))[-min(b.seq_len, 1 << 30):]
        after = self.places(i)
        kept = len(after) - n
        # rows that were there and now lie in another page: that page is a copy
        copies = {}
        for old, new in zip(before[len(before) - kept:], after[:kept]):
            assert old[1] == new[1]
            if old[0] != new[0]:
                copies[new[0]] = old[0]
        for new, old in copies.items():
            self.mem[new] = list(self.mem[old])
        for (g, r), v in zip(after[kept:], self.rows[i][kept:]):
            self.mem[g][r] = v
        return True

    def check(self):
        held = {}
        for i, b in enumerate(self.sessions):
            assert [self.mem[g][r] for g, r in self.places(i)] == self.rows[i]
            assert b.seq_len == len(self.rows[i])
            assert LIB.zrh_sequence_position(b.h) == b.base + b.seq_len
            for g in b.table()[1]:
                held.setdefault(g, []).append(i)
        bound = self.pages - LIB.zrh_pool_free_pages(self.pool)
        assert len(held) <= bound
        assert LIB.zrh_pool_shared_pages(self.pool) == sum(len(v) > 1 for v in held.values())
        total = sum(b.pages() for b in self.sessions)
        assert total == bound + sum(len(v) - 1 for v in held.values())

    def close(self):
        for b in self.sessions:
            b.close()
        assert LIB.zrh_pool_free_pages(self.pool) == self.pages
        LIB.zrh_pool_destroy(self.pool)


def test_fork_shares_pages_and_the_first_writer_copies_the_last():
    m = Model(16)
    a = m.new()
    m.reserve(a, 40)  # two full pages, one of 8 rows
    c = m.new()
    _lib.check(fork(m.sessions[a], m.sessions[c]))
    m.rows[c] = list(m.rows[a])
    assert m.sessions[a].table()[1] == m.sessions[c].table()[1] == [0, 1, 2]
    assert LIB.zrh_pool_shared_pages(m.pool) == 3 and LIB.zrh_pool_free_pages(m.pool) == 13
    m.reserve(a, 1)  # the parent writes first: it moves to a copy
    assert m.sessions[a].table()[1] == [0, 1, 3] and m.sessions[c].table()[1] == [0, 1, 2]
    m.reserve(c, 1)  # the last holder writes in place
    assert m.sessions[c].table()[1] == [0, 1, 2]
    m.check()
    assert LIB.zrh_pool_shared_pages(m.pool) == 2
    m.sessions[a].close()  # a page goes back with its last holder only
    del m.sessions[a], m.rows[a]
    m.check()
    assert LIB.zrh_pool_free_pages(m.pool) == 13
    m.close()


def test_full_last_page_is_not_copied():
    m = Model(8)
    a, c = m.new(), m.new()
    m.reserve(a, 32)
    _lib.check(fork(m.sessions[a], m.sessions[c]))
    m.rows[c] = list(m.rows[a])
    m.reserve(a, 1)
    m.reserve(c, 1)
    m.check()
    assert m.sessions[a].table()[1] == [0, 1, 2] and m.sessions[c].table()[1] == [0, 1, 3]
    m.close()


def test_truncation_into_a_shared_page_copies_before_the_next_write():
    m = Model(8)
    a, c = m.new(), m.new()
    m.reserve(a, 32)
    _lib.check(fork(m.sessions[a], m.sessions[c]))
    m.rows[c] = m.rows[a][:27]
    _lib.check(LIB.zrh_truncate(m.sessions[c].h, 5))
    m.check()
    m.reserve(c, 3)
    m.check()  # the parent's rows 27.. are as they were
    assert m.sessions[c].table()[1] == [0, 2]
    m.close()


def test_fork_replaces_what_the_child_held():
    m = Model(8)
    a, c = m.new(), m.new()
    m.reserve(a, 20)
    m.reserve(c, 50)
    assert LIB.zrh_pool_free_pages(m.pool) == 2
    _lib.check(fork(m.sessions[a], m.sessions[c]))
    m.rows[c] = list(m.rows[a])
    assert LIB.zrh_pool_free_pages(m.pool) == 6
    m.check()
    # again from the child's own sibling, and of an empty session
    _lib.check(fork(m.sessions[a], m.sessions[c]))
    m.check()
    e = m.new()
    _lib.check(fork(m.sessions[e], m.sessions[c]))
    m.rows[c] = []
    m.check()
    m.close()


def test_fork_refusals():
    m = Model(8)
    a, small = m.new(), m.new(16)
    m.reserve(a, 20)
    assert LIB.zrh_fork(None, m.sessions[a].h) == -1 and LIB.zrh_fork(m.sessions[a].h, None) == -1
    assert fork(m.sessions[a], m.sessions[a]) == -1
    assert "into itself" in LIB.zr_global_last_error().decode()
    assert fork(m.sessions[a], m.sessions[small]) == -1
    assert "fork of 20 rows into a 16-token window" in LIB.zr_global_last_error().decode()
    other = Model(4)
    b = other.new()
    assert fork(m.sessions[a], other.sessions[b]) == -1
    assert "between KV pools" in LIB.zr_global_last_error().decode()
    m.check()
    other.close()
    m.close()


def test_truncate_refusals_and_edges():
    m = Model(8)
    a = m.new()
    m.reserve(a, 33)
    for bad in (-1, 34):
        assert LIB.zrh_truncate(m.sessions[a].h, bad) == -1
    assert LIB.zrh_truncate(None, 0) == -1
    _lib.check(LIB.zrh_truncate(m.sessions[a].h, 0))
    m.check()
    _lib.check(LIB.zrh_truncate(m.sessions[a].h, 1))  # the last page falls empty
    m.rows[a] = m.rows[a][:32]
    m.check()
    assert m.sessions[a].pages() == 3 and idle(m.sessions[a]) == 1 and m.sessions[a].pages() == 2
    _lib.check(LIB.zrh_truncate(m.sessions[a].h, 32))
    m.rows[a] = []
    m.check()
    m.reserve(a, 5)
    m.check()
    m.close()


def test_trimmed_window_truncates_from_its_end():
    m = Model(8, max_seq=40)
    a = m.new()
    m.reserve(a, 40)
    m.reserve(a, 7)  # the window slides
    base = m.sessions[a].base
    assert base == 7
    _lib.check(LIB.zrh_truncate(m.sessions[a].h, 39))
    m.rows[a] = m.rows[a][:1]
    m.check()
    assert m.sessions[a].base == base and LIB.zrh_sequence_position(m.sessions[a].h) == base + 1
    m.close()


def test_failed_call_gives_back_shared_references_and_copies():
    # two forks decode in one batch: the first takes the pool's last page for its copy, the
    # second's own copy then finds none; nothing sticks
    m = Model(4)
    a, b, c = m.new(), m.new(), m.new()
    m.reserve(a, 40)
    for x in (b, c):
        _lib.check(fork(m.sessions[a], m.sessions[x]))
        m.rows[x] = list(m.rows[a])
    before = [s.table() for s in m.sessions]
    rc = _decode_batch(m.sessions, [1, 2, 3])
    assert rc == -2 and "KV pool exhausted" in LIB.zr_global_last_error().decode()
    assert [s.table() for s in m.sessions] == before
    assert LIB.zrh_pool_free_pages(m.pool) == 1 and LIB.zrh_pool_shared_pages(m.pool) == 3
    m.check()
    # with room the batch assembles, is refused for lack of a device, and leaves the tables alone
    m.sessions[c].close()
    del m.sessions[c], m.rows[c]
    before = [s.table() for s in m.sessions]
    rc = _decode_batch(m.sessions, [1, 2])
    assert rc == -1 and "bookkeeping-only" in LIB.zr_global_last_error().decode()
    assert [s.table() for s in m.sessions] == before
    m.check()
    m.close()


def test_idle_page_is_used_when_the_pool_is_empty():
    m = Model(3)
    a, b = m.new(), m.new()
    m.reserve(a, 40)
    _lib.check(LIB.zrh_truncate(m.sessions[a].h, 20))
    m.rows[a] = m.rows[a][:20]
    _lib.check(fork(m.sessions[a], m.sessions[b]))
    m.rows[b] = list(m.rows[a])
    assert LIB.zrh_pool_free_pages(m.pool) == 0
    assert not m.reserve(a, 20)  # a copy of the half page and a new page: the session's idle page is one of the two
    m.check()
    assert m.reserve(a, 1)  # the copy alone: the idle page takes it
    m.check()
    assert m.sessions[a].table()[1] == [0, 2] and m.sessions[b].table()[1] == [0, 1]
    m.close()


@pytest.mark.parametrize("seed", range(12))
def test_random_forks_keep_every_sessions_rows(seed):
    rng = np.random.default_rng(seed)
    m = Model(int(rng.choice([24, 64, 300])), int(rng.choice([40, 100, 4096])))
    m.new()
    for _ in range(250):
        i = int(rng.integers(len(m.sessions)))
        b, r = m.sessions[i], rng.random()
        if r < 0.45:
            m.reserve(i, int(rng.integers(1, 40)))
        elif r < 0.6:
            if len(m.sessions) < 8 and rng.random() < 0.6:
                j = m.new()
            else:
                j = int(rng.integers(len(m.sessions)))
            if j != i:
                _lib.check(fork(b, m.sessions[j]))
                m.rows[j] = list(m.rows[i])
        elif r < 0.75:
            n = int(rng.integers(0, b.seq_len + 1))
            _lib.check(LIB.zrh_truncate(b.h, n))
            m.rows[i] = m.rows[i][:len(m.rows[i]) - n]
        elif r < 0.82:
            keep = int(rng.integers(0, b.seq_len + 2))
            b.retain(keep)
            m.rows[i] = m.rows[i][max(0, len(m.rows[i]) - keep):]
        elif r < 0.87:
            b.clear()
            m.rows[i] = []
        elif r < 0.9 and len(m.sessions) > 1:
            b.close()
            del m.sessions[i], m.rows[i]
        elif r < 0.95:
            idle(b)
        else:
            old = [m.places(k) for k in range(len(m.sessions))]
            compact(m.pool)
            mem = {g: [None] * 16 for g in range(m.pages)}
            for k, places in enumerate(old):
                for (g, _), (h, _) in zip(places, m.places(k)):
                    mem[h] = m.mem[g]
            m.mem = {g: list(v) for g, v in mem.items()}
            # the free pages are the highest
            free = LIB.zrh_pool_free_pages(m.pool)
            assert all(g < m.pages - free for k in range(len(m.sessions)) for g, _ in m.places(k))
        m.check()
    m.close()


def test_compaction_counts_pages_with_rows_only():
    m = Model(10)
    a, b = m.new(), m.new()
    m.reserve(a, 48)
    m.reserve(b, 48)
    _lib.check(LIB.zrh_truncate(m.sessions[b].h, 20))  # pages 3, 4 hold rows, 5 is bound but idle
    m.rows[b] = m.rows[b][:28]
    m.sessions[a].close()
    del m.sessions[a], m.rows[a]
    assert compact(m.pool) == 2  # 3 -> 0 or so, 4 -> 1 or so; 5 is bound to another page without a copy
    assert LIB.zrh_pool_compact(None, None) == -1
    assert compact(m.pool) == 0
    _lib.check(LIB.zrh_pool_compact(m.pool, None))
    m.close()


def test_sessions_of_a_destroyed_pool_refuse_rows():
    m = Model(4)
    a = m.new()
    m.reserve(a, 5)
    LIB.zrh_pool_destroy(m.pool)
    b = m.sessions[a]
    assert LIB.zrh_kv_reserve(b.h, 1) == -1
    assert "pool was destroyed" in LIB.zr_global_last_error().decode()
    b.close()


def test_a_verified_step_that_cannot_run_leaves_every_session_as_it_was():
    """Without a device the step is assembled, refused and rolled back, shared pages and copies included."""
    m = Model(8, max_seq=64)
    a = m.new()
    m.reserve(a, 40)
    c, tight = m.new(), m.new(max_seq=41)
    for s in (c, tight):
        _lib.check(fork(m.sessions[a], m.sessions[s]))
        m.rows[s] = list(m.rows[a])
    i32, u32, f32 = (lambda x: x.ctypes.data_as(_lib.c_int_p)), (lambda x: x.ctypes.data_as(_lib.c_u32_p)), \
        (lambda x: x.ctypes.data_as(_lib.c_f32_p))

    def step(who, drafts, stride=300):
        n = len(who)
        h = (C.c_void_p * n)(*[m.sessions[s].h for s in who])
        k, toks = np.array(drafts, np.int32), np.zeros(max(1, sum(drafts) + n), np.uint32)
        u, t = np.zeros(toks.size, np.float32), np.zeros(n, np.float32)
        out, acc = np.zeros(n * 300, np.uint32), np.full(n, -7, np.int32)
        rc = LIB.zrh_verify_batch(C.cast(h, C.POINTER(C.c_void_p)), n, i32(k), u32(toks), f32(t), f32(u), None, u32(out),
                                  stride, i32(acc))
        assert np.all(acc == -7) and not out.any()
        return rc

    before = [m.places(s) for s in (a, c, tight)]
    free = LIB.zrh_pool_free_pages(m.pool)
    for who, drafts, kw in (([a, c], [2, 3], {}),          # both would take copies of the last page
                            ([a, c], [20, 20], {}),        # more pages than the pool has
                            ([a, tight], [2, 1], {}),      # the second window would slide
                            ([a, a], [1, 1], {}),
                            ([a], [256], {}), ([a], [-1], {}), ([a, c], [1, 4], dict(stride=4))):
        assert step(who, drafts, **kw) < 0, (who, drafts)
        assert [m.places(s) for s in (a, c, tight)] == before and LIB.zrh_pool_free_pages(m.pool) == free
        m.check()
    m.close()
