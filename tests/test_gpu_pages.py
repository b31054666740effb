"""GPU tests of the page cache (g4s_pages_*) against the row-by-row restatement
in beam_oracle.py.  Everything is whole numbers and bytes: equal or wrong."""
import numpy as np
import pytest

import beam_oracle as bo
from gemma4_sampler import beam, hip, native

pytestmark = pytest.mark.gpu
I32 = np.int32
BIG = (1 << 31) - 1


class Rig:
    """A page cache, its two states and its pool, beside the oracle's."""

    def __init__(self, P, N, rows, slots, planes=2, parts=2, token=32, outer=False, pad=0,
                 shift=0, stream=None):
        page = parts * P * token
        self.P, self.N, self.rows, self.slots = P, N, rows, slots
        self.planes, self.parts, self.token, self.shift = planes, parts, token, shift
        if outer:
            self.plane, self.page = page + pad, (page + pad) * planes
        else:
            self.page = page + pad
            self.plane = self.page * N
        self.cache = beam.PageCache(P, N, rows, slots, planes, parts, token,
                                    plane_stride=self.plane, page_stride=self.page,
                                    stream=stream)
        self.size = shift + max(self.plane * planes, self.page * N)
        self.rng = np.random.default_rng(N + rows)
        self.pool = self.rng.integers(0, 256, self.size, dtype=np.uint8)
        self.d_pool = hip.Buffer.from_array(self.pool)
        self.d_status = hip.Buffer.from_array(np.full(8, 99, I32))
        self.cur = bo.State(rows, slots, N)
        self.dev = [self.upload(self.cur), self.upload(self.cur)]

    def upload(self, s):
        bufs = [hip.Buffer.from_array(a) for a in (s.table, s.lengths, s.refs)]
        return bufs, beam.PageState(*bufs)

    def put(self, s):
        self.cur = s
        self.dev = [self.upload(s), self.upload(bo.State(self.rows, self.slots, self.N))]

    def pages(self, raw):
        """[plane][page][part][token] bytes of a pool"""
        v = np.lib.stride_tricks.as_strided(
            raw[self.shift:], (self.planes, self.N, self.parts, self.P, self.token),
            (self.plane, self.page, self.P * self.token, self.token, 1))
        return v

    def read(self, d):
        s = bo.State(self.rows, self.slots, self.N)
        s.table[:] = d[0][0].download(I32).reshape(s.table.shape)
        s.lengths[:], s.refs[:] = d[0][1].download(I32), d[0][2].download(I32)
        return s

    def check(self, want, copies, status, code_only=False):
        hip.synchronize()
        got_status = self.d_status.download(I32)
        assert tuple(got_status[:4]) == tuple(status) and (got_status[4:] == 99).all()
        got = self.read(self.dev[1])
        if status[0] == 0:
            assert np.array_equal(got.table, want.table)
        assert np.array_equal(got.lengths, want.lengths)
        assert np.array_equal(got.refs, want.refs)
        v = self.pages(self.pool)
        old = v.copy()
        for a, b, n in copies:
            v[:, b, :, :n] = old[:, a, :, :n]
        assert np.array_equal(self.d_pool.download(np.uint8), self.pool)
        before = self.read(self.dev[0])  # `from` is as it was
        for k in ("table", "lengths", "refs"):
            assert np.array_equal(getattr(before, k), getattr(self.cur, k)), k

    def advance(self, parents, grow, from_rows=None, keep=True):
        parents = np.asarray(parents, I32)
        rows = len(parents)
        from_rows = self.rows if from_rows is None else from_rows
        want = self.read(self.dev[1])
        g = np.zeros(rows, I32) if grow is None else np.asarray(grow, I32)
        status, copies = bo.advance(self.cur, from_rows, want, rows, parents, g, self.P)
        self.cache.advance(self.dev[0][1], from_rows, self.dev[1][1], rows,
                           hip.Buffer.from_array(parents),
                           None if grow is None else hip.Buffer.from_array(g),
                           self.d_pool.offset(self.shift) if self.planes else None,
                           self.d_status)
        self.check(want, copies, status)
        if status[0] == 0 and keep:
            self.cur = want
            self.dev.reverse()
        return status

    def compact(self, rows=None):
        rows = self.rows if rows is None else rows
        want = self.read(self.dev[1])
        status, moves = bo.compact(self.cur, want, rows, self.P)
        self.cache.compact(self.dev[0][1], self.dev[1][1], rows, self.d_pool.offset(self.shift),
                           self.d_status)
        self.check(want, [(a, b, self.P) for a, b in moves], status)
        self.cur = want
        self.dev.reverse()
        return status


SHAPES = [dict(P=4, N=40, rows=6, slots=8), dict(P=1, N=70, rows=5, slots=12, parts=1),
          dict(P=16, N=33, rows=7, slots=5, outer=True, pad=16),
          dict(P=3, N=60, rows=6, slots=9, token=4, pad=4, shift=4),
          dict(P=5, N=50, rows=6, slots=7, token=3, pad=1, shift=1, parts=3),
          dict(P=8, N=2100, rows=40, slots=300, planes=1, parts=1, token=16),
          dict(P=2, N=64, rows=6, slots=10, planes=0, parts=0, token=0)]


@pytest.mark.parametrize("shape", SHAPES)
def test_random_steps(shape):
    """Admissions, forks, appends, truncations, ends and compactions in any
    order, every state against the restatement."""
    rig = Rig(**shape)
    rng = np.random.default_rng(shape["N"])
    R, S, P = rig.rows, rig.slots, rig.P
    room = S * P
    for step in range(30):
        parents = rng.integers(-1, R, R)
        old = np.where(parents >= 0, rig.cur.lengths[parents], 0)
        grow = rng.choice([0, 1, 1, 1, 2, P, P + 1, -1, -P, -BIG], R)
        grow = np.where(parents < 0, rng.integers(0, max(2, min(room, 2 * P)), R), grow)
        grow = np.minimum(grow, room - old)
        if step % 3 == 0:
            parents = np.sort(parents)
            grow = np.where(parents < 0, 2, np.minimum(1, room - np.where(
                parents >= 0, rig.cur.lengths[parents], 0)))
        rig.advance(parents, grow if step % 5 else None, keep=True)
        if step % 7 == 6 and rig.planes:
            rig.compact()


def test_fork_rules():
    """Which of the rows that go on writing one page keeps it."""
    rig = Rig(4, 32, 8, 6)
    assert rig.advance([-1] * 8, [6, 0, 0, 8, 0, 0, 0, 0]) == (0, 28, 4, 0)
    # three writers of one partly filled page: the first keeps it, two copy; row 3's
    # pages are full: its forks take new pages alone
    assert rig.advance([0, 0, 0, 3, 3, -1, -1, -1], [1, 1, 1, 1, 2, 0, 0, 0])[2:] == (4, 2)
    # a reader beside two writers: both copy
    assert rig.advance([0, 0, 0, -1, 3, 4, -1, -1], [1, 0, 1, 0, 0, 0, 0, 0])[2:] == (2, 2)
    # back into a shared page, then on: the longer reader keeps its tokens
    assert rig.advance([1, 1, 1, -1, 4, 4, -1, -1], [-5, 0, -2, 0, 0, 0, 0, 0])[2:] == (0, 0)
    assert rig.advance([0, 1, 2, 3, 4, 5, -1, -1], [1] * 6 + [0, 0])[3] >= 3
    # nobody's rows end
    assert rig.advance([-1] * 8, None) == (0, 32, 0, 0)


def test_same_call_twice():
    """A step can be taken again from the same state: the same result."""
    rig = Rig(4, 64, 8, 8)
    rig.advance([-1] * 8, [5, 7, 9, 4, 0, 1, 2, 3])
    for _ in range(3):
        rig.advance([0, 0, 1, 1, 2, 2, 6, 7], [1] * 8, keep=False)


def test_rows_behind_the_last_stay():
    rig = Rig(4, 64, 8, 8)
    rig.advance([-1] * 8, [5] * 8)
    rig.advance([0, 1, 2], [1, 1, 1], keep=False)
    assert (rig.read(rig.dev[1]).lengths[3:] == 0).all()
    rig.put(rig.cur)
    marked = bo.State(8, 8, 64)
    marked.table[:], marked.lengths[:] = 55, 44
    rig.dev[1] = rig.upload(marked)
    rig.advance([0, 1, 2], [1, 1, 1], from_rows=5, keep=False)
    got = rig.read(rig.dev[1])
    assert (got.table[3:] == 55).all() and (got.lengths[3:] == 44).all()


def test_out_of_pages_is_all_or_nothing():
    rig = Rig(4, 12, 4, 12)
    rig.advance([-1] * 4, [9, 5, 4, 1])            # 3 + 2 + 1 + 1
    assert rig.advance([0, 1, 2, 3], [0, 0, 21, 0])[0] == native.G4S_ERR_OUT_OF_MEMORY
    assert rig.advance([0, 1, 2, 3], [0, 0, 20, 0], keep=False)[0] == 0
    # pages that the step itself frees are not handed out in it
    assert rig.advance([-1, -1, -1, -1], [24, 0, 0, 0])[0] == native.G4S_ERR_OUT_OF_MEMORY
    assert rig.advance([-1, 1, 2, 3], None)[0] == 0
    assert rig.advance([-1, 1, 2, 3], [24, 1, 0, 0])[0] == 0


@pytest.mark.parametrize("parents, grow", [
    ([0, 1, 4, 2], [1, 1, 1, 1]), ([0, -2, 1, 2], [0, 0, 0, 0]), ([0, BIG, 1, 2], None),
    ([0, -BIG - 1, 1, 2], None), ([0, 1, 2, 3], [0, 0, 40, 0]), ([0, 1, 2, 3], [BIG, 0, 0, 0])])
def test_bad_steps(parents, grow):
    rig = Rig(4, 30, 4, 10)
    rig.advance([-1] * 4, [9, 5, 4, 1])
    assert rig.advance(parents, grow)[0] == native.G4S_ERR_INVALID_ARGUMENT
    assert rig.advance([3, 2, 1, 0], [1, 1, 1, 1])[0] == 0  # nothing is left behind


@pytest.mark.parametrize("page", [-1, 30, BIG, -BIG - 1, 29])
def test_bad_pages(page):
    """A page outside the pool, or one that the state does not hold."""
    rig = Rig(4, 30, 4, 10)
    rig.advance([-1] * 4, [9, 5, 4, 1])
    for row, slot in [(0, 0), (0, 2), (3, 0)]:
        good = rig.cur.copy()
        bad = rig.cur.copy()
        bad.table[row, slot] = page
        rig.put(bad)
        assert rig.advance([3, 0, 1, 2], [1, 1, 1, 1])[0] == native.G4S_ERR_FORMAT
        want = rig.read(rig.dev[1])
        want.lengths[:], want.refs[:] = 0, 0
        rig.cache.compact(rig.dev[0][1], rig.dev[1][1], 4, rig.d_pool, rig.d_status)
        rig.check(want, [], (native.G4S_ERR_FORMAT, 30, 0, 0))
        rig.put(good)
        assert rig.advance([3, 0, 1, 2], [1, 1, 1, 1], keep=False)[0] == 0


def test_bad_lengths():
    rig = Rig(4, 30, 4, 10)
    rig.advance([-1] * 4, [9, 5, 4, 1])
    for n in (-1, 41, BIG, -BIG - 1):
        bad = rig.cur.copy()
        bad.lengths[1] = n
        good, rig.cur = rig.cur, bad
        rig.put(bad)
        assert rig.advance([0, 1, 2, 3], None)[0] == native.G4S_ERR_INVALID_ARGUMENT
        want = rig.read(rig.dev[1])
        want.lengths[:], want.refs[:] = 0, 0
        rig.cache.compact(rig.dev[0][1], rig.dev[1][1], 4, rig.d_pool, rig.d_status)
        rig.check(want, [], (native.G4S_ERR_INVALID_ARGUMENT, 30, 0, 0))
        rig.put(good)


def test_compact_edges():
    rig = Rig(4, 1030, 6, 200, planes=1, parts=1, token=16)
    assert rig.compact() == (0, 1030, 0, 0)                 # nothing live
    rig.advance([-1] * 6, [400, 396, 800, 4, 797, 0])
    assert rig.compact()[3] == 0                            # already together
    rig.advance([-1, 1, -1, 3, 4, -1], None)
    assert rig.compact()[3] > 0
    rig.advance([-1, 1, -1, 3, 4, -1], [800, 0, 800, 4, 3, 800])
    assert rig.compact()[3] == 0
    rig.advance([1, -1, 5, -1, 4, 2], None)                 # rows shared, low pages free
    rig.compact()
    rig.compact()


def test_compact_longest_rows():
    """A row of nearly 2^31 tokens, all of max_slots pages, behind one that ends:
    the tokens of its last page are counted past 32 bits."""
    P, S = 3000, 715827
    rig = Rig(P, 715900, 2, S, planes=0, parts=0, token=0)
    assert rig.advance([-1, -1], [7 * P, S * P])[:3] == (0, 66, 715834)
    rig.advance([-1, 1], None)
    assert rig.compact() == (0, 73, 0, 7)


def test_many_rows():
    """More rows than a workgroup has threads, all writing one page."""
    R = 1100
    rig = Rig(4, 3000, R, 3, planes=1, parts=1, token=16)
    rig.advance([-1] * R, [6] + [0] * (R - 1))
    assert rig.advance([0] * R, [1] * R)[2:] == (R - 1, R - 1)
    rig.advance(np.arange(R)[::-1], [2] * R)
    rig.compact()


def test_most_rows_and_pages():
    """The limits of the handle: 2,048 rows that write one page, in a pool of 2^20."""
    R, N = beam.PAGES_MAX_ROWS, beam.PAGES_MAX_PAGES
    rig = Rig(4, N, R, 600, planes=1, parts=1, token=4)
    # 512 rows of 599 pages, then the row that all others follow
    grow = np.zeros(R, I32)
    grow[:512], grow[512] = 4 * 599, 6
    assert rig.advance([-1] * R, grow) == (0, N - 512 * 599 - 2, 512 * 599 + 2, 0)
    assert rig.advance([512] * R, [1] * R)[2:] == (R - 1, R - 1)
    rig.advance(np.arange(R)[::-1], [2] * R)
    assert rig.compact()[3] > 0


def test_captured_steps():
    """Two steps, there and back between the states, in one captured graph that is
    replayed with other parents, eager steps of the same cache between."""
    from test_gpu_beam import _capture
    st = hip.Stream(nonblocking=True)
    rig = Rig(4, 300, 8, 30, stream=st)
    rig.advance([-1] * 8, [9, 5, 4, 1, 7, 16, 2, 3])
    rng = np.random.default_rng(5)
    d_par = [hip.Buffer(32), hip.Buffer(32)]
    d_grow = hip.Buffer.from_array(np.ones(8, I32))
    at = rig.d_pool.offset(0)

    def record():
        rig.cache.advance(rig.dev[0][1], 8, rig.dev[1][1], 8, d_par[0], d_grow, at, rig.d_status)
        rig.cache.advance(rig.dev[1][1], 8, rig.dev[0][1], 8, d_par[1], d_grow, at, rig.d_status)
    destroy, launch = _capture(st, record)
    for _ in range(5):
        parents = [np.sort(rng.integers(0, 8, 8)).astype(I32), rng.permutation(8).astype(I32)]
        st.synchronize()
        for d, p in zip(d_par, parents):
            d.upload(p)
        want = [rig.cur, rig.read(rig.dev[1])]
        for i in range(2):
            status, copies = bo.advance(want[0], 8, want[1], 8, parents[i], np.ones(8, I32), 4)
            v = rig.pages(rig.pool)
            old = v.copy()
            for a, b, n in copies:
                v[:, b, :, :n] = old[:, a, :, :n]
            want.reverse()
        launch()
        st.synchronize()
        got = rig.read(rig.dev[0])
        for k in ("table", "lengths", "refs"):
            assert np.array_equal(getattr(got, k), getattr(want[0], k)), k
        assert tuple(rig.d_status.download(I32)[:4]) == status
        assert np.array_equal(rig.d_pool.download(np.uint8), rig.pool)
        rig.cur = want[0]
        rig.advance(rng.integers(0, 8, 8), np.zeros(8, I32))  # eager, and back again
        rig.advance(np.arange(8), None)
    destroy()
    st.destroy()


def test_copy():
    for shape in SHAPES[:6]:
        rig = Rig(**shape)
        rng = np.random.default_rng(3)
        other = rng.integers(0, 256, rig.size, dtype=np.uint8)
        d_other = hip.Buffer.from_array(other)
        n = rig.N // 2
        src, dst = (rng.permutation(rig.N)[:n].astype(I32) for _ in range(2))
        tok = rng.integers(0, rig.P + 1, n).astype(I32)
        src[0], dst[1], tok[2], tok[3] = rig.N, -1, -7, BIG
        lists = [hip.Buffer.from_array(a) for a in (src, dst, tok)]
        for d_tok in (lists[2], None):
            rig.cache.copy(rig.d_pool.offset(rig.shift), d_other.offset(rig.shift), n, lists[0],
                           lists[1], d_tok)
            hip.synchronize()
            v, w = rig.pages(rig.pool), rig.pages(other)
            for i in range(n):
                k = rig.P if d_tok is None else min(max(int(tok[i]), 0), rig.P)
                if 0 <= src[i] < rig.N and 0 <= dst[i] < rig.N:
                    w[:, dst[i], :, :k] = v[:, src[i], :, :k]
            assert np.array_equal(d_other.download(np.uint8), other)
            assert np.array_equal(rig.d_pool.download(np.uint8), rig.pool)
        # within one pool
        src = np.arange(0, n, 2, dtype=I32)
        dst = src + 1
        rig.cache.copy(rig.d_pool.offset(rig.shift), rig.d_pool.offset(rig.shift), len(src),
                       hip.Buffer.from_array(src), hip.Buffer.from_array(dst))
        hip.synchronize()
        v = rig.pages(rig.pool)
        v[:, dst] = v[:, src]
        assert np.array_equal(rig.d_pool.download(np.uint8), rig.pool)


def test_pool_past_32_bits():
    """Pages more than 4 GiB apart in two planes."""
    P, N, token = 16, 40000, 8192
    page = P * token  # 128 KiB: planes of 4.9 GiB
    c = beam.PageCache(P, N, 4, 4, planes=2, parts=1, token_bytes=token)
    pool = hip.Buffer(2 * page * N)
    rng = np.random.default_rng(4)
    src, dst = np.array([N - 1, 3], I32), np.array([0, N - 2], I32)
    data = {}
    for plane in range(2):
        for p in (N - 1, 3, 0, N - 2):
            data[plane, p] = rng.integers(0, 256, page, dtype=np.uint8)
            pool.upload(data[plane, p], (plane * N + p) * page)
    c.copy(pool, pool, 2, hip.Buffer.from_array(src), hip.Buffer.from_array(dst),
           hip.Buffer.from_array(np.array([16, 5], I32)))
    hip.synchronize()
    for plane in range(2):
        for s, d, k in [(N - 1, 0, 16), (3, N - 2, 5)]:
            want = data[plane, d].copy()
            want[:k * token] = data[plane, s][:k * token]
            got = pool.download(np.uint8, page, (plane * N + d) * page)
            assert np.array_equal(got, want)
    c.close()


def test_refusals():
    rig = Rig(4, 30, 4, 10)
    a, b = rig.dev[0][1], rig.dev[1][1]
    one = hip.Buffer(4096)
    null = beam.PageState()
    mixed = beam.PageState(rig.dev[1][0][0], rig.dev[0][0][1], rig.dev[1][0][2])
    good = dict(src=a, src_rows=4, dst=b, rows=4, d_parents=one, d_grow=one, d_pool=rig.d_pool,
                d_status=rig.d_status)
    for change in [dict(src=None), dict(dst=None), dict(src=null), dict(dst=null), dict(dst=a),
                   dict(dst=mixed), dict(src_rows=0), dict(src_rows=5), dict(rows=0),
                   dict(rows=5), dict(d_parents=None), dict(d_pool=None), dict(d_status=None)]:
        with pytest.raises(native.SamplerError) as e:
            rig.cache.advance(**dict(good, **change))
        assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT, change
    good = dict(src=a, dst=b, rows=4, d_pool=rig.d_pool, d_status=rig.d_status)
    for change in [dict(src=None), dict(dst=a), dict(rows=0), dict(rows=5), dict(d_pool=None),
                   dict(d_status=None)]:
        with pytest.raises(native.SamplerError) as e:
            rig.cache.compact(**dict(good, **change))
        assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT, change
    good = dict(d_src_pool=rig.d_pool, d_dst_pool=rig.d_pool, n=2, d_src_pages=one,
                d_dst_pages=one)
    rig.cache.copy(**dict(good, n=0))
    for change in [dict(n=-1), dict(d_src_pool=None), dict(d_dst_pool=None),
                   dict(d_src_pages=None), dict(d_dst_pages=None),
                   dict(d_dst_pool=rig.d_pool.offset(64))]:
        with pytest.raises(native.SamplerError) as e:
            rig.cache.copy(**dict(good, **change))
        assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT, change


def test_overlapping_arrays_are_refused():
    """One workgroup writes while others read: the status over a table, parents
    inside the new state, lists inside the pool that is written."""
    N, R, S = 8, 2, 4
    c = beam.PageCache(4, N, R, S, planes=2, parts=1, token_bytes=16)
    pool_bytes = 2 * N * 64
    mem = hip.Buffer(8192).zero()
    at = {"from": (0, 64, 128), "to": (256, 320, 384)}
    pool, status, one, grow = (mem.offset(o) for o in (4096, 512, 576, 640))

    def state(key, **other):
        o = dict(zip(("table", "lengths", "refs"), at[key]))
        o.update(other)
        return beam.PageState(*(mem.offset(o[k]) for k in ("table", "lengths", "refs")))
    good = dict(src=state("from"), src_rows=R, dst=state("to"), rows=R, d_parents=one, d_grow=grow,
                d_pool=pool, d_status=status)
    bad = [dict(d_status=mem.offset(o)) for o in (0, 28, 64, 156, 256, 320, 384, 576, 636, 4096,
                                                  4096 + pool_bytes - 4)]
    bad += [{k: mem.offset(o)} for k in ("d_parents", "d_grow")
            for o in (256, 284, 320, 412, 512, 4096 + pool_bytes - 4)]
    bad += [dict(dst=state("to", **k)) for k in (dict(lengths=284), dict(refs=260),
                                                 dict(refs=320), dict(table=4096))]
    bad += [dict(d_pool=mem.offset(o)) for o in (0, 160, 384, 512, 644)]
    for change in bad:
        for only in (None, "compact"):
            args = dict(good, **change)
            if only:
                if "d_parents" in change or "d_grow" in change or \
                        change.get("d_status", one).value in (one.value, one.value + 60):
                    continue
                args = {k: args[k] for k in ("src", "dst", "rows", "d_pool", "d_status")}
                if change.get("d_pool", pool).value == mem.offset(644).value:
                    continue
            with pytest.raises(native.SamplerError) as e:
                (c.compact if only else c.advance)(**args)
            assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT, change
    c.advance(**good)
    c.advance(**dict(good, d_grow=one))                   # both are only read
    c.advance(**dict(good, d_pool=mem.offset(656), d_status=mem.offset(4096)))
    hip.synchronize()
    mem.upload(np.array([0, 1, 2, 3], I32), 4096 - 16)
    lists = [mem.offset(4096 - 8), mem.offset(4096 - 16)]
    good = dict(d_src_pool=mem.offset(1024), d_dst_pool=pool, n=2, d_src_pages=lists[0],
                d_dst_pages=lists[1], d_tokens=None)
    for k in ("d_src_pages", "d_dst_pages", "d_tokens"):
        for o in (4096 - 4, 4096 + pool_bytes - 4):
            with pytest.raises(native.SamplerError) as e:
                c.copy(**dict(good, **{k: mem.offset(o)}))
            assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT, (k, o)
    c.copy(**dict(good, d_tokens=mem.offset(1024)))       # inside the source: only read
    hip.synchronize()
    c.close()
