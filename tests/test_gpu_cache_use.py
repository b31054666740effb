"""GPU tests of the 8-bit cache as it is used: with the pages that g4s_pages_*
keeps, in captured graphs, on other streams, from two handles, at its largest
sizes; and what a live handle refuses."""
import ctypes

import numpy as np
import pytest

import beam_oracle as bo
import cache_oracle as co
from gemma4_sampler import beam, cache, hip, native
from test_gpu_beam import _capture
from test_gpu_cache import MARK, Rig, Vectors

pytestmark = pytest.mark.gpu
I32 = np.int32
DTYPE = {"f32": native.DTYPE_F32, "bf16": native.DTYPE_BF16}


# ------------------------------------------------------------------ refusals


class Calls:
    """A handle with arguments that it takes, to change one at a time."""

    def __init__(self):
        self.rig = r = Rig([20, 9], news=[5, 9], dtype="bf16", kv=2, group=2, d=64, rotary=64)
        n = r.tokens
        self.q, self.out = (Vectors(r.random(r.heads), "bf16") for _ in range(2))
        self.k, self.v = (Vectors(r.random(r.kv), "bf16") for _ in range(2))
        self.lse = hip.Buffer(n * r.heads * 4)
        self.positions = hip.Buffer.from_array(np.arange(n, dtype=I32))

    def append(self, **change):
        r = self.rig
        a = dict(state=r.state, rows=2, tokens=r.tokens, dtype=DTYPE["bf16"], d_pool=r.d_pool,
                 k_plane=2, v_plane=0, q=self.q.view, k=self.k.view, v=self.v.view,
                 q_out=self.out.view, d_starts=r.d_starts, d_positions=self.positions,
                 d_freqs=r.d_freqs)
        a.update(change)
        r.cache.append(**a)

    def attend(self, **change):
        r = self.rig
        a = dict(state=r.state, rows=2, tokens=r.tokens, dtype=DTYPE["bf16"], d_pool=r.d_pool,
                 k_plane=2, v_plane=0, q=self.q.view, out=self.out.view, scale=0.125, window=0,
                 d_starts=r.d_starts, d_lse=self.lse)
        a.update(change)
        r.cache.attend(**a)


@pytest.fixture(scope="module")
def calls():
    c = Calls()
    c.append()
    c.attend()
    hip.synchronize()
    return c


def view(v, data=None, ts=None, hs=None, shift=0):
    d = v.buf.offset(shift) if data is None else data
    return cache.View(d, v.ts if ts is None else ts, v.hs if hs is None else hs)


BOTH = [
    lambda c: dict(state=None), lambda c: dict(rows=0), lambda c: dict(rows=3),
    lambda c: dict(rows=-1), lambda c: dict(tokens=0), lambda c: dict(tokens=-5),
    lambda c: dict(tokens=cache.MAX_TOKENS + 1), lambda c: dict(d_starts=None),
    lambda c: dict(dtype=7), lambda c: dict(dtype=-1), lambda c: dict(d_pool=None),
    lambda c: dict(d_pool=c.rig.d_pool.offset(2)), lambda c: dict(k_plane=0),
    lambda c: dict(k_plane=3), lambda c: dict(v_plane=-1), lambda c: dict(v_plane=3),
    lambda c: dict(state=beam.PageState(None, c.rig.d_lengths, None)),
    lambda c: dict(state=beam.PageState(c.rig.d_table, None, None)),
    lambda c: dict(q=view(c.q, shift=8)), lambda c: dict(q=view(c.q, ts=c.q.ts + 4)),
    lambda c: dict(q=view(c.q, hs=c.q.hs + 1)), lambda c: dict(q=view(c.q, ts=-c.q.ts)),
    lambda c: dict(q=view(c.q, hs=-64)), lambda c: dict(q=view(c.q, hs=48)),
    lambda c: dict(q=view(c.q, ts=128)), lambda c: dict(q=view(c.q, ts=1 << 62)),
    lambda c: dict(q=view(c.q, data=ctypes.c_void_p(0))),
]


@pytest.mark.parametrize("change", BOTH)
def test_refused_by_both(calls, change):
    for call in (calls.append, calls.attend):
        with pytest.raises(native.SamplerError) as e:
            call(**change(calls))
        assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT
        assert calls.rig.cache.last_error()
    calls.attend()  # the handle works on, and its message is gone
    assert calls.rig.cache.last_error() == ""
    hip.synchronize()


@pytest.mark.parametrize("change", [
    lambda c: dict(q=None), lambda c: dict(q_out=None), lambda c: dict(k=None),
    lambda c: dict(v=None), lambda c: dict(q=None, q_out=None, k=None, v=None),
    lambda c: dict(d_freqs=None), lambda c: dict(k=view(c.k, shift=4)),
    lambda c: dict(v=view(c.v, ts=c.v.ts + 1)),
    lambda c: dict(q_out=view(c.q, hs=c.q.hs * c.q.n, ts=64)),  # q itself, other strides
    lambda c: dict(q_out=view(c.q, shift=32)),
    lambda c: dict(q_out=view(c.k)), lambda c: dict(q_out=view(c.v)),
    lambda c: dict(q_out=view(c.q, data=c.rig.d_pool)), lambda c: dict(k=view(c.k, data=c.rig.d_pool)),
    lambda c: dict(v=view(c.v, data=c.rig.d_pool)), lambda c: dict(q=view(c.q, data=c.rig.d_pool)),
    lambda c: dict(d_pool=c.rig.d_table), lambda c: dict(d_positions=c.out.buf),
    lambda c: dict(d_positions=c.rig.d_pool), lambda c: dict(d_freqs=c.out.buf),
    lambda c: dict(q_out=view(c.q, data=c.rig.d_lengths)),
    lambda c: dict(q_out=view(c.q, data=c.rig.d_starts)),
])
def test_refused_by_append(calls, change):
    with pytest.raises(native.SamplerError) as e:
        calls.append(**change(calls))
    assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("change", [
    lambda c: dict(q=None), lambda c: dict(out=None), lambda c: dict(scale=float("nan")),
    lambda c: dict(scale=float("inf")), lambda c: dict(window=-1), lambda c: dict(out=c.q.view),
    lambda c: dict(out=view(c.q, shift=16)), lambda c: dict(out=view(c.q, data=c.rig.d_pool)),
    lambda c: dict(out=view(c.out, data=c.rig.d_table)), lambda c: dict(d_lse=c.q.buf),
    lambda c: dict(d_lse=c.out.buf), lambda c: dict(d_lse=c.rig.d_pool),
    lambda c: dict(d_lse=c.rig.d_starts), lambda c: dict(d_lse=c.lse.offset(2)),
])
def test_refused_by_attend(calls, change):
    with pytest.raises(native.SamplerError) as e:
        calls.attend(**change(calls))
    assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT


def test_views_that_lie_side_by_side(calls):
    """Queries, keys, values and rotated queries as parts of each token's record."""
    r = calls.rig
    n, wide = r.tokens, (2 * r.heads + 2 * r.kv) * r.d
    b = hip.Buffer(n * wide * 2)
    parts = [cache.View(b.offset(2 * r.d * h), wide, r.d)
             for h in (0, r.heads, r.heads + r.kv, r.heads + 2 * r.kv)]
    calls.append(q=parts[0], k=parts[1], v=parts[2], q_out=parts[3])
    hip.synchronize()
    with pytest.raises(native.SamplerError):
        calls.append(q=parts[0], k=parts[1], v=parts[2],
                     q_out=cache.View(b.offset(2 * r.d * (r.heads + 2 * r.kv - 1)), wide, r.d))


# --------------------------------------------------------- streams and graphs


@pytest.mark.parametrize("news", [None, [30, 1, 0, 16]])
def test_another_stream(news):
    st = hip.Stream(nonblocking=True)
    rig = Rig([40, 17, 0, 90], news=news, stream=st, slots=7)
    for _ in range(2):
        rig.append()
        rig.attend()
    rig.cache.close()
    st.destroy()


class Fixed:
    """Calls of one rig on memory that stays, as a graph records them."""

    def __init__(self, rig, window=0):
        self.rig, self.window = rig, window
        n, d = rig.tokens, rig.dtype
        zero = [np.zeros((n, h, rig.d)) for h in (rig.heads, rig.kv)]
        self.q, self.turned, self.out = (Vectors(zero[0], d) for _ in range(3))
        self.k, self.v = (Vectors(zero[1], d) for _ in range(2))
        self.lse = hip.Buffer(n * rig.heads * 4)
        self.at = dict(d_starts=rig.d_starts)

    def fill(self):
        """new vectors"""
        r = self.rig
        for x, h in ((self.q, r.heads), (self.k, r.kv), (self.v, r.kv)):
            x.put(x.raw, r.random(h))
            x.buf.upload(x.raw)
        self.out.buf.zero()
        hip.synchronize()

    def append(self):
        r = self.rig
        r.cache.append(r.state, r.rows, r.tokens, DTYPE[r.dtype], r.d_pool, *r.planes,
                       q=self.q.view, k=self.k.view, v=self.v.view, q_out=self.turned.view,
                       d_freqs=r.d_freqs, **self.at)

    def attend(self):
        r = self.rig
        r.cache.attend(r.state, r.rows, r.tokens, DTYPE[r.dtype], r.d_pool, *r.planes,
                       self.turned.view, self.out.view, r.d ** -0.5, self.window, d_lse=self.lse,
                       **self.at)

    def results(self):
        return (self.out.buf.download(np.uint8), self.lse.download(np.uint32),
                self.rig.d_pool.download(np.uint8), self.turned.buf.download(np.uint8))


@pytest.mark.parametrize("shape, window", [
    (dict(lengths=[60, 0, 33, 7]), 0),
    (dict(lengths=[2500, 2500, 2499], d=512, group=4, P=32, B=32, dtype="f32", share=(3, 70)), 0),
    (dict(lengths=[1600, 40, 7], news=[300, 1, 7], dtype="f32"), 500),
    (dict(lengths=[900], news=[300], d=128, kv=1, group=8), 0),
])
def test_captured_and_replayed(shape, window):
    """One graph that appends and attends, replayed on new vectors and other lengths, with eager
    calls of the same handle between: every replay gives what eager calls give."""
    st = hip.Stream(nonblocking=True)
    rig = Rig(stream=st, **shape)
    f = Fixed(rig, window)
    pool = rig.pool.copy()

    def run():
        f.append()
        f.attend()
    f.fill()
    run()
    st.synchronize()
    destroy, launch = _capture(st, run)
    second, again = _capture(st, f.attend)
    lengths = rig.lengths.copy()
    for i in range(4):
        rig.d_lengths.upload(np.maximum(lengths - i, 0).astype(I32))
        f.fill()
        rig.d_pool.upload(pool)
        run()
        st.synchronize()
        want = f.results()
        f.out.buf.zero()
        rig.d_pool.upload(pool)
        hip.synchronize()
        launch()
        st.synchronize()
        for a, b in zip(f.results(), want):
            assert np.array_equal(a, b)
        f.out.buf.zero()
        hip.synchronize()
        again()
        st.synchronize()
        for a, b in zip(f.results(), want):
            assert np.array_equal(a, b)
    destroy()
    second()
    rig.cache.close()
    st.destroy()


def test_two_handles_at_once():
    """Handles of their own on streams of their own, over one pool."""
    sts = [hip.Stream(nonblocking=True) for _ in range(2)]
    rig = Rig([3000, 700], d=128, slots=200)
    other = [cache.KvCache(rig.geo, rig.heads, rig.kv, rig.d, rig.B, rig.rotary, stream=s)
             for s in sts]
    own = rig.cache
    want = Fixed(rig)
    want.fill()
    want.turned.buf.upload(want.q.raw)
    want.attend()
    hip.synchronize()
    ref = want.results()[:2]
    fs = [Fixed(rig) for _ in other]
    for f in fs:
        f.turned.buf.upload(want.q.raw)
    hip.synchronize()
    for _ in range(20):
        for f, h in zip(fs, other):
            rig.cache = h
            f.attend()
    hip.synchronize()
    for f in fs:
        for a, b in zip(f.results()[:2], ref):
            assert np.array_equal(a, b)
    rig.cache = own
    for h in other:
        h.close()
    for s in sts:
        s.destroy()


# -------------------------------------------------------- with pages, together


class Steps:
    """A search: a page cache, two states that change places, a cache over the pool, and the
    oracles of both beside them."""

    def __init__(self, P, B, N, rows, slots, kv, group, d, dtype, seed=0):
        self.rng = np.random.default_rng(seed)
        self.P, self.B, self.rows, self.dtype, self.d = P, B, rows, dtype, d
        self.kv, self.heads = kv, kv * group
        self.geo = cache.geometry(P, N, rows, slots, kv, d)
        self.pages = beam.PageCache(P, N, rows, slots, 2, kv, d + 4)
        self.cache = cache.KvCache(self.geo, self.heads, kv, d, B)
        self.pool = np.full(self.geo.page_stride * N * 2, MARK, np.uint8)
        self.d_pool = hip.Buffer.from_array(self.pool)
        self.d_status = hip.Buffer(32)
        self.cur, self.next = (bo.State(rows, slots, N) for _ in range(2))
        self.dev = [self.upload(self.cur), self.upload(self.next)]
        self.freqs = (10000.0 ** (-np.arange(d // 2) / (d // 2))).astype(np.float32)
        self.d_freqs = hip.Buffer.from_array(self.freqs)

    def upload(self, s):
        bufs = [hip.Buffer.from_array(a) for a in (s.table, s.lengths, s.refs)]
        return bufs, beam.PageState(*bufs)

    def cells(self):
        return self.pool.reshape(2, self.geo.n_pages, self.kv, self.P, self.d + 4)

    def advance(self, parents, grow):
        d_par = hip.Buffer.from_array(np.asarray(parents, I32))
        d_grow = hip.Buffer.from_array(np.asarray(grow, I32))
        self.pages.advance(self.dev[0][1], self.rows, self.dev[1][1], self.rows, d_par, d_grow,
                           self.d_pool, self.d_status)
        hip.synchronize()
        status, copies = bo.advance(self.cur, self.rows, self.next, self.rows,
                                    np.asarray(parents, I32), np.asarray(grow, I32), self.P)
        assert status[0] == 0 and tuple(self.d_status.download(I32)[:4]) == tuple(status)
        v, old = self.cells(), self.cells().copy()
        for a, b, n in copies:
            v[:, b, :, :n] = old[:, a, :, :n]
        self.turn()

    def compact(self):
        self.pages.compact(self.dev[0][1], self.dev[1][1], self.rows, self.d_pool, self.d_status)
        hip.synchronize()
        status, copies = bo.compact(self.cur, self.next, self.rows, self.P)
        assert tuple(self.d_status.download(I32)[:4]) == tuple(status)
        v, old = self.cells(), self.cells().copy()
        for a, b in copies:  # (whole pages)
            v[:, b] = old[:, a]
        self.turn()

    def turn(self):
        self.cur, self.next = self.next, self.cur
        self.dev.reverse()
        assert np.array_equal(self.dev[0][0][1].download(I32), self.cur.lengths)

    def step(self, news, window=0):
        """The new tokens of each row, appended and attended over; None: one each."""
        n = self.rows if news is None else int(np.sum(news))
        starts = None if news is None else np.concatenate([[0], np.cumsum(news)]).astype(I32)
        d_starts = None if news is None else hip.Buffer.from_array(starts)
        x = {c: Vectors(self.rng.standard_normal((n, h, self.d)), self.dtype)
             for c, h in (("q", self.heads), ("k", self.kv), ("v", self.kv))}
        out = Vectors(x["q"].values(), self.dtype, mark=True)
        dt = DTYPE[self.dtype]
        q = x["q"].values()
        # the queries are rotated in their own place, and read from there
        self.cache.append(self.dev[0][1], self.rows, n, dt, self.d_pool, 0, 1, q=x["q"].view,
                          k=x["k"].view, v=x["v"].view, q_out=x["q"].view, d_starts=d_starts,
                          d_freqs=self.d_freqs)
        self.cache.attend(self.dev[0][1], self.rows, n, dt, self.d_pool, 0, 1, x["q"].view,
                          out.view, self.d ** -0.5, window, d_starts)
        hip.synchronize()
        cells = co.Cache(self.pool, self.geo, self.B)
        co.append(cells, self.cur.table, self.cur.lengths, starts, self.rows, n, q,
                  x["k"].values(), x["v"].values(), q.copy(), None, self.freqs, self.d, False,
                  (0, 1))
        raw = self.d_pool.download(np.uint8)
        got = co.Cache(raw, self.geo, self.B)
        P = self.P
        for r in range(self.rows):  # what rows hold: codes, and the scales that count
            for t in range(max(int(self.cur.lengths[r]), 0)):
                p, i = self.cur.table[r, t // P], t % P
                assert np.array_equal(got.codes[:, p, :, i], cells.codes[:, p, :, i]), (r, t)
                if i % self.B == 0:
                    assert np.array_equal(got.scales[:, p, :, i], cells.scales[:, p, :, i]), (r, t)
        self.pool = raw
        turned = x["q"].download()  # (what the attention has read)
        want = co.attend(got, self.cur.table, self.cur.lengths, starts, self.rows, n, turned,
                         np.float32(self.d ** -0.5), window, (0, 1))
        far = co.limits(want, self.d, self.dtype)[0]
        assert (np.abs(out.download() - want.out) <= far).all()


@pytest.mark.parametrize("P, B, kv, group, d, dtype", [
    (16, 4, 2, 4, 64, "bf16"), (8, 8, 1, 2, 128, "f32"), (5, 1, 2, 8, 32, "bf16"),
    (32, 16, 1, 3, 256, "f32")])
def test_search_steps(P, B, kv, group, d, dtype):
    """Prompts, then beams that fork and end and share pages whose scales their copies carry, then
    compacted pages and chunks of several tokens."""
    s = Steps(P, B, 300, 6, 40, kv, group, d, dtype)
    news = [37, 3, 0, 21, 1, 90]
    s.advance([-1] * 6, news)
    s.step(news)
    for i in range(P + 2):
        parents = np.sort(s.rng.integers(0, 6, 6)) if i % 3 == 1 else np.arange(6)
        s.advance(parents, np.where(s.cur.lengths[parents] > 0, 1, 0) if i % 5 else np.ones(6))
        s.step(None, window=0 if i % 2 else 24)
    s.compact()
    news = [5, 0, 40, 1, 2, 9]
    s.advance(np.arange(6), news)
    s.step(news)


# ---------------------------------------------------------------------- sizes


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [48, 64, 128, 256, 512])
@pytest.mark.parametrize("B", [1, 5, 16, 32, 128])
def test_append_tiles(d, B, dtype):
    """Tiles of a few and of many tokens, heads of a workgroup that do not come out even, blocks
    that earlier tokens have begun."""
    for pairs, rotary in (("halves", d), ("neighbours", d // 4 * 2), ("halves", d // 2 - 2)):
        rig = Rig([B * 2 + 3, 7, 150], news=[B + 2, 7, 133], P=2 * B, B=B, kv=3, group=1, d=d,
                  dtype=dtype, rotary=rotary, pairs=pairs, seed=B)
        rig.append()


def test_append_many_prompts():
    """So many prompts that a workgroup takes several groups of heads."""
    rig = Rig([7] * 400, news=[3, 2, 4, 1] * 100, P=8, B=4, kv=5, group=2, d=32, rotary=32)
    rig.append()


@pytest.mark.parametrize("news", [[1], [0], [2], [17], [40]])
def test_one_row_with_fewer_tokens_than_views(news):
    """One row among tokens that are no row's."""
    rig = Rig([90], news=news, kv=1, group=4)
    rig.tokens = 50
    rig.append()
    rig.attend()
    rig.attend(window=30)


@pytest.mark.parametrize("length", [-1, 7 * 16 + 1])
@pytest.mark.parametrize("news", [None, [1], [40]])
def test_one_row_whose_length_is_none(length, news):
    """NaN for all of its queries, and nothing appended."""
    rig = Rig([90], news=news, kv=1, group=4)
    rig.lengths[0] = length
    rig.upload()
    rig.append()
    rig.attend()


@pytest.mark.parametrize("d", [512, 128, 16])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_most_rows(d, dtype):
    rng = np.random.default_rng(d)
    lengths = rng.integers(0, 6, beam.PAGES_MAX_ROWS)
    rig = Rig(lengths, P=2, B=2, kv=1, group=2, d=d, dtype=dtype, share=(8, 1))
    rig.attend()
    rig = Rig(lengths, P=2, B=2, kv=1, group=1, d=d, dtype=dtype)
    rig.append()
    rig.attend(window=3)


def test_most_heads():
    rig = Rig([40, 9], news=[3, 1], P=256, B=256, kv=8, group=64, d=512, slots=1)
    rig.append()
    rig.attend()
    rig = Rig([33, 70], news=[30, 1], kv=64, group=8, d=16, dtype="f32")
    rig.append()
    rig.attend()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kv, group, d", [(1, 2, 512), (2, 1, 256), (1, 3, 128), (1, 2, 48)])
def test_prompts_of_many_tiles(kv, group, d, dtype):
    rig = Rig([700, 430], news=[150, 130], P=32, B=8, kv=kv, group=group, d=d, dtype=dtype)
    rig.attend()
    rig.attend(window=77)


@pytest.mark.parametrize("rows, group, d", [(16, 4, 64), (40, 2, 256), (90, 4, 128), (300, 8, 64),
                                            (24, 1, 512)])
def test_pages_that_part_and_meet(rows, group, d):
    """Rows that begin with one page and part anywhere, some of which share pages again behind
    that, of one length or of many."""
    rng = np.random.default_rng(rows)
    for case in range(3):
        n = 40
        lengths = np.full(rows, 4 * n - 3) if case == 0 else rng.integers(1, 4 * n, rows)
        rig = Rig(lengths, P=4, B=4, kv=1, group=group, d=d, share=(16, 1), spare=8)
        for r in range(rows):
            first = r - r % 16
            used = -(-int(lengths[r]) // 4)
            part = int(rng.integers(1, n))
            slots = np.arange(used) < part
            if case == 2:
                slots |= rng.random(used) < 0.5
            for s in np.nonzero(slots)[0]:
                if s < -(-int(lengths[first]) // 4) and 4 * (s + 1) <= min(lengths[first], lengths[r]):
                    rig.table[r, s] = rig.table[first, s]
        rig.upload()
        rig.attend()
        rig.attend(window=61)


def test_offsets_past_32_bits():
    """Pages 3 GiB apart: what is read and written lies where 64-bit offsets say."""
    P, B, kv, d, rows, slots = 8, 4, 2, 32, 2, 3
    stride, page = 3 << 30, kv * P * (d + 4)
    N, plane = 4, 4096
    geo = cache.geometry(P, N, rows, slots, kv, d, 2, plane_stride=plane, page_stride=stride)
    near = cache.geometry(P, N, rows, slots, kv, d, 2)
    rng = np.random.default_rng(1)
    d_far = hip.Buffer(stride * (N - 1) + plane + page)
    table = np.array([[3, 1, 0], [2, -1, -1]], I32)
    lengths = np.array([20, 6], I32)
    state = beam.PageState(hip.Buffer.from_array(table), hip.Buffer.from_array(lengths), None)
    codes = co.encode(rng.standard_normal((2, N, kv, P, d)) * 100)
    cells = np.zeros((2, N, kv, P, d + 4), np.uint8)
    cells[..., :d] = codes
    cells[..., d:] = np.full((2, N, kv, P, 1), 2.0 ** -6, np.float32).view(np.uint8)
    d_near = hip.Buffer.from_array(cells)
    for p in range(2):
        for i in range(N):
            d_far.upload(cells[p, i].reshape(-1), stride * i + plane * p)
    results = []
    for news in (None, np.array([11, 3])):
        n = rows if news is None else int(news.sum())
        starts = None if news is None else hip.Buffer.from_array(
            np.concatenate([[0], np.cumsum(news)]).astype(I32))
        x = [rng.standard_normal((n, h, d)) for h in (4, kv, kv)]
        for g, pool in ((geo, d_far), (near, d_near)):
            c = cache.KvCache(g, 4, kv, d, B, 0)
            q, k, v = (Vectors(y, "bf16") for y in x)
            out = Vectors(x[0], "bf16")
            c.append(state, rows, n, DTYPE["bf16"], pool, 1, 0, q=q.view, k=k.view, v=v.view,
                     q_out=q.view, d_starts=starts)
            c.attend(state, rows, n, DTYPE["bf16"], pool, 1, 0, q.view, out.view, 0.2, 0, starts)
            hip.synchronize()
            if pool is d_far:
                at = np.stack([np.stack([d_far.download(np.uint8, page, stride * i + plane * p)
                                         for i in range(N)]) for p in range(2)])
            else:
                at = d_near.download(np.uint8).reshape(2, N, page)
            results.append((out.buf.download(np.uint8), at))
            c.close()
        for a, b in zip(*results[-2:]):
            assert np.array_equal(a, b)
    d_far.free()
