"""GPU tests of the 8-bit cache (g4s_cache_*) against the token-by-token
restatement in cache_oracle.py.  Codes and scales are equal or wrong; outputs in
floating point stay within what cache_oracle.limits derives."""
import numpy as np
import pytest

import cache_oracle as co
from gemma4_sampler import beam, cache, hip, native

pytestmark = pytest.mark.gpu
I32 = np.int32
MARK = 0x5A  # what memory holds that no call may write


def bf16(x):
    """to bf16 (ties to even) as uint16"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = (u + 0x7FFF + (u >> 16 & 1)) >> 16
    return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)


def widen(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


class Vectors:
    """Vectors [tokens, heads, dim] in device memory, with strides of their own."""

    def __init__(self, x, dtype, layout="tokens", pad=0, mark=False):
        n, heads, d = x.shape
        self.dtype, self.n, self.heads, self.d = dtype, n, heads, d
        d1 = d + pad
        if layout == "tokens":
            self.ts, self.hs = heads * d1 + pad, d1
        else:
            self.ts, self.hs = d1, n * d1 + pad
        self.size = (n - 1) * self.ts + (heads - 1) * self.hs + d
        self.raw = np.full(self.size * (4 if dtype == "f32" else 2), MARK, np.uint8)
        if not mark:
            self.put(self.raw, x)
        self.buf = hip.Buffer.from_array(self.raw)
        self.view = cache.View(self.buf, self.ts, self.hs)

    def cells(self, raw):
        t = np.float32 if self.dtype == "f32" else np.uint16
        size = np.dtype(t).itemsize
        return np.lib.stride_tricks.as_strided(
            raw.view(t), (self.n, self.heads, self.d), (self.ts * size, self.hs * size, size))

    def put(self, raw, x):
        self.cells(raw)[...] = x if self.dtype == "f32" else bf16(x)

    def values(self):
        """what the vectors hold, in 64 bits"""
        c = self.cells(self.raw)
        return (c if self.dtype == "f32" else widen(c)).astype(np.float64)

    def download(self):
        raw = self.buf.download(np.uint8)
        c = self.cells(raw)
        v = (c if self.dtype == "f32" else widen(c)).astype(np.float64)
        rest = raw.copy()
        self.cells(rest)[...] = self.cells(np.full_like(raw, MARK))
        assert (rest == MARK).all(), "bytes between the vectors were written"
        return v


class Rig:
    """A cache, its pool and one state, beside the oracle's."""

    def __init__(self, lengths, news=None, P=16, B=4, kv=2, group=4, d=64, rotary=None,
                 pairs="halves", dtype="bf16", planes=3, order=(2, 0), seed=0, slots=None,
                 outer=False, spare=3, stream=None, share=None):
        self.rng = rng = np.random.default_rng(seed)
        self.P, self.B, self.kv, self.heads, self.d, self.dtype = P, B, kv, kv * group, d, dtype
        self.lengths = np.asarray(lengths, I32)
        self.rows = len(self.lengths)
        used = -(-np.maximum(self.lengths, 0) // P)
        self.slots = int(max(used.max(), 1)) + 1 if slots is None else slots
        n_pages = int(used.sum()) + spare
        self.table = np.full((self.rows, self.slots), -7, I32)
        free = list(rng.permutation(n_pages))
        for r in range(self.rows):
            for s in range(used[r]):
                self.table[r, s] = free.pop()
        if share:  # rows in groups of share[0] have their first share[1] pages in common
            for r in range(self.rows):
                n = min(share[1], used[r], used[r - r % share[0]])
                self.table[r, :n] = self.table[r - r % share[0], :n]
        page = kv * P * (d + 4)
        strides = dict(plane_stride=page, page_stride=page * planes) if outer else {}
        self.geo = cache.geometry(P, n_pages, self.rows, self.slots, kv, d, planes, **strides)
        self.rotary = d if rotary is None else rotary
        self.pairs, self.planes = pairs, order
        self.cache = cache.KvCache(self.geo, self.heads, kv, d, B, self.rotary, pairs,
                                   stream=stream)
        self.news = None if news is None else np.asarray(news)
        self.starts = None if news is None else \
            np.concatenate([[0], np.cumsum(self.news)]).astype(I32)
        self.tokens = self.rows if news is None else int(self.starts[-1])
        self.pool = self.random_pool(planes, n_pages)
        self.d_pool = hip.Buffer.from_array(self.pool)
        self.freqs = (10000.0 ** (-np.arange(self.rotary // 2) /
                                  max(self.rotary // 2, 1))).astype(np.float32)
        self.upload()

    def upload(self):
        self.d_table = hip.Buffer.from_array(self.table)
        self.d_lengths = hip.Buffer.from_array(self.lengths)
        self.state = beam.PageState(self.d_table, self.d_lengths, None)
        self.d_starts = None if self.starts is None else hip.Buffer.from_array(self.starts)
        self.d_freqs = hip.Buffer.from_array(self.freqs) if len(self.freqs) else None

    def random_pool(self, planes, n_pages):
        """Any finite codes, small scales; where no token is, NaN codes and scales."""
        rng, d = self.rng, self.d
        cells = np.full((planes, n_pages, self.kv, self.P, d + 4), 0xFF, np.uint8)
        live = np.zeros((n_pages, self.P), bool)
        for r in range(self.rows):
            for t in range(max(int(self.lengths[r]), 0)):
                live[self.table[r, t // self.P], t % self.P] = True
        codes = co.encode(rng.standard_normal((planes, n_pages, self.kv, self.P, d)) * 100)
        scales = 2.0 ** rng.integers(-8, -5, (planes, n_pages, self.kv, self.P, 1))
        cells[..., :d] = np.where(live[:, None, :, None], codes, 0xFF)
        cells[..., d:] = np.where(live[:, None, :, None],
                                  scales.astype(np.float32).view(np.uint8), 0xFF)
        if self.geo.page_stride > self.geo.plane_stride:
            cells = np.ascontiguousarray(cells.swapaxes(0, 1))
        return cells.reshape(-1)

    def random(self, heads, size=1.0):
        return self.rng.standard_normal((self.tokens, heads, self.d)) * size

    # ------------------------------------------------------------- append

    def append(self, positions=None, q=True, kv=True, layout="tokens", pad=0, inplace=False,
               edit=None, run=None):
        """One append, compared.  `edit` changes the vectors before the upload, `run` makes the
        call otherwise."""
        x = dict(q=self.random(self.heads), k=self.random(self.kv, 3.0),
                 v=self.random(self.kv, 0.01))
        if edit:
            edit(x)
        vq = Vectors(x["q"], self.dtype, layout, pad) if q else None
        vo = (vq if inplace else Vectors(x["q"], self.dtype, layout, 2 * pad, mark=True)) if q \
            else None
        vk, vv = (Vectors(x[n], self.dtype, layout, pad) for n in "kv") if kv else (None, None)
        d_pos = None if positions is None else hip.Buffer.from_array(np.asarray(positions, I32))
        before = co.Cache(self.pool, self.geo, self.B)

        def call():
            self.cache.append(self.state, self.rows, self.tokens,
                              native.DTYPE_F32 if self.dtype == "f32" else native.DTYPE_BF16,
                              self.d_pool if kv else None, self.planes[0], self.planes[1],
                              q=vq and vq.view, k=vk and vk.view, v=vv and vv.view,
                              q_out=vo and vo.view, d_starts=self.d_starts, d_positions=d_pos,
                              d_freqs=self.d_freqs)
        (run or (lambda c: c()))(call)
        hip.synchronize()
        q_out = vo.values().copy() if q else None
        co.append(before, self.table, self.lengths, self.starts, self.rows, self.tokens,
                  vq.values() if q else None, vk.values() if kv else None,
                  vv.values() if kv else None, q_out, positions, self.freqs, self.rotary,
                  self.pairs == "neighbours", self.planes)
        raw = self.d_pool.download(np.uint8)
        got = co.Cache(raw, self.geo, self.B)
        same = (got.codes == before.codes) | ((got.codes & 127 == 127) & (before.codes & 127 == 127))
        assert same.all(), np.argwhere(~same)[:5]
        assert np.array_equal(got.scales.view(np.uint32), before.scales.view(np.uint32))
        self.pool = raw
        if q:
            half = np.finfo(np.float32).eps / 2 if self.dtype == "f32" else 2.0 ** -8
            err = np.abs(vo.download() - q_out)
            # (1e-15: what angles and products in 64 bits are off by)
            assert (err <= half * np.abs(q_out) + 1e-14 * (1 + np.abs(vq.values()).max())).all()
        return got

    # ------------------------------------------------------------- attend

    def attend(self, window=0, scale=None, lse=True, layout="tokens", pad=0, edit=None, run=None,
               size=1.0):
        x = self.random(self.heads, size)
        if edit:
            edit(x)
        scale = self.d ** -0.5 if scale is None else scale
        vq = Vectors(x, self.dtype, layout, pad)
        vo = Vectors(x, self.dtype, layout, 2 * pad, mark=True)
        d_lse = hip.Buffer.from_array(np.full((self.tokens, self.heads), 77.0, np.float32))

        def call():
            self.cache.attend(self.state, self.rows, self.tokens,
                              native.DTYPE_F32 if self.dtype == "f32" else native.DTYPE_BF16,
                              self.d_pool, self.planes[0], self.planes[1], vq.view, vo.view, scale,
                              window, self.d_starts, d_lse if lse else None)
        (run or (lambda c: c()))(call)
        hip.synchronize()
        want = co.attend(co.Cache(self.pool, self.geo, self.B), self.table, self.lengths,
                         self.starts, self.rows, self.tokens, vq.values(), np.float32(scale),
                         window, self.planes)
        assert np.array_equal(self.d_pool.download(np.uint8), self.pool)
        out, got_lse = vo.download(), d_lse.download(np.float32).reshape(self.tokens, self.heads)
        had = np.zeros(self.tokens, bool)
        for r in range(self.rows):
            a, b = (r, r + 1) if self.starts is None else self.starts[r:r + 2]
            had[a:b] = True
        mark = Vectors(x, self.dtype, mark=True).values()[0, 0, 0]
        assert (out[~had] == mark).all() and (got_lse[~had] == 77.0).all()
        far_out, far_lse = co.limits(want, self.d, self.dtype)

        def check(got, ref, far):
            nan = np.isnan(ref)
            assert np.array_equal(np.isnan(got), nan)
            inf = np.isinf(ref)
            assert np.array_equal(got[inf], ref[inf])
            fine = ~nan & ~inf
            off = np.abs(got - np.where(fine, ref, 0.0))[fine]
            assert (off <= far[fine]).all(), (off / far[fine]).max()
        check(out[had], want.out[had], far_out[had])
        if lse:
            check(got_lse[had].astype(np.float64), want.lse[had], far_lse[had])
        return out


# ------------------------------------------------------------------- append

SHAPES = [
    dict(lengths=[1]), dict(lengths=[5, 0, 17, 16]),
    dict(lengths=[37, 4, 20], news=[13, 4, 0]),
    dict(lengths=[70, 0, 33, 2], news=[50, 3, 33, 7]),
    dict(lengths=[29, 40], news=[9, 11], P=9, B=3, kv=3, group=1, d=80, dtype="f32"),
    dict(lengths=[100], news=[60], P=64, B=64, kv=1, group=8, d=128),
    dict(lengths=[21, 22], news=[5, 2], P=1, B=1, d=16, dtype="f32"),
    dict(lengths=[300, 17], news=[290, 1], P=100, B=50, kv=1, group=2, d=96, rotary=40),
    dict(lengths=[33, 64], news=[30, 1], kv=2, group=1, d=256, rotary=128, pairs="neighbours"),
    dict(lengths=[19, 34], d=512, kv=2, group=2, dtype="f32", B=16),
    dict(lengths=[19, 34], news=[2, 3], d=512, kv=1, group=3, B=16, rotary=0),
    dict(lengths=[40], news=[23], d=112, kv=4, group=2, B=1, rotary=22, dtype="f32", outer=True),
    dict(lengths=[600], news=[530], P=256, B=256, kv=1, group=1, d=16, rotary=6,
         pairs="neighbours"),
]


@pytest.mark.parametrize("shape", SHAPES)
def test_append(shape):
    rig = Rig(**shape)
    rig.append()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout, pad", [("tokens", 8), ("heads", 0), ("heads", 16)])
def test_append_strides(dtype, layout, pad):
    rig = Rig([30, 8, 50], news=[7, 3, 20], dtype=dtype, seed=3)
    rig.append(layout=layout, pad=pad)
    rig.append(layout=layout, pad=pad, inplace=True)


def test_append_one_side():
    """Queries alone, and keys and values alone."""
    rig = Rig([30, 8, 50], news=[7, 3, 20], seed=4)
    rig.append(kv=False)
    rig.append(q=False)


@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
def test_append_far_positions(pairs):
    rig = Rig([30, 8], news=[7, 3], dtype="f32", pairs=pairs)
    rig.append(positions=[0, 1, -1, (1 << 31) - 1, -(1 << 31), 1000003, 131071, 5, 99999999, 0])


def test_append_token_by_token():
    """Blocks filled one token at a time, their scales growing under their earlier codes."""
    rig = Rig([1, 14, 30], P=16, B=8, dtype="f32", slots=4, spare=12)
    for r in range(rig.rows):
        for s in range(rig.slots):
            if rig.table[r, s] < 0:
                rig.table[r, s] = next(p for p in range(rig.geo.n_pages) if p not in rig.table)
    for step in range(9):
        rig.upload()

        def edit(x):
            x["k"] *= 4.0 ** step
            x["v"] *= 0.25 ** step
        rig.append(edit=edit)
        rig.lengths += 1


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_odd_values(dtype):
    """Zeros, infinities, NaN, the smallest and the largest numbers, borders of codes."""
    rig = Rig([40, 33], news=[40, 20], B=4, dtype=dtype, rotary=0, d=16)

    def edit(x):
        v = x["v"]
        v[0:4] = 0.0
        v[4, 0, 3], v[5, 1, 2], v[9, 0, 0] = np.inf, -np.inf, np.nan
        v[12:16] = np.nan
        v[16:20] = -np.inf
        v[20:24] = 1e-42
        v[24:28] = 3e38
        v[28:32] = 2.0 ** -110
        k = x["k"]
        k[:, :, :] = np.sign(k) * co.E4M3[np.arange(k.size).reshape(k.shape) % 127] * \
            np.where(np.arange(k.size).reshape(k.shape) % 2, 1.0, 17 / 16)
        k[8:12] = 448.0
        k[12:16] = 450.0
    with np.errstate(all="ignore"):
        rig.append(edit=edit)


def test_append_pages_outside_the_pool():
    """Tokens whose page is no page are left out, the others are not; rows whose length is
    no length are left out, queries too."""
    rig = Rig([40, 20, 60, 8], news=[30, 20, 9, 8])
    rig.table[0, 1], rig.table[1, 0], rig.table[2, 3] = -1, rig.geo.n_pages, 1 << 30
    rig.upload()
    rig.append()
    rig.lengths[1], rig.lengths[3] = rig.slots * rig.P + 1, -1
    rig.upload()
    rig.append()


def test_append_starts_that_do_not_fit():
    rig = Rig([40, 20, 60], news=[5, 5, 5])
    rig.starts[:] = [0, 5, 4, 16]  # the second row has -1 tokens, the third too many
    rig.upload()
    rig.starts = np.array([0, 5, 5, 5], I32)
    # the other rows' tokens are those of no row
    rig.append(edit=None)


# ------------------------------------------------------------------- attend

SEEN = [
    dict(lengths=[1]), dict(lengths=[501], d=256, B=1), dict(lengths=[5, 0, 17, 16, 64]),
    dict(lengths=[1500, 3, 700], dtype="f32", d=128, kv=1, group=3),
    dict(lengths=[37, 4, 20], news=[13, 4, 0]),
    dict(lengths=[70, 0, 33, 2], news=[50, 3, 33, 7], dtype="f32"),
    dict(lengths=[129, 140], news=[129, 11], P=9, B=3, kv=3, group=1, d=80, dtype="f32"),
    dict(lengths=[200], news=[160], P=64, B=64, kv=1, group=8, d=128),
    dict(lengths=[21, 22], news=[5, 2], P=1, B=1, d=16, dtype="f32"),
    dict(lengths=[300, 17], news=[90, 1], P=100, B=50, kv=1, group=2, d=96),
    dict(lengths=[133, 64], news=[70, 1], kv=2, group=1, d=256),
    dict(lengths=[133, 64], news=[37, 1], kv=2, group=2, d=192, dtype="f32"),
    dict(lengths=[219, 34], d=512, kv=2, group=2, dtype="f32", B=16),
    dict(lengths=[119, 34], news=[25, 3], d=512, kv=1, group=3, B=16),
    dict(lengths=[119, 34], news=[25, 3], d=512, kv=1, group=2, B=16, dtype="f32"),
    dict(lengths=[75, 90], d=112, kv=1, group=17, B=1, outer=True),
    dict(lengths=[75, 90], d=64, kv=1, group=64, B=2, dtype="f32"),
    dict(lengths=[40, 41], news=[3, 2], d=64, kv=2, group=5),
]


@pytest.mark.parametrize("window", [0, 1, 33])
@pytest.mark.parametrize("shape", SEEN)
def test_attend(shape, window):
    Rig(**shape).attend(window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout, pad", [("tokens", 8), ("heads", 0), ("heads", 16)])
def test_attend_strides(dtype, layout, pad):
    Rig([30, 8, 90], news=[7, 3, 80], dtype=dtype, seed=3).attend(layout=layout, pad=pad)
    Rig([30, 8, 90], dtype=dtype, seed=3).attend(layout=layout, pad=pad, lse=False)


@pytest.mark.parametrize("scale", [0.0, -0.5, 3.0, 1e-30])
@pytest.mark.parametrize("news", [None, [60, 1]])
def test_attend_scales(scale, news):
    Rig([100, 7], news=news, dtype="f32").attend(scale=scale)


@pytest.mark.parametrize("news", [None, [9, 60, 2, 6]])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_bad_rows_and_pages(dtype, news):
    """A length that is none, a page that is none: NaN for who sees it, nobody else."""
    rig = Rig([40, 90, 60, 8], news=news, dtype=dtype)
    rig.lengths[0] = rig.slots * rig.P + 1
    rig.table[1, 4] = -1
    rig.table[2, 1] = rig.geo.n_pages
    rig.upload()
    rig.attend()
    rig.attend(window=20)


@pytest.mark.parametrize("news", [None, [30, 40]])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 16])
def test_attend_nan_in_the_cache(dtype, news, window):
    """NaN keys and values: for the queries that see them alone, values in their dims alone."""
    rig = Rig([50, 70], news=news, dtype=dtype, kv=2, group=3)
    cells = rig.pool.reshape(3, rig.geo.n_pages, rig.kv, rig.P, rig.d + 4)
    k, v = cells[rig.planes[0]], cells[rig.planes[1]]
    for row, t, dim in ((0, 30, 5), (0, 49, 63), (1, 2, 0), (1, 66, 17)):
        v[rig.table[row, t // rig.P], 0, t % rig.P, dim] = 0x7F
    k[rig.table[1, 40 // rig.P], 1, 40 % rig.P, 3] = 0xFF
    rig.d_pool.upload(rig.pool)
    rig.attend(window)


@pytest.mark.parametrize("news", [None, [30, 40]])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_odd_queries(dtype, news):
    """Infinite and NaN queries; zeros; scores far apart."""
    rig = Rig([50, 70], news=news, dtype=dtype)

    def edit(x):
        x[0, 0, 3], x[0, 1, 0], x[1, 2, 5] = np.inf, np.nan, -np.inf
        x[-1, 3] = 0.0
        x[-1, 4] *= 300.0
    with np.errstate(all="ignore"):
        rig.attend(edit=edit)


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("share", [(2, 3), (3, 100), (4, 9), (5, 2), (16, 6), (40, 4)])
@pytest.mark.parametrize("kv, group, d, dtype", [(2, 4, 64, "bf16"), (1, 1, 128, "f32"),
                                                 (1, 5, 256, "bf16"), (2, 8, 80, "f32"),
                                                 (1, 2, 512, "bf16"), (1, 16, 64, "bf16")])
def test_attend_shared_pages(kv, group, d, dtype, share, window):
    """Rows that have their first pages in common, equally long or not."""
    lengths = [150 + (r // share[0]) * 37 + (r % 3 if share[0] != 4 else 0) for r in range(21)]
    lengths[9], lengths[14] = 0, 20
    Rig(lengths, P=16, B=8, kv=kv, group=group, d=d, dtype=dtype, share=share).attend(window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_shared_pages_of_all_kinds(dtype):
    """A page that is none and NaN values in shared and in own pages, rows of several tokens
    beside them."""
    rig = Rig([90, 90, 91, 92, 70, 70, 70, 70, 33], news=[1, 1, 1, 1, 1, 2, 1, 1, 3], dtype=dtype,
              share=(4, 3))
    cells = rig.pool.reshape(3, rig.geo.n_pages, rig.kv, rig.P, rig.d + 4)
    v = cells[rig.planes[1]]
    v[rig.table[0, 1], 0, 3, 7] = 0x7F       # seen by the first four
    v[rig.table[2, 4], 1, 5, 9] = 0xFF       # by the third alone
    rig.d_pool.upload(rig.pool)
    rig.table[6, 2], rig.table[3, 5] = -1, rig.geo.n_pages
    rig.upload()
    rig.attend()
    rig.attend(window=40)


@pytest.mark.parametrize("shape", [
    dict(lengths=[2500, 2500, 2499], d=512, group=4, P=32, B=32, dtype="f32", share=(3, 70)),
    dict(lengths=[7000], d=256, group=16, kv=1, P=64, B=4),
    dict(lengths=[3000, 10, 2000], news=[4, 1, 2], d=512, group=4, kv=1, P=64, slots=400)])
def test_attend_parts_joined_by_their_own_launch(shape):
    """Parts of more than a workgroup joins by itself."""
    rig = Rig(**shape)
    rig.attend()
    rig.attend(window=1700)
    rig.attend()


def test_attend_many_rows():
    """More rows than a workgroup has threads, in groups or alone, some ended."""
    rng = np.random.default_rng(5)
    lengths = rng.integers(0, 40, 1300)
    lengths[rng.random(1300) < 0.2] = 0
    Rig(lengths, P=8, B=8, kv=1, group=4, d=16, share=(4, 2)).attend()
    Rig(lengths[:700], news=rng.integers(0, 3, 700), P=8, B=8, kv=1, group=4, d=16).attend()


def test_attend_same_bits():
    """The same call gives the same bits, also where its work is split."""
    for shape in (dict(lengths=[3000], d=128), dict(lengths=[900, 40], news=[300, 1], dtype="f32")):
        a = Rig(**shape).attend()
        b = Rig(**shape).attend()
        assert np.array_equal(a, b)
