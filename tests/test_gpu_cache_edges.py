"""GPU tests of the 8-bit cache at the borders of its kernels' ranges: rows of several blocks
of query columns, and the calls that follow on the same handle."""
import numpy as np
import pytest

import cache_oracle as co
from gemma4_sampler import beam, cache, hip, native
from test_gpu_cache import Rig, Vectors
from test_gpu_cache_use import Calls

pytestmark = pytest.mark.gpu


def single_tokens(rig):
    """The rig's rows with one query each from here on, by the same handle."""
    rig.news = rig.starts = rig.d_starts = None
    rig.tokens = rig.rows


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [192, 256, 512])
@pytest.mark.parametrize("group, new", [(1, 17), (4, 6), (8, 4), (3, 11), (1, 48), (8, 6), (7, 7)])
def test_rows_of_several_blocks_of_columns(group, new, d, dtype):
    """17 to 49 columns a row in tables that the rows fill, and single tokens behind them."""
    for lengths, news in (([64], [new]), ([992, 500, 64], [new, 1, new]), ([300] * 5, [new] * 5)):
        rig = Rig(lengths, news=news, kv=1, group=group, d=d, dtype=dtype, slots=-(-max(lengths) // 16))
        rig.attend()
        rig.attend(window=40)
        single_tokens(rig)
        rig.attend()
        rig.attend(window=40)


@pytest.mark.parametrize("kv, group, new, length, d, dtype", [
    (2, 4, 6, 8100, 256, "bf16"), (2, 4, 10, 3000, 256, "f32"), (1, 8, 3, 8100, 256, "f32"),
    (1, 8, 4, 8100, 512, "bf16"), (2, 4, 8, 500, 512, "f32")])
def test_few_new_tokens_behind_long_contexts(kv, group, new, length, d, dtype):
    rig = Rig([length], news=[new], P=64, B=32, kv=kv, group=group, d=d, dtype=dtype,
              slots=8192 // 64 if length > 2000 else 9)
    for _ in range(2):
        rig.attend()
    single_tokens(rig)
    for _ in range(2):
        rig.attend()


# ----------------------------------------------- what a query does not see

SCALES = [0xFFFFFFFF, 0x7F800000, 0x7F000000, 0xFF800000, 0x7FC00000]


def cells(rig):
    return rig.pool.reshape(3, rig.geo.n_pages, rig.kv, rig.P, rig.d + 4)


def unwritten_first_page(rig, bits):
    """Page 0 becomes no row's, with codes that are numbers and scales that are none."""
    c = cells(rig)
    spare = next(p for p in range(1, rig.geo.n_pages) if p not in rig.table)
    c[:, spare] = c[:, 0]
    rig.table[rig.table == 0] = spare
    c[:, 0, ..., :rig.d] = co.encode(rig.rng.standard_normal(c[:, 0, ..., :rig.d].shape) * 100)
    c[:, 0, ..., rig.d:] = np.full(c.shape[2:4] + (1,), bits, np.uint32).view(np.uint8)
    rig.d_pool.upload(rig.pool)


def scales_that_are_none_give_nan(monkeypatch, rig):
    """The oracle's values under a scale that is no number from 0 to 2^119, in either plane."""
    plain = co.Cache.value

    def value(self, plane, table, row, t, head):
        at = self.place(table, row, t)
        if at is not None:
            page, o = at
            for p in rig.planes:
                if not 0 <= self.scales[p, page, head, o - o % self.block] <= 2.0 ** 119:
                    return np.full(self.d, np.nan)
        return plain(self, plane, table, row, t, head)
    monkeypatch.setattr(co.Cache, "value", value)


@pytest.mark.parametrize("bits", SCALES)
@pytest.mark.parametrize("shape, bad", [
    (dict(lengths=[70, 53], news=[40, 10], group=4), [(0, 3), (1, 3)]),
    (dict(lengths=[53, 30], news=[10, 1], group=1, d=256), [(0, 3)]),
    (dict(lengths=[90, 90, 91, 92], group=2, d=512, share=(4, 3)), [(1, 4), (3, 3)]),
    (dict(lengths=[150], news=[100], kv=1, group=1, d=512), [(0, 5)]),
    (dict(lengths=[150], news=[120], kv=1, group=1, d=256), [(0, 5)])])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pages_outside_the_pool_and_an_unwritten_first_page(dtype, shape, bad, bits):
    """Whoever does not see the page is not touched by what stands in another one."""
    rig = Rig(dtype=dtype, **shape)
    unwritten_first_page(rig, bits)
    for row, slot in bad:
        rig.table[row, slot] = -1 if slot % 2 else rig.geo.n_pages
    rig.upload()
    rig.attend()
    rig.attend(window=20)


@pytest.mark.parametrize("bits", SCALES)
@pytest.mark.parametrize("plane", [0, 1])
@pytest.mark.parametrize("shape, at", [
    (dict(lengths=[70, 53], news=[40, 10], group=4), [(0, 50), (1, 50)]),
    (dict(lengths=[53, 30], news=[10, 1], group=1, d=256), [(0, 48)]),
    (dict(lengths=[90, 90, 91, 92], group=2, d=512, share=(4, 3)), [(1, 70), (3, 91)]),
    (dict(lengths=[100, 40], group=2, d=64), [(0, 99), (1, 0)]),
    (dict(lengths=[150], news=[100], kv=1, group=1, d=512), [(0, 90)])])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.filterwarnings("ignore:invalid value")
def test_scales_that_are_none(monkeypatch, dtype, shape, at, plane, bits):
    """NaN for who sees a token under such a scale, nobody else."""
    rig = Rig(dtype=dtype, **shape)
    c = cells(rig)
    for row, t in at:
        t -= t % rig.B
        c[rig.planes[plane], rig.table[row, t // rig.P], 0, t % rig.P, rig.d:] = \
            np.full(1, bits, np.uint32).view(np.uint8)
    rig.d_pool.upload(rig.pool)
    scales_that_are_none_give_nan(monkeypatch, rig)
    rig.attend()
    rig.attend(window=20)


@pytest.mark.parametrize("bits", SCALES)
@pytest.mark.parametrize("group, d, dtype", [(4, 64, "bf16"), (2, 256, "f32"), (1, 512, "bf16")])
@pytest.mark.filterwarnings("ignore:invalid value")
def test_slots_that_the_window_has_left_behind(group, d, dtype, bits):
    """Rows of one first page and different lengths: slots between their windows name an
    unwritten page."""
    rig = Rig([60, 400, 399, 250], group=group, d=d, dtype=dtype, share=(4, 1))
    unwritten_first_page(rig, bits)
    for row, length in enumerate(rig.lengths):
        rig.table[row, 1:(length - 20) // rig.P] = 0 if row % 2 else -1
    rig.upload()
    rig.attend(window=20)


# ------------------------------------------------- roundings of bf16 outputs


def two_pieces(to, dim, dtype):
    """cache_oracle.limits where the weights of bf16 outputs are kept in two bf16 pieces: what
    the first one leaves is at most 2^-8 of a weight, and the second is off by 2^-8 of that."""
    out, lse = plain_limits(to, dim, dtype)
    return out - (2.0 ** -8 - 2.0 ** -16) * to.mass, lse


plain_limits = co.limits


@pytest.mark.parametrize("window", [0, 33])
@pytest.mark.parametrize("shape", [
    dict(lengths=[501], d=256, B=1), dict(lengths=[1500, 3, 700], d=128, kv=1, group=3),
    dict(lengths=[150, 150, 151, 149], d=512, group=2, share=(4, 6)), dict(lengths=[90] * 5, share=(5, 3)),
    dict(lengths=[200], news=[160], P=64, B=64, kv=1, group=8, d=128),
    dict(lengths=[129, 140], news=[129, 11], P=9, B=3, kv=3, group=1, d=80),
    dict(lengths=[300, 17], news=[90, 1], kv=1, group=2, d=64),
    dict(lengths=[333, 64], news=[70, 1], kv=2, group=1, d=256),
    dict(lengths=[219, 34], news=[55, 3], d=512, kv=1, group=3, B=16)])
def test_weights_of_bf16_outputs(monkeypatch, shape, window):
    """Outputs near zero under values that are not: the weights are not rounded to bf16."""
    monkeypatch.setattr(co, "limits", two_pieces)
    Rig(dtype="bf16", **shape).attend(window, size=0.5)


# ------------------------------------------------------------------ refusals


@pytest.fixture(scope="module")
def calls():
    return Calls()


def refused(call, **change):
    with pytest.raises(native.SamplerError) as e:
        call(**change)
    assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT
    return str(e.value)


@pytest.mark.parametrize("by", [1, 2, 3])
def test_addresses_between_integers(calls, by):
    r = calls.rig
    for name, change in (
            ("table", dict(state=beam.PageState(r.d_table.offset(by), r.d_lengths, None))),
            ("lengths", dict(state=beam.PageState(r.d_table, r.d_lengths.offset(by), None))),
            ("d_starts", dict(d_starts=r.d_starts.offset(by)))):
        for call in (calls.append, calls.attend):
            assert name in refused(call, **change)
    assert "d_positions" in refused(calls.append, d_positions=calls.positions.offset(by))
    assert "d_freqs" in refused(calls.append, d_freqs=r.d_freqs.offset(by))


# ---------------------------------------------------------- scales of scores


@pytest.mark.parametrize("news", [None, [60, 1]])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.0, 1e-38, -3e-38, 1e-40])
def test_small_scales_of_large_products(scale, dtype, news):
    """Products of queries and keys next to the largest number: a scale of 0 is one, and a
    tiny one is not rounded up."""
    Rig([100, 7], news=news, dtype=dtype).attend(scale=scale, size=2e35)


@pytest.mark.parametrize("news", [None, [60, 1]])
def test_largest_scale(news):
    Rig([100, 7], news=news).attend(scale=2.0 ** 127, size=0.0)


@pytest.mark.parametrize("scale", [2.4e38, -3e38])
def test_scales_that_are_too_large_to_base_two(calls, scale):
    assert "scale" in refused(calls.attend, scale=scale)


# --------------------------------------------------- parts of a head's record


def test_views_that_lie_side_by_side_in_each_head():
    """Keys, values and queries of each head one behind the other, queries rotated in place: taken, and
    what views of their own give."""
    r = Rig([20, 9, 30], news=[5, 9, 2], kv=3, group=1, d=64)
    n, d = r.tokens, r.d
    x = r.rng.standard_normal((n, 3, 3, d))  # token, head, part
    qkv = Vectors(x.reshape(n, 9, d), "bf16")
    parts = [cache.View(qkv.buf.offset(2 * d * i), 9 * d, 3 * d) for i in range(3)]
    apart = [Vectors(x[:, :, i], "bf16") for i in range(3)]
    pools = []
    for k, v, q in (parts, [a.view for a in apart]):
        r.d_pool.upload(r.pool)
        r.cache.append(r.state, r.rows, n, native.DTYPE_BF16, r.d_pool, *r.planes, q=q, k=k, v=v, q_out=q,
                       d_starts=r.d_starts, d_freqs=r.d_freqs)
        hip.synchronize()
        pools.append(r.d_pool.download(np.uint8))
    assert np.array_equal(*pools) and not np.array_equal(pools[0], r.pool)
    got = qkv.download().reshape(n, 3, 3, d)
    for i in range(3):
        assert np.array_equal(got[:, :, i], apart[i].download()), i
    beside = cache.View(qkv.buf.offset(2 * d + 16), 9 * d, 3 * d)
    assert "overlaps" in refused(r.cache.append, state=r.state, rows=r.rows, tokens=n,
                                 dtype=native.DTYPE_BF16, d_pool=r.d_pool, k_plane=2, v_plane=0,
                                 q=parts[2], k=parts[0], v=parts[1], q_out=beside,
                                 d_starts=r.d_starts, d_freqs=r.d_freqs)


# ------------------------------------------------------------- largest sizes


def page_values(rng, P, d, size):
    """A page of one head: its cells, and what its tokens stand for."""
    codes = co.encode(rng.standard_normal((P, d)) * size)
    cells = np.zeros((P, d + 4), np.uint8)
    cells[:, :d] = codes
    cells[:, d:] = np.full((P, 1), 2.0 ** -5, np.float32).view(np.uint8)
    return cells, co.E4M3[codes] * 2.0 ** -5


@pytest.mark.parametrize("rows, new, window", [(1, 1, 0), (4, 1, 0), (1, 1, 70000), (4, 1, 70000),
                                               (1, 300, 70000), (2, 40, 1 << 30), (1, 300, 1 << 30),
                                               (1, 1, (1 << 31) - 1)])
def test_longest_context(rows, new, window):
    """Rows of 2^30 tokens, all in the pages that their tables name over and over: a
    full page and, behind it, one of each row's own."""
    P, d, slots = 65536, 16, 16384
    if window == 1 << 30:
        slots = 1024  # (several tokens that see all of 2^26)
    rng = np.random.default_rng(rows + new)
    pages = [[page_values(rng, P, d, 40) for _ in range(rows + 1)] for _ in range(2)]
    pool = np.stack([np.stack([c for c, _ in plane]) for plane in pages])
    geo = cache.geometry(P, rows + 1, rows, slots, 1, d)
    length = slots * P - np.arange(rows) * 100
    table = np.zeros((rows, slots), np.int32)
    table[:, -1] = np.arange(rows) + 1
    q = rng.standard_normal((rows * new, 1, d))
    vq, out = Vectors(q, "f32"), Vectors(q, "f32")
    lse = hip.Buffer(rows * new * 4)
    starts = None if new == 1 else hip.Buffer.from_array((np.arange(rows + 1) * new).astype(np.int32))
    d_pool = hip.Buffer.from_array(pool.reshape(-1))
    bufs = [hip.Buffer.from_array(x) for x in (table, length.astype(np.int32))]
    h = cache.KvCache(geo, 1, 1, d, 64, 0)
    h.attend(beam.PageState(*bufs, None), rows, rows * new, native.DTYPE_F32, d_pool, 0, 1, vq.view,
             out.view, 0.25, window, starts, lse)
    hip.synchronize()
    got, got_lse = out.download()[:, 0], lse.download(np.float32)
    x = vq.values()[:, 0]
    for r in range(rows):
        for i in range(0, new, 37):
            at = length[r] - new + i  # its place
            lo = max(0, at - window + 1) if window else 0
            count = np.zeros((2, P))  # how often it sees each token of the two pages
            first, last = lo // P, at // P
            for slot in range(first, last + 1) if last - first < 4 else (first, last):
                c = count[int(slot == slots - 1)]
                a, b = max(lo - slot * P, 0), min(at - slot * P + 1, P)
                c[a:b] += 1
            if last - first >= 4:
                count[0] += last - first - 1
            k, v = (np.concatenate([plane[0][1], plane[r + 1][1]]) for plane in pages)
            s, n = 0.25 * (k @ x[r * new + i]), count.reshape(-1)
            m = s.max()
            w = n * np.exp(s - m)
            want = m + np.log(w.sum())
            # sums of as many terms as a lane adds one by one: 2^30 / (256 x 8 x 64) steps of 16, or
            # 2^26 / (64 x 64) of 16 where a prompt's tokens are split 64 ways
            off = 262144 * 2.0 ** -24
            assert abs(got_lse[r * new + i] - want) <= off + 1e-5 * abs(want), (r, i)
            mass = (w @ np.abs(v)) / w.sum()
            assert (np.abs(got[r * new + i] - (w @ v) / w.sum()) <= 2 * off * mass).all(), (r, i)
    h.close()


@pytest.mark.parametrize("rows", [1, 2048])
def test_most_tokens(rows):
    """A call of 2^20 tokens: appended and attended over with a window, compared at some of them."""
    N, P, B, d, window = cache.MAX_TOKENS, 256, 16, 16, 40
    rng = np.random.default_rng(rows)
    news = np.full(rows, N // rows)
    news[-1] += N - news.sum()
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    used = -(-news // P)
    slots, n_pages = int(used.max()), int(used.sum())
    table = np.full((rows, slots), -1, np.int32)
    order, at = rng.permutation(n_pages), 0
    for r in range(rows):
        table[r, :used[r]] = order[at:at + used[r]]
        at += used[r]
    geo = cache.geometry(P, n_pages, rows, slots, 1, d)
    x = rng.standard_normal((3, N, 1, d)).astype(np.float32)
    q, k, v = (Vectors(a, "bf16") for a in x)
    out = Vectors(x[0], "bf16")
    d_pool = hip.Buffer(2 * geo.plane_stride)
    d_pool.zero()
    bufs = [hip.Buffer.from_array(a) for a in (table, news.astype(np.int32), starts)]
    state = beam.PageState(bufs[0], bufs[1], None)
    h = cache.KvCache(geo, 1, 1, d, B, 0)
    h.append(state, rows, N, native.DTYPE_BF16, d_pool, 0, 1, q=q.view, k=k.view, v=v.view, q_out=q.view,
             d_starts=bufs[2])
    h.attend(state, rows, N, native.DTYPE_BF16, d_pool, 0, 1, q.view, out.view, 0.25, window, bufs[2])
    hip.synchronize()
    got = out.download()[:, 0]
    assert np.array_equal(q.download(), q.values())
    kv = [a.values()[:, 0] for a in (k, v)]
    picks = np.unique(np.concatenate([rng.integers(0, N, 300), starts[:-1], starts[1:] - 1]))
    for i in picks[rng.permutation(len(picks))[:600]]:
        r = int(np.searchsorted(starts, i, side="right")) - 1
        t = i - starts[r]
        lo = max(0, t - window + 1)
        seen = []
        for y in kv:
            vals = []
            for b in range(lo // B, t // B + 1):
                blk = y[starts[r] + b * B:min(starts[r] + b * B + B, starts[r + 1])]
                s = co.scale_of(np.abs(blk).max())
                c = co.encode(blk / s)
                vals.append(np.where(c >= 128, -1.0, 1.0) * co.E4M3[c & 127] * s)
            seen.append(np.concatenate(vals)[lo - lo // B * B:t - lo // B * B + 1])
        s = 0.25 * (seen[0] @ q.values()[i, 0])
        w = np.exp(s - s.max())
        w /= w.sum()
        mass, want = w @ np.abs(seen[1]), w @ seen[1]
        # (2^-16 of the weights; 2 x 24 x 2^-24 of scores' size, some 20; 56 x 2^-23 of sums)
        assert (np.abs(got[i] - want) <= 2.0 ** -8 * np.abs(want) + 1e-4 * mass).all(), i
    h.close()
