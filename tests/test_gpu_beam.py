"""GPU tests of g4s_beam_select and g4s_beam_reorder against the plain forms
of beam_oracle.py.

Tolerances.  The kernel's lse is off by at most 2e-7 absolutely (the header's
bound); a score is rounded once to binary32 (2^-24 of its magnitude).  numpy's
binary64 sums are off by less than 1e-9 here.  Tokens and parents are equal
wherever the oracle's neighbouring scores of different beams lie further apart
than twice the lse bound, which the tests assert of their own inputs."""
import numpy as np
import pytest

import beam_oracle as bo
from gemma4_sampler import beam, hip, native

pytestmark = pytest.mark.gpu
F32, I32 = np.float32, np.int32
LSE = 2e-7
NONE = -np.inf


def run_select(x, scores, beams, n, cap=30.0, stride=None, search=None, stream=None, lse=True,
               inplace=False):
    R, V = x.shape
    batch = R // beams
    esize = x.dtype.itemsize
    per = 16 // esize
    stride = (V + per - 1) // per * per if stride is None else stride
    buf = np.zeros((R, stride), x.dtype)
    buf[:, :V] = x
    buf[:, V:] = 0x7F80 if x.dtype == np.uint16 else np.inf  # never read
    own = search is None
    if own:
        search = beam.BeamSearch(V, batch, max(beams, (n + 1) // 2), cap, stream=stream)
    d_x, d_s = hip.Buffer.from_array(buf), hip.Buffer.from_array(np.asarray(scores, F32))
    d_p, d_t = (hip.Buffer.from_array(np.full(batch * n + 4, 77, np.int32)) for _ in range(2))
    d_o = d_s if inplace else hip.Buffer.from_array(np.full(batch * n + 4, 77, F32))
    d_l = hip.Buffer.from_array(np.full(R + 4, 77, F32)) if lse else None
    search.select(d_x, batch, beams, d_s, n, d_p, d_t, d_o, d_lse=d_l,
                  dtype=native.DTYPE_F32 if esize == 4 else native.DTYPE_BF16, row_stride=stride)
    hip.synchronize()
    p, t, o = d_p.download(np.int32), d_t.download(np.int32), d_o.download(F32)
    assert (p[batch * n:] == 77).all() and (t[batch * n:] == 77).all()
    if lse:
        l = d_l.download(F32)
        assert (l[R:] == 77).all()
    if own:
        search.close()
    return (p[:batch * n].reshape(batch, n), t[:batch * n].reshape(batch, n),
            o[:batch * n].reshape(batch, n), l[:R] if lse else None)


def close(got, want):
    same = got == want  # infinities
    with np.errstate(invalid="ignore"):
        return (same | (np.abs(got - want) <= LSE + np.abs(want) * 2.0 ** -24 * 1.01)).all()


def check(x, scores, beams, n, cap=30.0, **kw):
    p, t, s, lse = bo.select(x, scores, beams, n, cap)
    gap = np.abs(np.diff(s, axis=1)) <= 2 * LSE
    with np.errstate(invalid="ignore"):
        gap &= (p[:, 1:] != p[:, :-1]) & np.isfinite(s[:, 1:]) & (np.diff(s, axis=1) != 0)
    assert not gap.any(), "the input has scores too close to tell apart"
    gp, gt, gs, gl = run_select(x, scores, beams, n, cap, **kw)
    assert np.array_equal(gp, p) and np.array_equal(gt, t)
    assert close(gs.astype(np.float64), s), np.nanmax(np.abs(gs - s))
    if gl is not None:
        assert close(gl.astype(np.float64), lse)


def peaky(rng, R, V, dtype):
    x = (rng.standard_normal((R, V)) * 3).astype(F32)
    at = rng.integers(0, V, (R, min(16, V)))
    np.put_along_axis(x, at, np.take_along_axis(x, at, 1) + rng.uniform(
        6, 12, at.shape).astype(F32), 1)
    return x if dtype == "f32" else bo.bf16(x)


def running(rng, R):
    return -rng.uniform(0, 3, R).cumsum().astype(F32) - F32(4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V, batch, beams, n", [
    (2, 1, 1, 1), (3, 2, 2, 4), (63, 1, 4, 8), (257, 3, 5, 10), (8191, 2, 3, 6),
    (8192, 1, 4, 8), (8193, 2, 4, 4), (16385, 1, 32, 64), (40009, 5, 2, 3),
    (100003, 1, 8, 16), (262144, 1, 4, 8)])
def test_select(dtype, V, batch, beams, n):
    rng = np.random.default_rng(V + beams)
    check(peaky(rng, batch * beams, V, dtype), running(rng, batch * beams), beams, n)


@pytest.mark.parametrize("cap", [0.0, -1.0, 5.0, 50.0, 1000.0])
def test_softcaps(cap):
    rng = np.random.default_rng(5)
    x = peaky(rng, 8, 20011, "f32") * F32(4)
    check(x, running(rng, 8), 4, 8, cap=cap)
    check(bo.bf16(x), running(rng, 8), 4, 8, cap=cap)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e9, 1e15, 1e30])
def test_softcaps_far_above_the_logits(cap, dtype):
    """A cap that is practically none leaves the logits as they are: the error of
    the softcap is relative to its value, not to the cap."""
    rng = np.random.default_rng(50)
    x = peaky(rng, 8, 20011, "f32") * F32(2)
    x[:, 100] = 1e-3
    check(x if dtype == "f32" else bo.bf16(x), running(rng, 8), 4, 8, cap=cap)


def test_most_beams():
    rng = np.random.default_rng(6)
    check(peaky(rng, 128, 3001, "f32"), running(rng, 128), 64, 128)
    check(peaky(rng, 64, 70001, "bf16"), running(rng, 64), 64, 128)


@pytest.mark.parametrize("batch, beams, n", [(65535, 1, 2), (1023, 64, 128), (21845, 3, 3)])
def test_most_rows(batch, beams, n):
    """As many rows as a call takes, of a handful of logits."""
    rng = np.random.default_rng(51)
    x = rng.permuted(np.tile(np.arange(5, dtype=F32) * F32(1.25), (batch * beams, 1)), axis=1)
    x += rng.integers(-2, 3, (batch * beams, 1)).astype(F32)
    x[7], x[8, 1:] = NONE, np.nan
    # scores a third apart, logits multiples of a quarter: no two candidates are near
    s = np.tile(-np.arange(beams) * F32(0.3125) - F32(1), batch).astype(F32)
    x += (np.arange(batch * beams) % beams % 7)[:, None].astype(F32) * F32(0.03)
    check(x, s, beams, n)


@pytest.mark.parametrize("dtype, batch, beams, n", [("f32", 1, 1, 128), ("f32", 1, 3, 6),
                                                    ("bf16", 1, 1, 2), ("bf16", 2, 4, 8)])
def test_longest_rows(dtype, batch, beams, n):
    rng = np.random.default_rng(52)
    V = 1 << 22
    x = peaky(rng, batch * beams, V, dtype)
    x[0, V - 1] = 25 if dtype == "f32" else bo.bf16(np.array([25], F32))[0]
    check(x, running(rng, batch * beams), beams, n)


def test_flat_rows_and_offsets():
    """Rows whose mass lies in many tokens, far from 0 and from the cap."""
    rng = np.random.default_rng(7)
    for mid in (-25.0, 0.0, 18.0, 45.0):
        x = (rng.standard_normal((4, 50021)) * 0.5 + mid).astype(F32)
        check(x, running(rng, 4), 2, 4)
        check(bo.bf16(x), running(rng, 4), 2, 4)


def test_dead_beams_and_first_step():
    rng = np.random.default_rng(8)
    x = peaky(rng, 12, 9001, "f32")
    s = np.full(12, NONE, F32)
    s[[0, 4]] = 0  # the third sequence has no live beam
    check(x, s, 4, 8)
    s[5], s[6], s[7], s[8] = np.nan, -1e30, np.finfo(F32).min, -7.5
    check(x, s, 4, 8)
    x[s != s] = np.nan  # a dead row is not read
    check(x, s, 4, 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fill", [NONE, "lowest", np.nan, -1e30])
def test_masked_logits(dtype, fill):
    rng = np.random.default_rng(9)
    x = peaky(rng, 6, 12289, "f32")
    if fill == "lowest":
        fill = np.finfo(F32).min if dtype == "f32" else -3.38953139e38
    x[0, rng.random(12289) < 0.7] = fill
    x[1] = fill                    # nothing left
    x[2] = fill
    x[2, [5, 9000, 12288]] = [1, 2, 2]  # fewer than n, in two chunks
    x[3, :8192] = fill             # a chunk without candidates
    if dtype == "bf16":
        finite = np.isfinite(x)
        b = bo.bf16(np.where(finite, x, 0))
        b[x == NONE], b[np.isnan(x)] = 0xFF80, 0x7FC1
        if fill == -1e30:
            assert bo.widen(b[1])[0] <= F32(-1e30)
        x = b
    check(x, running(rng, 6), 3, 6)
    check(x, running(rng, 6), 1, 2)


def test_fewer_candidates_than_asked():
    rng = np.random.default_rng(10)
    x = rng.standard_normal((4, 3)).astype(F32)
    check(x, running(rng, 4), 2, 8)
    x[:] = NONE
    check(x, running(rng, 4), 2, 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ties(dtype):
    """Equal logits: the lowest tokens of the lowest beams, in masses too."""
    rng = np.random.default_rng(11)
    x = np.zeros((8, 30011), F32)       # everything equal
    x[4:] = rng.integers(0, 3, (4, 30011))
    x[7, 20000:20040] = 5
    s = np.array([-1, -1, -1, -2, -3, -3.5, -4, -9], F32)
    s[4:] += rng.uniform(0, .1, 4).astype(F32)
    x[2, ::2] = -0.0                    # equal to +0
    check(x if dtype == "f32" else bo.bf16(x), s, 4, 16)


def test_equal_beams():
    """Two beams with the same logits and score tie exactly: the lower first."""
    rng = np.random.default_rng(12)
    x = peaky(rng, 3, 50001, "f32")
    x[2] = x[0]
    check(x, np.array([-1.5, -1.75, -1.5], F32), 3, 12)


def test_saturated_softcap():
    """Distinct logits beyond the cap round to one score: the larger first."""
    x = np.full((2, 5000), -1, F32)
    x[0, 100:140] = 2000 + np.arange(40)[::-1] * F32(0.25)
    x[0, 4000:4040] = 540 + np.arange(40) * F32(0.001)
    x[1, 7] = 33
    check(x, np.array([-2, -1], F32), 2, 100, cap=30.0)


def test_infinite_logits():
    rng = np.random.default_rng(13)
    x = peaky(rng, 4, 20001, "f32")
    x[0, [3, 15000]] = np.inf
    x[2, 9000] = np.inf
    x[3, :700] = np.inf  # more than a workgroup's list holds
    for cap in (0.0, 30.0):
        check(x, running(rng, 4), 4, 8, cap=cap)
        check(x, running(rng, 4), 2, 8, cap=cap)


def test_infinite_score():
    rng = np.random.default_rng(14)
    x = peaky(rng, 2, 5001, "f32")
    check(x, np.array([-1, np.inf], F32), 2, 4)


def special_rows(rng, V):
    """Rows that the common way does not suit, 24 of them: (name, logits)."""
    n = rng.standard_normal
    wave = (np.arange(V) % 8192 < 64)
    rows = [("ascending", np.linspace(-20, 20, V)), ("descending", np.linspace(20, -20, V)),
            ("low start", np.where(np.arange(V) < 17000, -28 + n(V) * .01, n(V) * 3)),
            ("low tiles", np.where(np.arange(V) % 16384 < 8000, -30, n(V))),
            ("zero", np.zeros(V)), ("equal", np.full(V, -7.25)),
            ("two values", rng.integers(0, 2, V) * 3.0), ("negative", -np.abs(n(V)) - 5),
            ("tiny", n(V) * 1e-6), ("tinier", n(V) * 1e-9), ("both signs tiny", n(V) * 3e-8),
            ("masked half", np.where(rng.random(V) < .5, NONE, n(V) * 3)),
            ("masked lowest", np.where(rng.random(V) < .9, -3.38e38, n(V) * 3)),
            ("masked tiles", np.where(np.arange(V) < 20000, NONE, n(V) * 3)),
            ("all but one", np.where(np.arange(V) == V - 3, -12.0, NONE)),
            ("nothing", np.full(V, NONE)), ("nan", np.where(wave, np.nan, n(V) * 3)),
            ("mostly nan", np.where(rng.random(V) < .999, np.nan, n(V))),
            ("negative nan", np.where(rng.random(V) < .1, -np.nan, -np.abs(n(V)))),
            ("large", n(V) * 40), ("few large", np.where(wave, n(V) * 60, n(V) * 2)),
            ("very negative", n(V) - 70), ("infinite", np.where(rng.random(V) < 1e-3, np.inf,
                                                                 n(V))),
            ("large and masked", np.where(rng.random(V) < .3, NONE, n(V) * 35))]
    return rows


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap, V, batch, beams, n", [
    (30.0, 40009, 57, 6, 12), (0.0, 40009, 57, 6, 6), (50.0, 33000, 6, 64, 128),
    (100.0, 20000, 50, 6, 12), (30.0, 262144, 8, 12, 24)])
def test_many_rows(dtype, cap, V, batch, beams, n):
    """Batches whose workgroups take several tiles each (and bf16 looks its
    terms up), with rows of every other kind among them."""
    rng = np.random.default_rng(20 + batch)
    x = (rng.standard_normal((batch * beams, V), dtype=F32) * F32(3))
    at = rng.integers(0, V, (batch * beams, 8))
    np.put_along_axis(x, at, rng.uniform(10, 18, at.shape).astype(F32), 1)
    special = special_rows(rng, V)
    for i, (_, row) in enumerate(special):
        with np.errstate(over="ignore"):
            x[1 + i * 3 % (batch * beams - 1)] = row.astype(F32)
    if dtype == "bf16":
        odd = ~np.isfinite(x)
        b = bo.bf16(np.where(odd, 0, x))
        b[odd] = (x[odd].view(np.uint32) >> 16) | (np.isnan(x[odd]) * 0x40).astype(np.uint32)
        x = b
    # one beam a sequence is far ahead, and scores of neighbours never near
    s = (-np.arange(batch * beams) % beams * 40).astype(F32) + \
        rng.uniform(-3, 0, batch * beams).astype(F32)
    check(x, s, beams, n, cap=cap)
    check(x, running(rng, batch * beams), beams, n, cap=cap)


@pytest.mark.parametrize("V, batch, beams, n", [
    (32767, 8, 9, 18), (32768, 8, 8, 16), (32769, 13, 5, 10), (65536, 4, 8, 9), (65537, 3, 11, 22),
    (262143, 2, 4, 8), (262144, 1, 8, 16), (100003, 7, 3, 6)])
def test_bf16_rows_of_few_tiles(V, batch, beams, n):
    """About the fewest rows, and the shortest, whose terms are looked up: a
    workgroup has one tile or two, the last of them with a few tokens."""
    rng = np.random.default_rng(V + batch)
    x = peaky(rng, batch * beams, V, "bf16")
    x[1, :16384] = 0xFF80               # a tile without candidates
    x[2, -5:] = bo.bf16(np.array([21, 22, 23, 24, 25], F32))
    x[3] = 0xFF80
    x[4, V - 1], x[5, 7] = 0x7FC1, 0x7F80
    check(x, running(rng, batch * beams), beams, n)
    s = running(rng, batch * beams)
    s[::3] = NONE
    check(x, s, beams, beams, inplace=True)


@pytest.mark.parametrize("V, batch, beams, n", [
    (32768, 24, 8, 16), (32769, 48, 4, 8), (40000, 20, 8, 16), (49151, 33, 4, 4),
    (49152, 11, 4, 8), (49153, 6, 7, 14)])
def test_bf16_rows_of_two_and_three_tiles(V, batch, beams, n):
    """Batches about the fewest whose terms are looked up, in rows of two tiles
    and of a few logits more than two and three."""
    rng = np.random.default_rng(V)
    x = peaky(rng, batch * beams, V, "bf16")
    x[1, :16384] = 0xFF80
    x[2, -1:] = bo.bf16(np.array([25], F32))
    x[3] = 0xFF80
    x[4, V - 1], x[5, 7] = 0x7FC1, 0x7F80
    s = running(rng, beams)
    check(x, np.concatenate([s + F32(b * 2.0 ** -6) for b in range(batch)]), beams, n)


def test_stride_no_lse_and_scores_in_place():
    rng = np.random.default_rng(15)
    x = peaky(rng, 6, 10007, "bf16")
    check(x, running(rng, 6), 3, 3, stride=16384, lse=False)
    check(x, running(rng, 6), 3, 3, inplace=True)


@pytest.mark.parametrize("batch", [1, 40])
def test_scores_in_place_with_dead_beams(batch):
    """The scores of dead rows are overwritten by live ones while other
    workgroups of those rows may not have started; three calls in a row."""
    rng = np.random.default_rng(30 + batch)
    V, W = 100003, 4
    search = beam.BeamSearch(V, batch, W, 30.0)
    for _ in range(3):
        x = peaky(rng, batch * W, V, "f32")
        s = np.full(batch * W, NONE, F32)
        s[::W] = rng.uniform(-3, 0, batch).astype(F32)
        check(x, s, W, W, inplace=True, search=search)
    search.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_top_logits_beyond_the_cap(dtype):
    """Raw logits of 40 to 90 before the softcap, a few in each row."""
    rng = np.random.default_rng(33)
    x = (rng.standard_normal((12, 50021)) * 4).astype(F32)
    at = rng.integers(0, 50021, (12, 40))
    np.put_along_axis(x, at, rng.uniform(36, 90, at.shape).astype(F32), 1)
    np.put_along_axis(x, at[:, ::2] // 2, rng.uniform(-90, -36, (12, 20)).astype(F32), 1)
    check(x if dtype == "f32" else bo.bf16(x), running(rng, 12), 4, 8)


def test_calls_in_a_row_and_smaller_shapes():
    """One handle, shapes that grow and shrink: nothing of a call is left over."""
    rng = np.random.default_rng(16)
    search = beam.BeamSearch(30001, 6, 8, 30.0)
    for batch, beams, n, dtype in [(6, 8, 16, "f32"), (1, 1, 1, "bf16"), (2, 8, 16, "f32"),
                                   (3, 5, 7, "bf16"), (6, 8, 8, "f32")]:
        check(peaky(rng, batch * beams, 30001, dtype), running(rng, batch * beams), beams, n,
              search=search)
    search.close()


def test_other_stream_and_another_handle():
    rng = np.random.default_rng(17)
    streams = [hip.Stream(nonblocking=True) for _ in range(2)]
    for st in streams:
        check(peaky(rng, 4, 9999, "f32"), running(rng, 4), 4, 8, stream=st)
    for st in streams:
        st.destroy()


def test_two_handles_side_by_side():
    """Calls of two handles on two streams, none waited for before the last."""
    rng = np.random.default_rng(40)
    V, W, n = 60013, 4, 8
    jobs = []
    for k in range(2):
        st = hip.Stream(nonblocking=True)
        jobs.append((st, beam.BeamSearch(V, 6, W, 30.0, stream=st)))
    calls = []
    for k in range(6):
        st, search = jobs[k % 2]
        batch = 1 + k
        x, s = peaky(rng, batch * W, V, "f32"), running(rng, batch * W)
        stride = (V + 3) // 4 * 4
        buf = np.zeros((batch * W, stride), F32)
        buf[:, :V] = x
        d = [hip.Buffer.from_array(a) for a in (buf, s)] + [hip.Buffer(4 * batch * n)
                                                            for _ in range(3)]
        calls.append((search, batch, stride, x, s, d))
    hip.synchronize()
    for search, batch, stride, _, _, d in calls:
        search.select(d[0], batch, W, d[1], n, d[2], d[3], d[4], row_stride=stride)
    hip.synchronize()
    for _, batch, _, x, s, d in calls:
        p, t, o, _ = bo.select(x, s, W, n, 30.0)
        assert np.array_equal(d[2].download(I32).reshape(p.shape), p)
        assert np.array_equal(d[3].download(I32).reshape(t.shape), t)
        assert close(d[4].download(F32).reshape(o.shape).astype(np.float64), o)
    for st, search in jobs:
        search.close()
        st.destroy()


def test_select_refusals():
    s = beam.BeamSearch(1000, 2, 4, 30.0)
    d = hip.Buffer(8 * 1000 * 4)
    o = hip.Buffer(4096)
    good = dict(d_logits=d, batch=2, beams=4, d_scores=o, n_select=8, d_parents=o.offset(512),
                d_tokens=o.offset(1024), d_out=o.offset(1536))
    for change in [dict(batch=0), dict(batch=3), dict(beams=0), dict(beams=5), dict(n_select=0),
                   dict(n_select=9), dict(dtype=2), dict(row_stride=999), dict(row_stride=1002),
                   dict(row_stride=1 << 60), dict(d_logits=d.offset(4)), dict(d_logits=None),
                   dict(d_scores=None), dict(d_parents=None), dict(d_tokens=None),
                   dict(d_out=None), dict(d_out=o), dict(d_out=o.offset(28))]:
        with pytest.raises(native.SamplerError) as e:
            s.select(**dict(good, **change))
        assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT, change
    s.close()


def test_select_refuses_overlapping_arrays():
    """Results of one sequence are written while scores and logits of others,
    or its own, are still read."""
    s = beam.BeamSearch(1000, 2, 4, 30.0)
    d = hip.Buffer(8 * 1000 * 4)
    o = hip.Buffer(8192).zero()
    good = dict(d_logits=d.zero(), batch=2, beams=4, d_scores=o, n_select=4,
                d_parents=o.offset(512), d_tokens=o.offset(1024), d_out=o.offset(1536),
                d_lse=o.offset(2048))
    out = ["d_parents", "d_tokens", "d_out", "d_lse"]
    clashes = [{k: o.offset(28)} for k in out] + [{k: o} for k in out if k != "d_out"] + \
        [{k: d.offset(8 * 4000 - 4)} for k in out] + [{k: d.offset(2000)} for k in out] + \
        [{a: good[b]} for a in out for b in out if a != b] + \
        [{"d_tokens": o.offset(512 + 28)}, {"d_out": o, "d_lse": o.offset(4)},
         {"d_out": o, "d_parents": o}, {"d_out": o, "n_select": 3}, {"d_out": o, "n_select": 8}]
    for change in clashes:
        with pytest.raises(native.SamplerError) as e:
            s.select(**dict(good, **change))
        assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT and "overlaps" in str(e.value)
    for change in [{}, {"d_out": o}, {"d_lse": None}, {"d_lse": o.offset(32)},
                   {"d_parents": o.offset(1536 + 32)}]:
        s.select(**dict(good, **change))
    hip.synchronize()
    s.close()


# ----------------------------------------------------------------- reorder


def reordered(data, parents, beams, inplace):
    out = data.copy()
    for r, p in enumerate(parents):
        b = r // beams
        if p // beams == b and p >= 0:
            out[:, r] = data[:, p]
    return out


@pytest.mark.parametrize("inplace", [True, False])
@pytest.mark.parametrize("batch, beams, planes, row, stride, shift", [
    (1, 1, 1, 16, 16, 0), (1, 4, 3, 4096, 4096, 0), (2, 3, 2, 5008, 5024, 0),
    (1, 5, 2, 1000, 1004, 4), (3, 8, 1, 333, 350, 1), (1, 16, 2, 20000, 20000, 0),
    (2, 17, 1, 4112, 4112, 0), (1, 32, 2, 1028, 1040, 0), (1, 64, 1, 7777, 7777, 3),
    (5, 64, 2, 64, 80, 0)])
def test_reorder(inplace, batch, beams, planes, row, stride, shift):
    rng = np.random.default_rng(row + beams)
    R = batch * beams
    s = beam.BeamSearch(100, batch, beams, 30.0)
    for kind in range(3):
        if kind == 0:    # any parents, most of them more than once
            par = np.repeat(np.arange(batch), beams) * beams + rng.integers(0, beams, R)
        elif kind == 1:  # a permutation: every row is overwritten while another needs it
            par = np.concatenate([b * beams + rng.permutation(beams) for b in range(batch)])
        else:            # rows that stay: none, another sequence's, out of range
            par = np.repeat(np.arange(batch), beams) * beams + rng.integers(0, beams, R)
            par[::3] = rng.choice([-1, -5, R, R + 7, (1 << 31) - 1, -(1 << 31)], len(par[::3]))
            if batch > 1:
                par[1] = R - 1
        data = rng.integers(0, 256, (planes, R, stride), dtype=np.uint8)
        raw = np.zeros(shift + data.size + 64, np.uint8)
        raw[shift:shift + data.size] = data.reshape(-1)
        d = hip.Buffer.from_array(raw)
        other = rng.integers(0, 256, raw.size, dtype=np.uint8)
        e = d if inplace else hip.Buffer.from_array(other)
        s.reorder(d.offset(shift), e.offset(shift), planes, R * stride, batch, beams, stride, row,
                  hip.Buffer.from_array(par.astype(np.int32)))
        hip.synchronize()
        want = (raw if inplace else other).copy()
        w = want[shift:shift + data.size].reshape(data.shape)
        w[:, :, :row] = reordered(data, par, beams, inplace)[:, :, :row]
        assert np.array_equal(e.download(np.uint8), want), kind
        if not inplace:
            assert np.array_equal(d.download(np.uint8), raw)
    s.close()


def test_reorder_planes_inside_rows():
    """[row][plane][bytes]: the planes' stride is below the rows'."""
    rng = np.random.default_rng(3)
    data = rng.integers(0, 256, (8, 3, 48), dtype=np.uint8)
    par = np.array([1, 0, 3, 3, 7, 6, 5, 4], np.int32)
    s = beam.BeamSearch(100, 2, 4, 30.0)
    d = hip.Buffer.from_array(data)
    s.reorder(d, d, 3, 48, 2, 4, 144, 48, hip.Buffer.from_array(par))
    hip.synchronize()
    assert np.array_equal(d.download(np.uint8).reshape(data.shape), data[par])
    s.close()


def test_reorder_refusals():
    s = beam.BeamSearch(100, 2, 4, 30.0)
    d, e = hip.Buffer(1 << 16), hip.Buffer(4096)
    good = dict(d_src=d, d_dst=d, planes=2, plane_stride=8192, batch=2, beams=4, row_stride=1024,
                row_bytes=1024, d_parents=e)
    s.reorder(**dict(good, row_bytes=0))
    for change in [dict(batch=3), dict(beams=5), dict(planes=0), dict(planes=-1),
                   dict(row_bytes=-1), dict(row_bytes=1025), dict(row_stride=-1024),
                   dict(plane_stride=8191), dict(plane_stride=512), dict(planes=1 << 40),
                   dict(d_src=None), dict(d_dst=None), dict(d_parents=None),
                   dict(d_dst=d.offset(16384 - 16)), dict(d_dst=d.offset(16))]:
        with pytest.raises(native.SamplerError) as err:
            s.reorder(**dict(good, **change))
        assert err.value.code == native.G4S_ERR_INVALID_ARGUMENT, change
    s.close()


def test_reorder_refuses_parents_in_the_destination():
    s = beam.BeamSearch(100, 2, 4, 30.0)
    d, e = hip.Buffer(1 << 16).zero(), hip.Buffer(1 << 16).zero()
    size = 8192 + 7 * 1000 + 900
    for src, par in [(d, d), (d, d.offset(size - 4)), (d, d.offset(7992)), (e, d.offset(996))]:
        with pytest.raises(native.SamplerError) as err:
            s.reorder(src, d, 2, 8192, 2, 4, 1000, 900, par)
        assert err.value.code == native.G4S_ERR_INVALID_ARGUMENT
    s.reorder(d, d, 2, 8192, 2, 4, 1000, 900, d.offset(size))
    s.reorder(e, d, 2, 8192, 2, 4, 1000, 900, e)
    hip.synchronize()
    s.close()


def test_reorder_rows_past_32_bits():
    """Rows of more than 2^32 bytes at an odd address, a thread a byte."""
    row = (1 << 32) + 1027
    rng = np.random.default_rng(19)
    s = beam.BeamSearch(100, 1, 2, 30.0)
    d = hip.Buffer(1 + 2 * row).zero()
    at = [0, 1 << 31, (1 << 32) - 300, row - 600]
    data = {(r, a): rng.integers(1, 256, 600, dtype=np.uint8) for r in range(2) for a in at}
    for (r, a), piece in data.items():
        d.upload(piece, 1 + r * row + a)
    s.reorder(d.offset(1), d.offset(1), 1, 0, 1, 2, row, row,
              hip.Buffer.from_array(np.array([1, 0], I32)))
    hip.synchronize()
    for (r, a), piece in data.items():
        assert np.array_equal(d.download(np.uint8, 600, 1 + (1 - r) * row + a), piece), (r, a)
    s.close()


@pytest.fixture
def earlier():
    """A failing HIP call of the caller's own, whose error stays with the thread
    until it is asked for."""
    import ctypes

    def fail():
        assert hip.lib().hipSetDevice(ctypes.c_int(1 << 20)) != 0
    yield fail
    hip.lib().hipGetLastError()


def test_an_earlier_failure_is_not_the_calls(earlier):
    """The calls report their own launches."""
    rng = np.random.default_rng(21)
    earlier()
    s = beam.BeamSearch(1001, 1, 3, 30.0)
    x = peaky(rng, 3, 1001, "f32")
    orig = s.select
    s.select = lambda *a, **k: (earlier(), orig(*a, **k))
    check(x, running(rng, 3), 3, 6, search=s)
    d, par = hip.Buffer(3 * 64).zero(), hip.Buffer.from_array(np.array([1, 0, 2], I32))
    data = rng.integers(0, 256, (3, 64), dtype=np.uint8)
    d.upload(data)
    earlier()
    s.reorder(d, d, 1, 0, 1, 3, 64, 64, par)
    hip.synchronize()
    assert np.array_equal(d.download(np.uint8).reshape(3, 64), data[[1, 0, 2]])
    earlier()
    c = beam.PageCache(4, 8, 2, 4, planes=1, parts=1, token_bytes=16)
    states = []
    for _ in range(2):
        bufs = [hip.Buffer(4 * n).zero() for n in (8, 2, 8)]
        states.append((bufs, beam.PageState(*bufs)))
    (_, a), (_, b) = states
    pool, status, one = hip.Buffer(8 * 64).zero(), hip.Buffer(16), hip.Buffer(64).zero()
    for call in (lambda: c.advance(a, 2, b, 2, one, None, pool, status),
                 lambda: c.compact(a, b, 2, pool, status),
                 lambda: c.copy(pool, pool, 1, one,
                                hip.Buffer.from_array(np.array([1], I32)))):
        earlier()
        call()
        hip.synchronize()
    s.close()
    c.close()


def test_captured_step():
    """Selection and reordering in one captured graph, replayed on new logits
    with eager calls between."""
    rng = np.random.default_rng(18)
    st = hip.Stream(nonblocking=True)
    V, W = 20000, 4
    s = beam.BeamSearch(V, 2, W, 30.0, stream=st)
    R = 2 * W
    d_x = hip.Buffer(R * V * 4)
    d_s, d_p, d_t = hip.Buffer(4 * R), hip.Buffer(4 * R), hip.Buffer(4 * R)
    d_state, d_l = hip.Buffer(R * 4096), hip.Buffer(4 * R)
    d_first = hip.Buffer(4 * R)
    graph, run = _capture(st, lambda: (
        s.select(d_x, 2, W, d_first, W, d_p, d_t, d_s, d_lse=d_l),
        s.reorder(d_state, d_state, 1, 0, 2, W, 4096, 4096, d_p)))
    for _ in range(4):
        x, sc = peaky(rng, R, V, "f32"), running(rng, R)
        data = rng.integers(0, 256, (R, 4096), dtype=np.uint8)
        st.synchronize()
        d_x.upload(x)
        d_first.upload(sc)
        d_state.upload(data)
        run()
        st.synchronize()
        p, t, o, _ = bo.select(x, sc, W, W, 30.0)
        assert np.array_equal(d_p.download(np.int32).reshape(2, W), p)
        assert np.array_equal(d_t.download(np.int32).reshape(2, W), t)
        assert close(d_s.download(F32).reshape(2, W).astype(np.float64), o)
        assert np.array_equal(d_state.download(np.uint8).reshape(data.shape),
                              data[p.reshape(-1)])
        check(peaky(rng, 3, V, "f32"), running(rng, 3), 3, 3, search=s)
    graph()
    s.close()
    st.destroy()


def _capture(st, record):
    """(destroy, launch) of a graph of the launches that record() makes on st."""
    import ctypes
    L = hip.lib()
    g, x = ctypes.c_void_p(), ctypes.c_void_p()
    hip.check(L.hipStreamBeginCapture(st.handle, ctypes.c_int(1)), "hipStreamBeginCapture")
    try:
        record()
    finally:
        rc = L.hipStreamEndCapture(st.handle, ctypes.byref(g))
    hip.check(rc, "hipStreamEndCapture")
    hip.check(L.hipGraphInstantiate(ctypes.byref(x), g, None, None, ctypes.c_size_t(0)),
              "hipGraphInstantiate")

    def destroy():
        L.hipGraphExecDestroy(x)
        L.hipGraphDestroy(g)
    return destroy, lambda: hip.check(L.hipGraphLaunch(x, st.handle), "hipGraphLaunch")
