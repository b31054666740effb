"""g4s_beam_generate against a plain search on the host, with a model whose
logits depend on the whole history.  The history that the model sees is read
back from the beams' states: a contiguous one that the loop reorders in place,
and a paged cache that it forks, both holding one token per position.  So a
state that did not follow its beam gives other logits, and other results."""
import ctypes

import numpy as np
import pytest

import beam_oracle as bo
from gemma4_sampler import beam, hip, native

pytestmark = pytest.mark.gpu
F32, I32 = np.float32, np.int32
V, P, ROOM = 400, 4, 40
ENDS = (1, 106, 50)


def model(history, ends=2.0):
    rng = np.random.default_rng([7, *history])
    x = (rng.standard_normal(V) * 2).astype(F32)
    x[list(ENDS)] += F32(ends)
    return x


def plain_search(prompt, W, max_tokens, n_best, early, penalty, ends, gaps):
    """(tokens, score) of the n best, by the definition in the header."""
    beams, done = [((), F32(0))], []

    def worth(score, length):
        return F32(np.float64(score) / np.float64(length) ** np.float64(F32(penalty)))

    def add(tokens, score):
        s = worth(score, len(tokens))
        at = next((i for i, d in enumerate(done) if s > d[1]), len(done))
        done.insert(at, (tokens, s))
        del done[W:]

    for length in range(1, max_tokens + 1):
        rows = np.stack([model(prompt + h, ends) for h, _ in beams])
        p, t, s, _ = bo.select(rows, [x for _, x in beams], len(beams), 2 * W, 30.0)
        d = np.diff(s[0])
        gaps.append(np.abs(d[np.isfinite(d)]).min())
        following = []
        for i in range(2 * W):
            if p[0, i] < 0 or len(following) == W:
                break
            h = beams[p[0, i]][0] + (int(t[0, i]),)
            if t[0, i] in ENDS:
                if i < W:
                    add(h, F32(s[0, i]))
            else:
                following.append((h, F32(s[0, i])))
        beams = following
        if not beams:
            break
        if length == max_tokens:
            for h, x in beams:
                add(h, x)
            break
        if len(done) >= W and (early or done[-1][1] >= worth(beams[0][1], length)):
            break
    return done[:n_best]


class Engine:
    """The caller's side: states, cache, and the model step."""

    def __init__(self, prompts, W, ends, stream=None, pages=200):
        self.B, self.W, self.prompts, self.ends = len(prompts), W, prompts, ends
        self.R = R = self.B * W
        self.slots = ROOM // P
        self.stream = stream
        self.cache = beam.PageCache(P, pages, R, self.slots, planes=1, parts=1, token_bytes=4,
                                    stream=stream)
        self.pool = hip.Buffer.from_array(np.full(pages * P, -9, I32))
        first = bo.State(R, self.slots, pages)
        spare = bo.State(R, self.slots, pages)
        pool = np.full(pages * P, -9, I32)
        state = np.full((R, ROOM), -7, I32)
        at = 0
        for b, prompt in enumerate(prompts):
            n = -(-len(prompt) // P)
            first.table[b * W, :n] = range(at, at + n)
            first.refs[at:at + n] = 1
            first.lengths[b * W] = len(prompt)
            pool[at * P:at * P + len(prompt)] = prompt
            state[b * W, :len(prompt)] = prompt
            at += n
        self.pool.upload(pool)
        self.state = hip.Buffer.from_array(state)
        self.bufs = [[hip.Buffer.from_array(a) for a in (s.table, s.lengths, s.refs)]
                     for s in (first, spare)]
        self.beam_cache = beam.BeamCache(self.cache, [beam.PageState(*b) for b in self.bufs],
                                         self.pool)
        self.beam_states = beam.BeamStates(self.state, 1, 0, ROOM * 4, ROOM * 4)
        rows = np.zeros((R, V), F32)
        for b, prompt in enumerate(prompts):
            rows[b * W] = model(prompt, ends)
        rows[np.arange(R) % W != 0] = np.nan  # rows without a beam yet
        self.logits = hip.Buffer.from_array(rows)
        self.length = len(prompts[0])
        self.calls = 0

    def forward(self, step):
        hip.synchronize()
        self.calls += 1
        tokens, parents = step.Tokens(), step.Parents()
        table = self.bufs[step.state][0].download(I32).reshape(self.R, self.slots)
        lengths = self.bufs[step.state][1].download(I32)
        pool = self.pool.download(I32)
        state = self.state.download(I32).reshape(self.R, ROOM)
        rows = self.logits.download(F32).reshape(self.R, V)
        assert np.array_equal(hip.Buffer.download(_at(step.d_tokens, self.R), I32), tokens)
        assert np.array_equal(hip.Buffer.download(_at(step.d_parents, self.R), I32), parents)
        for r in range(self.R):
            if tokens[r] < 0:
                assert parents[r] == -1 and lengths[r] == 0
                rows[r] = np.nan
                continue
            n = int(lengths[r])
            pool[table[r, (n - 1) // P] * P + (n - 1) % P] = tokens[r]
            state[r, n - 1] = tokens[r]
        for r in np.flatnonzero(tokens >= 0):
            n = int(lengths[r])
            seen = tuple(int(pool[table[r, i // P] * P + i % P]) for i in range(n))
            assert seen == tuple(int(x) for x in state[r, :n])
            rows[r] = model(seen, self.ends)
        self.pool.upload(pool)
        self.state.upload(state)
        self.logits.upload(rows)
        return True


class _At(hip.Buffer):
    def __init__(self, addr, nbytes):
        self.nbytes, self.ptr = nbytes, ctypes.c_void_p(addr)

    def free(self):
        pass


def _at(addr, count):
    return _At(addr, 4 * count)


PROMPTS = [(5, 9, 200, 3, 7), (11, 300), (42,), (8, 8, 8, 8)]


@pytest.mark.parametrize("B, W, n_best, max_tokens, early, penalty, ends", [
    (1, 4, 4, 12, False, 1.0, 2.0), (4, 3, 2, 9, True, 0.0, 3.0), (2, 1, 1, 6, False, 1.0, 1.0),
    (3, 5, 5, 10, False, 2.0, 6.0), (2, 4, 1, 1, False, 1.0, 0.0), (2, 8, 3, 7, True, -0.5, 4.0)])
def test_generate(B, W, n_best, max_tokens, early, penalty, ends):
    gaps, want = [], []
    for prompt in PROMPTS[:B]:
        want.append(plain_search(prompt, W, max_tokens, n_best, early, penalty, ends, gaps))
    # neighbouring candidates are further apart than lse's bound and the
    # rounding of the scores they came from
    assert min(gaps) > 4e-7 + max(abs(float(d[1])) for w in want for d in w) * 2.0 ** -23
    st = hip.Stream(nonblocking=True)
    eng = Engine(PROMPTS[:B], W, ends, st)
    s = beam.BeamSearch(V, B, W, 30.0, stream=st)
    got = s.Generate(eng.logits, B, W, max_tokens, eng.forward, n_best=n_best, early_stop=early,
                     length_penalty=penalty, states=eng.beam_states, cache=eng.beam_cache)
    assert eng.calls < max_tokens
    for g, w in zip(got, want):
        assert [tuple(int(x) for x in t) for t, _ in g] == [t for t, _ in w]
        # one rounding of the sum per token, and lse's bound
        for (t, a), (_, b) in zip(g, w):
            raw = abs(b) * len(t) ** penalty
            tol = len(t) * (2e-7 + raw * 2.0 ** -24) / len(t) ** penalty + abs(b) * 2.0 ** -23
            assert abs(a - b) <= tol
    s.close()
    st.destroy()


def test_generate_without_states():
    """A model of the last token alone needs neither states nor pages."""
    eng = Engine(PROMPTS[:2], 3, 2.0)
    s = beam.BeamSearch(V, 2, 3, 30.0)
    steps = []

    def forward(step):
        steps.append((step.Tokens(), step.Parents()))
        rows = np.stack([model((int(max(t, 0)),)) for t in step.Tokens()])
        eng.logits.upload(rows)
        return True
    got = s.Generate(eng.logits, 2, 3, 5, forward)
    assert all(len(g) == 1 for g in got)
    assert (steps[0][1] == [0, 0, 0, 3, 3, 3]).all()
    s.close()


def test_generate_without_candidates():
    """A sequence whose prompt leaves no token, one whose second step leaves none, and
    one that goes on beside them."""
    W, prompts = 3, PROMPTS[:3]
    eng = Engine(prompts, W, 2.0)
    s = beam.BeamSearch(V, 3, W, 30.0)
    rows = eng.logits.download(F32).reshape(9, V)
    rows[0] = -np.inf
    eng.logits.upload(rows)

    def forward(step):
        assert (step.Tokens()[:W] == -1).all()
        ok = eng.forward(step)
        rows = eng.logits.download(F32).reshape(9, V)
        rows[W:2 * W] = np.nan
        eng.logits.upload(rows)
        return ok
    got = s.Generate(eng.logits, 3, W, 6, forward, n_best=W, states=eng.beam_states,
                     cache=eng.beam_cache)
    first = bo.select(model(prompts[1], 2.0)[None], [0.0], 1, 2 * W, 30.0)[1][0]
    ends = [int(t) for t in first[:W] if t in ENDS]
    assert got[0] == [] and [[int(x) for x in t] for t, _ in got[1]] == [[e] for e in ends]
    gaps = []
    want = plain_search(prompts[2], W, 6, W, False, 1.0, 2.0, gaps)
    assert min(gaps) > 4e-7 + max(abs(float(d[1])) for d in want) * 2.0 ** -23
    assert [tuple(int(x) for x in t) for t, _ in got[2]] == [t for t, _ in want]
    s.close()


@pytest.mark.skipif(hip.device_count() < 2, reason="needs a second device")
def test_generate_whose_forward_leaves_another_device_current():
    """On the null stream: the loop's launches and copies go to the search's device."""
    found = []
    for other in (0, 1):
        eng = Engine(PROMPTS[:2], 3, 2.0)
        s = beam.BeamSearch(V, 2, 3, 30.0)

        def forward(step):
            hip.check(hip.lib().hipSetDevice(ctypes.c_int(0)))
            ok = eng.forward(step)
            hip.check(hip.lib().hipSetDevice(ctypes.c_int(other)))
            return ok
        found.append(s.Generate(eng.logits, 2, 3, 6, forward, states=eng.beam_states,
                                cache=eng.beam_cache))
        now = ctypes.c_int(-1)
        hip.check(hip.lib().hipGetDevice(ctypes.byref(now)))
        assert now.value == 0
        s.close()
    for a, b in zip(*found):
        assert [(tuple(t), x) for t, x in a] == [(tuple(t), x) for t, x in b]


def test_generate_refusals_and_failures():
    eng = Engine(PROMPTS[:2], 3, 0.0, pages=6)
    s = beam.BeamSearch(V, 2, 3, 30.0)

    def run(**kw):
        args = dict(d_logits=eng.logits, batch=2, beams=3, max_tokens=4, forward=eng.forward)
        return s.Generate(**dict(args, **kw))
    st = hip.Stream(nonblocking=True)
    other = beam.PageCache(P, 6, 6, eng.slots, planes=1, parts=1, token_bytes=4, stream=st)
    elsewhere = beam.BeamCache(other, [beam.PageState(*b) for b in eng.bufs], eng.pool)
    for kw in [dict(beams=4), dict(beams=0), dict(batch=3), dict(max_tokens=0), dict(n_best=0),
               dict(n_best=4), dict(length_penalty=float("nan")), dict(dtype=3),
               dict(row_stride=V - 1), dict(cache=elsewhere)]:
        with pytest.raises(native.SamplerError) as e:
            run(**kw)
        assert e.value.code == native.G4S_ERR_INVALID_ARGUMENT, kw
    with pytest.raises(native.SamplerError) as e:
        run(forward=lambda step: False)
    assert e.value.code == native.G4S_ERR_ABORTED
    with pytest.raises(native.SamplerError) as e:  # 6 pages: too few for the beams
        run(cache=eng.beam_cache)
    assert e.value.code == native.G4S_ERR_OUT_OF_MEMORY and "pages" in str(e.value)
    with pytest.raises(ZeroDivisionError):
        run(forward=lambda step: 1 // 0)
    s.close()
    other.close()
    st.destroy()
