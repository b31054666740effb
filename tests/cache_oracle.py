"""The 8-bit cache of gemma4_cache.h in 64 bits, token by token.

E4M3 values are told apart by a table of all of them; nothing here comes from
the library."""
import numpy as np

E4M3 = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
                 for e in range(16) for m in range(8)])
E4M3[127] = np.nan
E4M3 = np.concatenate([E4M3, -E4M3])


def encode(x):
    """Codes of the nearest e4m3 values, ties to even; NaN gives 0x7F or 0xFF."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    a = np.where(np.isnan(a), 0.0, a)
    hi = np.minimum(np.searchsorted(E4M3[:127], a), 126)
    lo = np.maximum(hi - 1, 0)
    up, down = E4M3[hi] - a, a - E4M3[lo]
    code = np.where(up < down, hi, np.where(up > down, lo, np.where(hi % 2 == 0, hi, lo)))
    code = np.where(a == E4M3[hi], hi, code)
    code = np.where(np.isnan(x), 127, code)
    return (code + 128 * np.signbit(x)).astype(np.uint8)


def scale_of(top):
    """Least power of two (2^-100 .. 2^119) with top <= 448 * scale."""
    e = -100
    while e < 119 and top > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


class Cache:
    """codes [plane][page][head][token][dim], scales [plane][page][head][token]
    of a pool's bytes, and a state's table and lengths."""

    def __init__(self, pool, geo, block):
        self.geo, self.block = geo, block
        self.d = geo.token_bytes - 4
        cells = np.lib.stride_tricks.as_strided(
            pool, (geo.planes, geo.n_pages, geo.parts, geo.page_tokens, geo.token_bytes),
            (geo.plane_stride, geo.page_stride, geo.page_tokens * geo.token_bytes,
             geo.token_bytes, 1))
        self.codes = cells[..., :self.d].copy()
        self.scales = np.ascontiguousarray(cells[..., self.d:]).view(np.float32)[..., 0].copy()

    def place(self, table, row, t):
        """page and place in it of a row's token, or None"""
        page = int(table[row, t // self.geo.page_tokens])
        return (page, t % self.geo.page_tokens) if 0 <= page < self.geo.n_pages else None

    def value(self, plane, table, row, t, head):
        at = self.place(table, row, t)
        if at is None:
            return np.full(self.d, np.nan)
        page, o = at
        return E4M3[self.codes[plane, page, head, o]] * \
            float(self.scales[plane, page, head, o - o % self.block])


def rows_of(starts, lengths, rows, tokens, room):
    """(row, first token, count, length) of the rows; a bad length is None"""
    out = []
    for r in range(rows):
        a, b = (r, r + 1) if starts is None else (int(starts[r]), int(starts[r + 1]))
        n = int(lengths[r])
        out.append((r, a, b - a, n if 0 <= n <= room else None))
    return out


def rotate(x, position, freqs, rotary, neighbours):
    """x [heads, dim] in 64 bits"""
    y = x.copy()
    half = rotary // 2
    angle = np.float64(position) * freqs.astype(np.float64)
    c, s = np.cos(angle), np.sin(angle)
    i = np.arange(half) * 2 if neighbours else np.arange(half)
    j = i + 1 if neighbours else i + half
    y[:, i] = x[:, i] * c - x[:, j] * s
    y[:, j] = x[:, j] * c + x[:, i] * s
    return y


def append(cache, table, lengths, starts, rows, tokens, q, k, v, q_out, positions, freqs, rotary,
           neighbours, planes=(0, 1)):
    """In place on `cache` and q_out (64 bits)."""
    B, geo = cache.block, cache.geo
    room = geo.max_slots * geo.page_tokens
    for r, a, n, length in rows_of(starts, lengths, rows, tokens, room):
        if length is None:
            continue
        new = {}
        for i in range(n):
            t = length - n + i
            if t < 0:
                continue
            p = t if positions is None else int(positions[a + i])
            if q is not None:
                q_out[a + i] = rotate(q[a + i], p, freqs, rotary, neighbours)
            if k is not None:
                new.setdefault(t // B, []).append(
                    (t, rotate(k[a + i], p, freqs, rotary, neighbours), v[a + i]))
        for b, toks in new.items():
            at = cache.place(table, r, b * B)
            if at is None:
                continue
            page, o = at
            before = toks[0][0] - b * B
            for plane, which in zip(planes, (1, 2)):
                for h in range(geo.parts):
                    x = np.stack([tok[which][h] for tok in toks])
                    fin = np.abs(x[np.isfinite(x)])
                    s = scale_of(fin.max() if fin.size else 0.0)
                    if before:
                        old = float(cache.scales[plane, page, h, o])
                        if old >= s:
                            s = old
                        else:
                            was = cache.codes[plane, page, h, o:o + before]
                            cache.codes[plane, page, h, o:o + before] = \
                                encode(np.where(was >= 128, -1.0, 1.0) *
                                       E4M3[was & 127] * (old / s))
                    cache.scales[plane, page, h, o] = s
                    cache.codes[plane, page, h, o + before:o + before + len(toks)] = encode(x / s)


class Attended:
    """out [tokens, heads, dim] and lse [tokens, heads] in 64 bits, and what errors scale with:
    `mass`, the weighted mean of |value|; `size`, the largest sum of |q * key| * |scale|;
    `seen`, how many tokens."""

    def __init__(self, tokens, heads, dim):
        self.out = np.full((tokens, heads, dim), 77.0)
        self.lse = np.full((tokens, heads), 77.0)
        self.mass = np.zeros((tokens, heads, dim))
        self.size = np.zeros((tokens, heads))
        self.seen = np.zeros((tokens, heads), np.int64)


def attend(cache, table, lengths, starts, rows, tokens, q, scale, window, planes=(0, 1)):
    geo = cache.geo
    room = geo.max_slots * geo.page_tokens
    heads = q.shape[1]
    group = heads // geo.parts
    to = Attended(tokens, heads, cache.d)
    for r, a, n, length in rows_of(starts, lengths, rows, tokens, room):
        if length is None:
            to.out[a:a + n], to.lse[a:a + n] = np.nan, np.nan
            continue
        kv = [np.array([[cache.value(p, table, r, t, h) for t in range(length)]
                        for h in range(geo.parts)]).reshape(geo.parts, length, cache.d)
              for p in planes]
        for i in range(n):
            t = length - n + i
            lo = max(0, t - window + 1) if window else 0
            if t < 0:
                to.out[a + i], to.lse[a + i] = 0.0, -np.inf
                continue
            for h in range(heads):
                x, k, v = q[a + i, h], kv[0][h // group, lo:t + 1], kv[1][h // group, lo:t + 1]
                to.seen[a + i, h] = t + 1 - lo
                if not np.isfinite(x).all() or np.isnan(k).any():
                    to.out[a + i, h], to.lse[a + i, h] = np.nan, np.nan
                    continue
                s = scale * (k @ x)
                m = s.max()
                to.lse[a + i, h] = m + np.log(np.exp(s - m).sum())
                p = np.exp(s - to.lse[a + i, h])
                to.out[a + i, h], to.mass[a + i, h] = p @ v, p @ np.abs(v)
                to.size[a + i, h] = (np.abs(scale) * (np.abs(k) @ np.abs(x))).max()
    return to


def limits(to, dim, dtype):
    """How far outputs and lse may be off, by the arithmetic that gemma4_cache.h states.

    A score is a sum of dim products (exact) in 32 bits, scaled and taken to base two: it is off by
    at most (dim + 8) / 2^24 of `size`, and so is the maximum under it.  A sum over the tokens
    seen, with a rounding each and a few for the exponential and the joining: seen + 16 steps
    of 2^-23.  Weights are rounded to bf16 (2^-8) for bf16 outputs alone."""
    score = (dim + 8) * 2.0 ** -24 * to.size
    sums = (to.seen + 16) * 2.0 ** -23
    weight, half = (0.0, 2.0 ** -24) if dtype == "f32" else (2.0 ** -8, 2.0 ** -8)
    rel = 2 * score + sums + weight
    out = rel[..., None] * to.mass + half * np.abs(to.out) + 1e-37
    lse = score + sums + 2.0 ** -23 * np.abs(np.where(np.isfinite(to.lse), to.lse, 0.0))
    return out, lse
