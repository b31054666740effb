"""Plain restatements, on the host, of what include/gemma4_beam.h defines:
the selection in binary64, and one step of a paged cache row by row."""
import numpy as np

MASKED = np.float32(-1e30)


def widen(x):
    """binary32 values of float32 or bf16 (uint16) logits"""
    return x if x.dtype == np.float32 else (x.astype(np.uint32) << 16).view(np.float32)


def bf16(x):
    """float32 rounded to bf16 bits, to nearest even (finite x)"""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def softcap64(x, cap):
    x = x.astype(np.float64)
    return cap * np.tanh(x / cap) if cap > 0 else x


def row_terms(x, cap):
    """(unmasked, y - top, log of the sum relative to top, top) of a row"""
    x = widen(x)
    with np.errstate(invalid="ignore"):
        ok = x > MASKED
    if not ok.any():
        return ok, None, None, -np.inf
    y = softcap64(np.where(ok, x, 0), cap)
    top = y[ok].max()
    with np.errstate(invalid="ignore"):
        d = np.where(y == top, 0.0, y - top)
    return ok, d, np.log(np.exp(d[ok]).sum()), top


def select(rows, scores, beams, n, cap):
    """(parents, tokens, scores in binary64, lse) for `rows` (R x V logits)"""
    R = len(rows)
    lse = np.full(R, -np.inf)
    out = []
    for b in range(R // beams):
        cand = []
        for w in range(beams):
            r = b * beams + w
            s = np.float64(scores[r])
            if not s > MASKED:
                continue
            ok, d, ls, top = row_terms(rows[r], cap)
            if d is None:
                continue
            lse[r] = top + ls
            x = widen(rows[r])
            at = np.flatnonzero(ok & (d > -np.inf))
            # larger logits first, then lower tokens
            at = at[np.lexsort((at, -x[at].astype(np.float64)))][:n]
            sc = np.minimum.accumulate(s + (d[at] - ls))
            cand += [(-sc[i], w, i, r, int(at[i])) for i in range(len(at))]
        cand.sort()
        cand = cand[:n]
        short = n - len(cand)
        out.append(([c[3] for c in cand] + [-1] * short, [c[4] for c in cand] + [-1] * short,
                    [-c[0] for c in cand] + [-np.inf] * short))
    p, t, s = (np.array([o[i] for o in out]) for i in range(3))
    return p.astype(np.int32), t.astype(np.int32), s, lse


class State:
    """table, lengths and refs of a paged cache"""

    def __init__(self, rows, slots, n_pages):
        self.table = np.full((rows, slots), -1, np.int32)
        self.lengths = np.zeros(rows, np.int32)
        self.refs = np.zeros(n_pages, np.int32)

    def copy(self):
        o = State(*self.table.shape, len(self.refs))
        o.table[:], o.lengths[:], o.refs[:] = self.table, self.lengths, self.refs
        return o


def advance(src, from_rows, dst, rows, parents, grow, P):
    """One step from src into dst; (status, copies) with copies as (source page,
    destination page, tokens)."""
    S, N = src.table.shape[1], len(src.refs)

    def refused(code):
        dst.lengths[:rows] = 0
        dst.refs[:] = 0
        return (code, N, 0, 0), []

    used, new, keeps, bad = [], [], [], False
    for r in range(rows):
        p = int(parents[r])
        old = int(src.lengths[p]) if 0 <= p < from_rows else 0
        length = max(0, old + int(grow[r]))
        if not -1 <= p < from_rows or not 0 <= old <= S * P or length > S * P:
            bad, old, length, p = True, 0, 0, -1
        keep = min(old, length)
        row = [int(src.table[p, i]) for i in range(-(-keep // P))]
        if any(not 0 <= g < N or src.refs[g] <= 0 for g in row):
            return refused(-8)
        used.append(row)
        new.append(length)
        keeps.append(keep)
    if bad:
        return refused(-1)
    free = [g for g in range(N) if src.refs[g] <= 0]
    writer = [used[r][-1] if new[r] > keeps[r] and keeps[r] % P else -1 for r in range(rows)]
    taken, copies, final = 0, [], []
    for r in range(rows):
        row, w = list(used[r]), writer[r]
        if w >= 0:
            holders = [q for q in range(rows) if w in used[q]]
            alone = all(writer[q] == w for q in holders) and holders[0] == r
            if not alone:
                if taken >= len(free):
                    return refused(-4)
                copies.append((w, free[taken], keeps[r] % P))
                row[-1] = free[taken]
                taken += 1
        while len(row) < -(-new[r] // P):
            if taken >= len(free):
                return refused(-4)
            row.append(free[taken])
            taken += 1
        final.append(row)
    dst.refs[:] = 0
    for r in range(rows):
        dst.table[r, :len(final[r])] = final[r]
        dst.lengths[r] = new[r]
        for g in final[r]:
            dst.refs[g] += 1
    return (0, int((dst.refs == 0).sum()), taken, len(copies)), copies


def compact(src, dst, rows, P):
    """Compaction of src into dst; (status, moves)."""
    N = len(src.refs)
    live = [g for g in range(N) if src.refs[g] > 0]
    n = len(live)
    holes = [g for g in range(n) if src.refs[g] <= 0]
    to = dict(zip([g for g in live if g >= n], holes))
    for r in range(rows):
        k = -(-int(src.lengths[r]) // P)
        dst.table[r, :k] = [to.get(int(g), int(g)) for g in src.table[r, :k]]
        dst.lengths[r] = src.lengths[r]
    dst.refs[:] = 0
    for g in live:
        dst.refs[to.get(g, g)] = src.refs[g]
    return (0, N - n, 0, len(to)), sorted(to.items())
