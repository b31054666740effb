"""What beam search asks of the library in each decode step, as cases that can
be timed and compared: the selection over beams and vocabulary, the reordering
of the beams' states, and the pages of a cache that the beams share.

Kinds of case:
  select   the best n continuations of every sequence's beams: scores plus
           log-softmax of the softcapped logits
  reorder  rows of contiguous states follow their parents, in place or into a
           second buffer
  advance  one step of a paged cache's tables: rows follow their parents, grow,
           shrink or end; a partly filled page that two rows would write is
           copied first
  compact  the live pages moved into the low end of the pool
  copy     pages copied between pools, the last ones partly filled

`run` calls the library where `own` is true, and computes the same by
elementary torch operations where it is false.
"""
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
V = 262144      # the model's vocabulary
CAP = 30.0      # final logit softcap
DEVICE = "cuda"
MASKED = -1e30  # a logit that is not above this is no candidate


def listed():
    return [
        # one conversation searched with four beams: every step waits for this call
        dict(name="select_1x4_f32", kind="select", vocab=V, batch=1, beams=4, n=8, dtype="f32",
             cap=CAP, banned=0.0, first=False),
        # a few requests on a smaller, odd vocabulary, some tokens banned by a grammar
        dict(name="select_3x5_bf16_odd", kind="select", vocab=100003, batch=3, beams=5, n=10,
             dtype="bf16", cap=CAP, banned=0.02, first=False),
        # a serving batch on the engine's fp32 logits
        dict(name="select_16x4_f32", kind="select", vocab=V, batch=16, beams=4, n=8, dtype="f32",
             cap=CAP, banned=0.0, first=False),
        # the largest batch, eight beams each, bf16 logits
        dict(name="select_64x8_bf16", kind="select", vocab=V, batch=64, beams=8, n=16,
             dtype="bf16", cap=CAP, banned=0.0, first=False),
        # short states of four beams of one sequence, moved where they are
        dict(name="reorder_1x4_inplace", kind="reorder", batch=1, beams=4, planes=12,
             row_bytes=65536, pad=0, inplace=True),
        # long states of a batch into the buffer of the next step, rows of an odd size
        dict(name="reorder_16x4", kind="reorder", batch=16, beams=4, planes=8,
             row_bytes=1500016, pad=112, inplace=False),
        # one sequence's four beams, a short prompt in small pages
        dict(name="advance_1x4", kind="advance", batch=1, beams=4, page_tokens=16, tokens=501,
             spread=1, slots=64, n_pages=256, planes=16, parts=1, token_bytes=512, outer=False,
             mixed=False),
        # a serving batch with long contexts, pages by head, some requests ending and starting
        dict(name="advance_48x4_long", kind="advance", batch=48, beams=4, page_tokens=32,
             tokens=3800, spread=900, slots=256, n_pages=8192, planes=16, parts=2,
             token_bytes=256, outer=False, mixed=True),
        # a small pool after a few requests ended
        dict(name="compact_200", kind="compact", rows=6, page_tokens=16, tokens=270, spread=40,
             slots=40, n_pages=200, planes=8, parts=1, token_bytes=512, outer=False),
        # a large pool, half of it free in holes all over
        dict(name="compact_6000", kind="compact", rows=40, page_tokens=32, tokens=2300,
             spread=400, slots=128, n_pages=6000, planes=16, parts=2, token_bytes=256,
             outer=False),
        # a prompt's pages put aside
        dict(name="copy_7", kind="copy", pairs=7, page_tokens=16, n_pages=64, planes=8, parts=1,
             token_bytes=512, outer=False),
        # many sequences' pages brought back, planes of a page side by side
        dict(name="copy_1501", kind="copy", pairs=1501, page_tokens=32, n_pages=3500, planes=16,
             parts=2, token_bytes=256, outer=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw_pages(rng, budget):
    """Geometry of a pool of at most `budget` bytes."""
    while True:
        c = dict(page_tokens=rng.choice([8, 16, 32, 64]), parts=rng.choice([1, 1, 2, 4]),
                 planes=_log_int(rng, 1, 64), token_bytes=16 * _log_int(rng, 2, 64),
                 outer=rng.random() < 0.3)
        page = c["page_tokens"] * c["parts"] * c["token_bytes"] * c["planes"]
        if page * 128 <= budget:
            return c, budget // page


def draw(rng):
    kind = rng.choice(["select", "select", "select", "reorder", "advance", "advance", "compact",
                       "copy"])
    if kind == "select":
        vocab = V if rng.random() < 0.3 else _log_int(rng, 8000, V)
        dtype = rng.choice(["f32", "bf16"])
        beams = rng.choice([1, 2, 3, 4, 5, 8, 10, 16, 32])
        most = 64 * 8 * V // vocab // beams // (2 if dtype == "f32" else 1)
        return dict(kind=kind, vocab=vocab, batch=_log_int(rng, 1, max(1, min(most, 256))),
                    beams=beams, n=beams * rng.choice([1, 2, 2]), dtype=dtype,
                    cap=rng.choice([CAP, CAP, 0.0]), banned=rng.choice([0.0, 0.0, 0.05, 0.5]),
                    first=rng.random() < 0.2)
    if kind == "reorder":
        batch, beams, planes = _log_int(rng, 1, 32), rng.choice([2, 3, 4, 5, 8, 16, 32]), \
            _log_int(rng, 1, 48)
        most = 8 * 64 * 1500016 // (batch * beams * planes)
        row = _log_int(rng, 4096, max(4097, min(most, 4 << 20)))
        row -= row % rng.choice([4, 16, 16])
        return dict(kind=kind, batch=batch, beams=beams, planes=planes, row_bytes=row,
                    pad=rng.choice([0, 16, 64]) if row % 16 == 0 else rng.choice([0, 4]),
                    inplace=rng.random() < 0.5)
    if kind == "advance":
        c, most = _draw_pages(rng, 1 << 31)
        batch, beams = _log_int(rng, 1, 48), rng.choice([1, 2, 4, 4, 5, 8])
        # pages of a sequence: its prompt's, and up to four of each beam's own
        n_pages = min(most, 8192)
        while batch > 1 and batch * (10 * beams + 8) > n_pages:
            batch //= 2
        each = n_pages // batch - 8 * beams - 2
        if each < 2:
            each, beams = max(2, n_pages // batch - 10), 1
        tokens = _log_int(rng, 1, max(2, min(each, 250) * c["page_tokens"] * 3 // 4))
        spread = max(1, tokens // 5)
        slots = -(-(tokens + spread + 16) // c["page_tokens"]) + rng.choice([4, 5, 16])
        return dict(c, kind=kind, batch=batch, beams=beams, tokens=tokens, spread=spread,
                    slots=slots, n_pages=n_pages, mixed=rng.random() < 0.6)
    c, most = _draw_pages(rng, 3 << 28)
    n_pages = _log_int(rng, 64, max(65, min(most, 16384)))
    if kind == "copy":
        return dict(c, kind=kind, pairs=_log_int(rng, 1, max(1, n_pages * 2 // 5)),
                    n_pages=n_pages)
    rows = _log_int(rng, 1, 64)
    tokens = max(1, n_pages * rng.choice([2, 5, 8]) // (10 * rows) * c["page_tokens"] - 3)
    spread = max(1, tokens // 4)
    while rows > 1 and rows * (tokens + spread + c["page_tokens"]) > n_pages * c["page_tokens"]:
        rows -= 1
    if tokens + spread > n_pages * c["page_tokens"]:
        tokens, spread = n_pages * c["page_tokens"] // 2, 1
    return dict(c, kind=kind, rows=rows, tokens=tokens, spread=spread,
                slots=-(-(tokens + spread) // c["page_tokens"]) + 3, n_pages=n_pages)


# --------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    return g


def _np(seed):
    return np.random.RandomState(seed % (1 << 31))


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEVICE)


def _stride(case):
    """Logits per row: the vocabulary, padded to whole 16-byte vectors."""
    return (case["vocab"] + 7) // 8 * 8


def _logits(case, seed):
    """N(0, 3^2) with 16 candidates raised by 6..12 in each row, as a trained
    model's logits look; banned tokens at the type's lowest value, or -inf."""
    g = _gen(seed)
    R, n = case["batch"] * case["beams"], case["vocab"]
    x = torch.zeros(R, _stride(case), device=DEVICE)
    x[:, :n] = torch.randn(R, n, generator=g, device=DEVICE) * 3.0
    at = torch.randint(0, n, (R, 16), generator=g, device=DEVICE)
    up = 6.0 + 6.0 * torch.rand(R, 16, generator=g, device=DEVICE)
    x.scatter_(1, at, x.gather(1, at) + up)
    t = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    x = x.to(t)
    if case["banned"]:
        off = torch.rand(R, n, generator=g, device=DEVICE) < case["banned"]
        lowest = torch.finfo(t).min if seed % 2 else float("-inf")
        x[:, :n] = x[:, :n].masked_fill(off, lowest)
    return x


def _scores(case, seed):
    """Running log-probabilities, best beam first; before the first token one
    beam of each sequence counts, the others are -inf."""
    B, W = case["batch"], case["beams"]
    if case["first"]:
        s = torch.full((B, W), float("-inf"), device=DEVICE)
        s[:, 0] = 0.0
        return s.reshape(-1)
    s = -20.0 * torch.rand(B, 1, generator=_gen(seed + 1), device=DEVICE)
    step = 1.5 * torch.rand(B, W, generator=_gen(seed + 2), device=DEVICE)
    return (s - step.cumsum(1)).reshape(-1)


def _pool_shape(case):
    """Pools are planes x pages x parts x tokens x words, or pages outermost."""
    a = (case["planes"], case["n_pages"])
    return ((a[1], a[0]) if case["outer"] else a) + \
        (case["parts"], case["page_tokens"], case["token_bytes"] // 4)


def _pool(case, seed):
    return torch.randint(-(1 << 31), 1 << 31, _pool_shape(case), generator=_gen(seed),
                         device=DEVICE, dtype=torch.int32)


def _page_bytes(case):
    return case["parts"] * case["page_tokens"] * case["token_bytes"]


def _lengths(case, count):
    """Tokens of each sequence: fixed by the case, so that its work is too."""
    return [case["tokens"] + (i * 389) % case["spread"] for i in range(count)]


def _survivors(case, r):
    """Parents of one sequence's beams: half of the beams (rounded up) go on,
    in turn, in any order."""
    W = case["beams"]
    keep = r.permutation(W)[:(W + 1) // 2]
    return r.permutation(np.array([keep[i % len(keep)] for i in range(W)]))


def _slots_of(tokens, P):
    return -(-tokens // P)


def _tables(case, seed):
    """A paged cache in use: every sequence's beams share the pages of its
    prompt and hold their own pages behind a fork some tokens ago."""
    r = _np(seed)
    P, W, B = case["page_tokens"], case["beams"], case["batch"]
    free = list(r.permutation(case["n_pages"]))
    table = np.full((B * W, case["slots"]), -1, np.int32)
    lens = np.zeros(B * W, np.int32)
    refs = np.zeros(case["n_pages"], np.int32)
    for b, length in enumerate(_lengths(case, B)):
        used = _slots_of(length, P)
        shared = max(0, used - 1 - b % 3)
        common = [free.pop() for _ in range(shared)]
        for w in range(W):
            row = common + [free.pop() for _ in range(used - shared)]
            table[b * W + w, :used] = row
            lens[b * W + w] = length
            refs[row] += 1
    return table, lens, refs


def _moves(case, seed):
    """Parents and growth of every row. mixed: every 7th sequence ends, every
    11th goes back 5 tokens, every 13th was ended before and starts again from
    nothing with a prompt of 20 tokens; the rest take one token more."""
    r = _np(seed + 3)
    W, B = case["beams"], case["batch"]
    parents = np.zeros(B * W, np.int32)
    grow = np.ones(B * W, np.int32)
    for b in range(B):
        at = slice(b * W, b * W + W)
        parents[at] = b * W + _survivors(case, r)
        if not case["mixed"]:
            continue
        if b % 7 == 6:
            parents[at], grow[at] = -1, 0
        elif b % 11 == 10:
            grow[at] = -5
        elif b % 13 == 12:
            parents[at], grow[at] = -1, 20
    return parents, grow


def _fragments(case, seed):
    """A pool of sequences whose neighbours have ended: rows of pages in any
    order, the second half of the rows sharing its first pages with the first."""
    r = _np(seed)
    P, R = case["page_tokens"], case["rows"]
    free = list(r.permutation(case["n_pages"]))
    table = np.full((R, case["slots"]), -1, np.int32)
    lens = np.array(_lengths(case, R), np.int32)
    refs = np.zeros(case["n_pages"], np.int32)
    for i in range(R):
        used = _slots_of(int(lens[i]), P)
        old = i - (R + 1) // 2
        same = min(used, _slots_of(int(lens[old]), P)) // 4 if old >= 0 else 0
        row = list(table[old, :same]) if same else []
        row += [free.pop() for _ in range(used - same)]
        table[i, :used] = row
        refs[row] += 1
    return table, lens, refs


def _live(case):
    """Pages that are in use in `_fragments`."""
    P, R = case["page_tokens"], case["rows"]
    lens = _lengths(case, R)
    live = 0
    for i in range(R):
        used = _slots_of(lens[i], P)
        old = i - (R + 1) // 2
        live += used - (min(used, _slots_of(lens[old], P)) // 4 if old >= 0 else 0)
    return live


def _binding():
    at = os.path.join(ROOT, "gemma4.pas_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from gemma4_sampler import beam
    return beam


def _page_cache(case, rows):
    page = _page_bytes(case)
    strides = dict(plane_stride=page, page_stride=page * case["planes"]) if case["outer"] else \
        dict(plane_stride=page * case["n_pages"], page_stride=page)
    return _binding().PageCache(case["page_tokens"], case["n_pages"], max_rows=rows,
                                max_slots=case.get("slots", 1), planes=case["planes"],
                                parts=case["parts"], token_bytes=case["token_bytes"], **strides)


def _two_states(st, case, made):
    """The state as it is, and arrays for the one that follows."""
    st["from"] = [_i32(a) for a in made]
    rows = made[0].shape[0]
    st["to"] = [torch.full((rows, case["slots"]), -1, dtype=torch.int32, device=DEVICE),
                torch.zeros(rows, dtype=torch.int32, device=DEVICE),
                torch.zeros(case["n_pages"], dtype=torch.int32, device=DEVICE)]
    st["status"] = torch.zeros(4, dtype=torch.int32, device=DEVICE)
    if own:
        beam = _binding()
        st["cache"] = _page_cache(case, rows)
        st["states"] = [beam.PageState(*(t.data_ptr() for t in st[k])) for k in ("from", "to")]


def prepare(case, seed):
    st = dict(case=case)
    kind = case["kind"]
    if kind in ("select", "reorder"):
        B, W = case["batch"], case["beams"]
        if own:
            st["search"] = _binding().BeamSearch(case.get("vocab", V), max_batch=B, max_beams=W,
                                                 softcap=case.get("cap", CAP))
    if kind == "select":
        st["logits"], st["scores"] = _logits(case, seed), _scores(case, seed)
        i32 = dict(dtype=torch.int32, device=DEVICE)
        st["out"] = dict(parents=torch.zeros(B, case["n"], **i32),
                         tokens=torch.zeros(B, case["n"], **i32),
                         scores=torch.zeros(B, case["n"], device=DEVICE),
                         lse=torch.zeros(B * W, device=DEVICE))
    elif kind == "reorder":
        r = _np(seed + 3)
        if case["inplace"]:
            # the beams that go on stay where they are: doing it twice changes nothing
            parents = np.zeros((B, W), np.int32)
            for b in range(B):
                keep = r.permutation(W)[:(W + 1) // 2]
                parents[b] = b * W + keep[np.arange(W) % len(keep)]
                parents[b, keep] = b * W + keep
                gone = np.setdiff1d(np.arange(W), keep)
                parents[b, gone] = b * W + keep[:len(gone)]
        else:
            parents = np.stack([b * W + _survivors(case, r) for b in range(B)])
        st["parents"] = _i32(parents.reshape(-1))
        shape = (case["planes"], B * W, (case["row_bytes"] + case["pad"]) // 4)
        st["src"] = torch.randint(-(1 << 31), 1 << 31, shape, generator=_gen(seed),
                                  device=DEVICE, dtype=torch.int32)
        st["dst"] = st["src"] if case["inplace"] else torch.zeros_like(st["src"])
    elif kind == "advance":
        _two_states(st, case, _tables(case, seed))
        st["parents"], st["grow"] = (_i32(a) for a in _moves(case, seed))
        st["pool"] = _pool(case, seed)
    elif kind == "compact":
        _two_states(st, case, _fragments(case, seed))
        st["pool"] = _pool(case, seed)
    else:
        r = _np(seed + 4)
        P, n = case["page_tokens"], case["pairs"]
        st["pool"], st["pool2"] = _pool(case, seed), _pool(case, seed + 1)
        st["src"], st["dst"] = (_i32(r.permutation(case["n_pages"])[:n]) for _ in range(2))
        tokens = np.full(n, P)
        tokens[::5] = 1 + np.arange(len(tokens[::5])) * 7 % P  # every fifth ends inside its page
        st["tokens"] = _i32(tokens)
        if own:
            st["cache"] = _page_cache(case, 1)
    return st


# ------------------------------------------------------------ plain forms


def _best_of_rows(x, n):
    """Each row's n largest candidates, the larger logit first and of equal
    ones the lower token: (logits, tokens, which of them exist)."""
    bits = x.view(torch.int32).to(torch.int64) & 0xFFFFFFFF
    bits = torch.where(x == 0, 0, bits)
    order = torch.where(bits >= 1 << 31, 0xFFFFFFFF - bits, bits + (1 << 31))
    order = torch.where(x > MASKED, order, 0)
    low = (1 << 31) - 1
    key = (order << 31) + (low - torch.arange(x.shape[1], device=x.device))
    top = torch.topk(key, n, dim=1).values
    tokens = low - (top & low)
    return x.gather(1, tokens), tokens, (top >> 31) > 0


def _select(st):
    """Softcap, normaliser and scores in 64 bits: candidates of different
    beams lie next to each other, and which of them is the better one has to
    come out whole."""
    case = st["case"]
    B, W, n, cap = case["batch"], case["beams"], case["n"], case["cap"]

    def capped(x):
        x = x.double()
        return cap * torch.tanh(x / cap) if cap > 0 else x

    found, norms = [], []
    for lo in range(0, B * W, 64):
        x = st["logits"][lo:lo + 64, :case["vocab"]].float().contiguous()
        y = torch.where(x > MASKED, capped(x), float("-inf"))
        m = y.max(dim=1, keepdim=True).values
        lse = m + torch.log(torch.exp(y - m).sum(dim=1, keepdim=True))
        best, tokens, real = _best_of_rows(x, n)
        score = st["scores"][lo:lo + 64].unsqueeze(1)
        real = real & (score > MASKED)
        norms.append(torch.where(score > MASKED, lse, float("-inf")).squeeze(1))
        found.append((torch.where(real, score.double() + (capped(best) - lse), float("-inf")),
                      tokens, real))
    score, tokens, real = (torch.cat(t).reshape(B, W * n) for t in zip(*found))
    score, at = torch.sort(score, dim=1, descending=True, stable=True)
    score, at = score[:, :n], at[:, :n]
    real = real.gather(1, at)
    row = torch.arange(B, device=at.device).unsqueeze(1) * W + at // n
    return dict(parents=torch.where(real, row, -1).int(),
                tokens=torch.where(real, tokens.gather(1, at), -1).int(), scores=score.float(),
                lse=torch.cat(norms).float())


def _reorder(st):
    case = st["case"]
    words = case["row_bytes"] // 4
    st["dst"][:, :, :words] = st["src"][:, :, :words][:, st["parents"].long()]
    return st["dst"]


def _pages_of(pool, case, ids):
    return pool[ids] if case["outer"] else pool[:, ids]


def _copy_pages(src_pool, dst_pool, case, src, dst, tokens):
    """The first tokens[i] tokens of page src[i] into page dst[i]."""
    t = torch.arange(case["page_tokens"], device=src.device) < tokens.unsqueeze(1)
    shape = (len(src), 1, 1, case["page_tokens"], 1) if case["outer"] else \
        (1, len(src), 1, case["page_tokens"], 1)
    new = torch.where(t.reshape(shape), _pages_of(src_pool, case, src),
                      _pages_of(dst_pool, case, dst))
    if case["outer"]:
        dst_pool[dst] = new
    else:
        dst_pool[:, dst] = new


def _advance(st):
    case = st["case"]
    P, S, N = case["page_tokens"], case["slots"], case["n_pages"]
    table, lens, refs = st["from"]
    parents, grow = st["parents"].long(), st["grow"].long()
    R = len(parents)
    alive = parents >= 0
    par = parents.clamp(min=0)
    old = torch.where(alive, lens[par].long(), 0)
    new = (old + grow).clamp(min=0)
    keep = torch.minimum(old, new)
    kept = (keep + P - 1) // P
    slot = torch.arange(S, device=DEVICE)
    rows = torch.where(slot < kept.unsqueeze(1), table[par].long(), -1)
    holders = torch.zeros(N + 1, dtype=torch.long, device=DEVICE)
    holders.index_add_(0, torch.where(rows >= 0, rows, N).reshape(-1),
                       torch.ones(R * S, dtype=torch.long, device=DEVICE))
    # the partly filled page that a growing row goes on writing
    writes = (new > keep) & (keep % P != 0)
    page = rows.gather(1, (kept - 1).clamp(min=0).unsqueeze(1)).squeeze(1)
    page = torch.where(writes, page, N)
    writers = torch.zeros(N + 1, dtype=torch.long, device=DEVICE)
    writers.index_add_(0, page, torch.ones(R, dtype=torch.long, device=DEVICE))
    index = torch.arange(R, device=DEVICE)
    first = torch.full((N + 1,), R, dtype=torch.long, device=DEVICE)
    first.scatter_reduce_(0, page, index, "amin")
    stays = (holders[page] == writers[page]) & (first[page] == index)
    copies = writes & ~stays
    # free pages, the lowest first: a row's copy, then its new slots
    need = (new + P - 1) // P - kept + copies.long()
    base = need.cumsum(0) - need
    free = torch.argsort((refs != 0).int(), stable=True)
    k = slot - kept.unsqueeze(1) + copies.long().unsqueeze(1)
    fresh = (slot < ((new + P - 1) // P).unsqueeze(1)) & (k >= 0)
    took = free[(base.unsqueeze(1) + k).clamp(0, N - 1)]
    result = torch.where(fresh, took, rows)
    st["to"][0].copy_(torch.where(result >= 0, result.int(), st["to"][0]))
    st["to"][1].copy_(new)
    held = torch.zeros(N + 1, dtype=torch.long, device=DEVICE)
    held.index_add_(0, torch.where(result >= 0, result, N).reshape(-1),
                    torch.ones(R * S, dtype=torch.long, device=DEVICE))
    st["to"][2].copy_(held[:N])
    at = copies.nonzero().squeeze(1)
    _copy_pages(st["pool"], st["pool"], case, page[at], free[base[at]], (keep % P)[at])
    st["status"].copy_(torch.stack([torch.zeros_like(need.sum()), (held[:N] == 0).sum(),
                                    need.sum(), copies.sum()]))


def _compact(st):
    case = st["case"]
    table, lens, refs = st["from"]
    live = refs > 0
    n = live.sum()
    index = torch.arange(case["n_pages"], device=DEVICE)
    src = (live & (index >= n)).nonzero().squeeze(1)
    dst = (~live & (index < n)).nonzero().squeeze(1)
    to = index.clone()
    to[src] = dst
    used = (lens.long() + case["page_tokens"] - 1) // case["page_tokens"]
    held = torch.arange(case["slots"], device=DEVICE) < used.unsqueeze(1)
    st["to"][0].copy_(torch.where(held, to[table.clamp(min=0).long()].int(), st["to"][0]))
    st["to"][1].copy_(lens)
    after = torch.where(index < n, refs, 0)
    after[dst] = refs[src]
    st["to"][2].copy_(after)
    pages = _pages_of(st["pool"], case, src)
    if case["outer"]:
        st["pool"][dst] = pages
    else:
        st["pool"][:, dst] = pages
    moved = torch.full_like(n, len(src))
    st["status"].copy_(torch.stack([n * 0, case["n_pages"] - n, n * 0, moved]))


def _run_plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "select":
        return _select(st)
    if kind == "reorder":
        return _reorder(st)
    if kind == "copy":
        _copy_pages(st["pool"], st["pool2"], case, st["src"].long(), st["dst"].long(),
                    st["tokens"])
    else:
        (_advance if kind == "advance" else _compact)(st)
    return _page_outputs(st)


def _page_outputs(st):
    if st["case"]["kind"] == "copy":
        return st["pool2"]
    return dict(table=st["to"][0], lengths=st["to"][1], refs=st["to"][2], status=st["status"],
                pool=st["pool"])


# -------------------------------------------------------------- one pass


def run(st):
    if not own:
        return _run_plain(st)
    case = st["case"]
    kind = case["kind"]
    if kind == "select":
        native = _binding().native
        o = st["out"]
        st["search"].select(st["logits"].data_ptr(), case["batch"], case["beams"],
                            st["scores"].data_ptr(), case["n"], o["parents"].data_ptr(),
                            o["tokens"].data_ptr(), o["scores"].data_ptr(),
                            d_lse=o["lse"].data_ptr(), dtype=native.DTYPE_F32 if case["dtype"] == "f32" else
                            native.DTYPE_BF16, row_stride=_stride(case))
        return o
    if kind == "reorder":
        row = case["row_bytes"] + case["pad"]
        st["search"].reorder(st["src"].data_ptr(), st["dst"].data_ptr(), case["planes"],
                             row * case["batch"] * case["beams"], case["batch"], case["beams"],
                             row, case["row_bytes"], st["parents"].data_ptr())
        return st["dst"]
    if kind == "advance":
        rows = case["batch"] * case["beams"]
        st["cache"].advance(st["states"][0], rows, st["states"][1], rows,
                            st["parents"].data_ptr(), st["grow"].data_ptr(),
                            st["pool"].data_ptr(), st["status"].data_ptr())
    elif kind == "compact":
        st["cache"].compact(st["states"][0], st["states"][1], case["rows"],
                            st["pool"].data_ptr(), st["status"].data_ptr())
    else:
        st["cache"].copy(st["pool"].data_ptr(), st["pool2"].data_ptr(), case["pairs"],
                         st["src"].data_ptr(), st["dst"].data_ptr(), st["tokens"].data_ptr())
    return _page_outputs(st)


def _copied_tokens(case):
    """Tokens that `_moves` makes rows copy, in all: of a sequence's beams the
    second of each pair of twins, where the last page is partly filled."""
    W, P = case["beams"], case["page_tokens"]
    total = 0
    for b, length in enumerate(_lengths(case, case["batch"])):
        if case["mixed"] and (b % 7 == 6 or b % 11 == 10 or b % 13 == 12):
            continue
        total += (W // 2) * (length % P)
    return total


def work(case):
    kind = case["kind"]
    if kind == "select":
        each = 4 if case["dtype"] == "f32" else 2
        rows = case["batch"] * (1 if case["first"] else case["beams"])
        size = rows * case["vocab"] * each + 8 * case["batch"] * case["beams"] + \
            12 * case["batch"] * case["n"]
        # per logit: softcap, exponential and sum
        return {"bytes": size, "flops": 6 * rows * case["vocab"]}
    if kind == "reorder":
        W = case["beams"]
        rows = (W // 2) * 2 if case["inplace"] else W + (W + 1) // 2
        return {"bytes": case["batch"] * (rows * case["planes"] * case["row_bytes"] + 4 * W),
                "flops": 0}
    P = case["page_tokens"]
    token = case["planes"] * case["parts"] * case["token_bytes"]
    if kind == "advance":
        used = sum(_slots_of(n, P) for n in _lengths(case, case["batch"])) * case["beams"]
        rows = case["batch"] * case["beams"]
        return {"bytes": 2 * token * _copied_tokens(case) + 8 * used + 8 * case["n_pages"] +
                16 * rows + 16, "flops": 0}
    if kind == "compact":
        live = _live(case)
        moved = live * (case["n_pages"] - live) // case["n_pages"]  # on average
        used = sum(_slots_of(n, P) for n in _lengths(case, case["rows"]))
        return {"bytes": 2 * token * P * moved + 8 * used + 8 * case["n_pages"] +
                8 * case["rows"] + 16, "flops": 0}
    n = case["pairs"]
    part = (n + 4) // 5
    tokens = (n - part) * P + sum(1 + i * 7 % P for i in range(part))
    return {"bytes": 2 * token * tokens + 12 * n, "flops": 0}


# ------------------------------------------------------------- 64 bits


def exact(case, seed):
    """Scores of the selected candidates from the definition: every candidate
    of a sequence's beams in one list; the logarithm of each beam's softmax
    denominator. All else is whole numbers."""
    if case["kind"] != "select":
        return None
    B, W, n = case["batch"], case["beams"], case["n"]
    x = _logits(case, seed)[:, :case["vocab"]].reshape(B, W, -1)
    s = _scores(case, seed).reshape(B, W)
    out = torch.full((B, n), float("-inf"), dtype=torch.float64, device=DEVICE)
    norms = torch.full((B, W), float("-inf"), dtype=torch.float64, device=DEVICE)
    for b in range(B):
        z = x[b].double()
        off = z <= MASKED
        if case["cap"] > 0:
            z = torch.tanh(z / case["cap"]) * case["cap"]
        z = z.masked_fill(off, float("-inf"))
        total = torch.logsumexp(z, dim=1)
        norms[b] = torch.where(s[b] > MASKED, total, norms[b])
        z = z - total[:, None] + s[b].double()[:, None]
        best = torch.sort(z.flatten(), descending=True).values[:n]
        out[b, :len(best)] = best
    return dict(parents=None, tokens=None, scores=out, lse=norms.reshape(-1))
