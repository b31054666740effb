"""Host side of the 8-bit cache (include/gemma4_cache.h): what the entry
points refuse without a GPU, the Pascal unit against the header, and the rules that
the kernels run, on the CPU."""
import ctypes
import math
import os
import random
import subprocess

import numpy as np
import pytest

import test_beam_abi as shared
from gemma4_sampler import beam, cache, hip, native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "gemma4_cache.h")
UNIT = os.path.join(ROOT, "gemma4.pas_amd", "pascal", "Gemma4.Cache.pas")
HOST = os.path.join(ROOT, "tests", "native", "build", "libcache_host.so")
INVALID = native.G4S_ERR_INVALID_ARGUMENT

GOOD = dict(heads=8, kv_heads=2, head_dim=64, scale_tokens=4, rotary_dims=64,
            rotary_pairs="halves")


def geo(**change):
    g = dict(page_tokens=16, n_pages=8, max_rows=4, max_slots=4, planes=2, parts=2,
             token_bytes=68)
    g.update(change)
    page = g["page_tokens"] * g["parts"] * g["token_bytes"]
    return beam.PageGeometry(g["page_tokens"], g["n_pages"], g["max_rows"], g["max_slots"],
                             g["planes"], g["parts"], g["token_bytes"],
                             g.get("plane_stride", page * g["n_pages"]),
                             g.get("page_stride", page))


@pytest.mark.parametrize("change", [
    dict(heads=0), dict(heads=7), dict(heads=1024, kv_heads=64), dict(kv_heads=0),
    dict(heads=130, kv_heads=2), dict(head_dim=0), dict(head_dim=72), dict(head_dim=528),
    dict(head_dim=8), dict(head_dim=-64), dict(scale_tokens=0), dict(scale_tokens=3),
    dict(scale_tokens=32), dict(rotary_dims=-2), dict(rotary_dims=66), dict(rotary_dims=33),
    dict(rotary_pairs=2), dict(rotary_pairs=-1), dict(kv_heads=4), dict(head_dim=128)])
def test_config_limits(change):
    with pytest.raises(native.SamplerError) as e:
        cache.KvCache(geo(), **dict(GOOD, **change))
    assert e.value.code == INVALID


@pytest.mark.parametrize("change", [
    dict(planes=1), dict(planes=0), dict(parts=1), dict(parts=3), dict(token_bytes=64),
    dict(token_bytes=72), dict(page_stride=16 * 2 * 68 + 2),
    dict(plane_stride=16 * 2 * 68 * 8 + 1), dict(n_pages=0), dict(page_tokens=18),
    dict(max_slots=0), dict(page_stride=100),
    dict(page_tokens=65536, max_slots=16385, n_pages=1)])
def test_geometry_limits(change):
    with pytest.raises(native.SamplerError) as e:
        cache.KvCache(geo(**change), **GOOD)
    assert e.value.code == INVALID


def test_geometry_of_a_cache():
    a, b = cache.geometry(16, 8, 4, 4, 2, 64), geo()
    for f, _ in beam.PageGeometry._fields_:
        assert getattr(a, f) == getattr(b, f), f


@pytest.mark.skipif(hip.device_count() > 0, reason="checks the no-device error path")
def test_create_without_device():
    with pytest.raises(native.SamplerError) as e:
        cache.KvCache(geo(), **GOOD)
    assert e.value.code == native.G4S_ERR_NO_DEVICE


def test_null_handles():
    L = cache.load()
    out = ctypes.c_void_p(7)
    assert L.g4s_cache_create(None, None, None, None) == INVALID
    assert L.g4s_cache_create(ctypes.byref(out), None, None, None) == INVALID
    assert out.value is None
    assert L.g4s_cache_create(ctypes.byref(out), ctypes.byref(geo()), None, None) == INVALID
    assert L.g4s_cache_destroy(None) == 0
    assert L.g4s_cache_append(None, None, 1, None, 1, 0, None, None, None, None, None, None, None,
                              0, 1) == INVALID
    assert L.g4s_cache_attend(None, None, 1, None, 1, 0, None, None, 0, 1, 1.0, 0, None,
                              None) == INVALID
    assert L.g4s_cache_last_error(None) == b"cache is NULL"


# --------------------------------------------------------------- Pascal unit


@pytest.fixture
def unit(monkeypatch):
    """The comparisons of test_beam_abi, of this unit and header."""
    monkeypatch.setattr(shared, "UNIT", UNIT)
    monkeypatch.setattr(shared, "HEADER", HEADER)
    monkeypatch.setattr(shared, "PAS2C", dict(
        shared.PAS2C, PG4SCache="g4s_cache*", PPG4SCache="g4s_cache**",
        PG4SCacheConfig="g4s_cache_config*", PG4SCacheView="g4s_cache_view*"))


def test_pascal_externals_match_the_header(unit):
    shared.test_pascal_externals_match_the_header()


@pytest.mark.parametrize("c_name, p_name", [("g4s_cache_config", "TG4SCacheConfig"),
                                            ("g4s_cache_view", "TG4SCacheView")])
def test_pascal_records_match_the_structs(unit, c_name, p_name):
    shared.test_pascal_records_match_the_structs(c_name, p_name)


def test_pascal_and_python_constants_match_the_header(unit):
    import re
    want = {n: int(v) for n, v in re.findall(r"#define\s+(G4S_\w+)\s+(\d+)", shared._c(HEADER))}
    got = {n: int(v) for n, v in re.findall(r"\b(G4S_\w+)\s*=\s*(\d+)\s*;", shared._pascal())}
    assert got == want
    for name in ("HEADS", "KV_HEADS", "GROUP", "HEAD_DIM", "SCALE_TOKENS", "TOKENS", "CONTEXT"):
        assert getattr(cache, "MAX_" + name) == want["G4S_CACHE_MAX_" + name]
    assert cache.ROTARY == {"halves": want["G4S_ROTARY_HALVES"],
                            "neighbours": want["G4S_ROTARY_NEIGHBOURS"]}


# ------------------------------------------------------- rules of the kernels


@pytest.fixture(scope="module")
def host():
    if not os.path.exists(HOST):
        subprocess.run(["make", "-s", "-C", os.path.join(ROOT, "tests", "native")], check=True)
    L = ctypes.CDLL(HOST)
    L.t_cache_offset.restype = ctypes.c_int64
    L.t_cache_offset.argtypes = [ctypes.c_int64] + [ctypes.c_int32] * 5
    L.t_scale_exponent.argtypes = [ctypes.c_double]
    L.t_row_tokens.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32,
                               ctypes.c_int64, ctypes.c_void_p]
    return L


def test_divide(host):
    assert host.t_divide_all(1, 65537) == 0
    rng = random.Random(1)
    for _ in range(20000):
        n, d = rng.randrange(1 << 31), rng.randrange(1, 65537)
        assert host.t_divide(n, d) == n // d


MAX = (1 << 31) - 1


@pytest.mark.parametrize("starts, row, length, tokens, room, want", [
    (None, 3, 9, 4, 64, (3, 1, 9, 0)), (None, 0, 0, 1, 64, (0, 1, 0, 0)),
    (None, 0, 65, 1, 64, (0, 1, 0, 1)), (None, 0, -1, 1, 64, (0, 1, 0, 1)),
    (None, 0, MAX, 1, MAX, (0, 1, MAX, 0)),
    ([0, 5, 9], 1, 9, 9, 64, (5, 4, 9, 0)), ([0, 5, 9], 1, 9, 8, 64, (5, 0, 9, 0)),
    ([0, 5, 5], 1, 9, 9, 64, (5, 0, 9, 0)), ([0, 5, 4], 1, 9, 9, 64, (5, 0, 9, 0)),
    ([-3, 5, 9], 0, 9, 9, 64, (-3, 0, 9, 0)), ([0, MAX, -MAX], 0, 9, 9, 64, (0, 0, 9, 0)),
    ([MAX, -MAX, 0], 0, 9, 9, 64, (MAX, 0, 9, 0))])
def test_row_tokens(host, starts, row, length, tokens, room, want):
    out = np.zeros(4, np.int32)
    lengths = np.full(row + 1, length, np.int32)
    s = None if starts is None else np.array(starts, np.int32)
    host.t_row_tokens(None if s is None else s.ctypes.data, lengths.ctypes.data, row, tokens, room,
                      out.ctypes.data)
    assert tuple(int(x) for x in out) == want


def test_offsets_pass_32_bits(host):
    # the last token of the last head of the last page of a pool of some 70 GB
    page = 4 * 32 * 516
    assert host.t_cache_offset(page, 32 * 516, 516, (1 << 20) - 1, 31, 3) == \
        ((1 << 20) - 1) * page + 3 * 32 * 516 + 31 * 516


def test_scale_exponent(host):
    for top in [0.0, 1e-320, 448.0, math.nextafter(448.0, 500), math.nextafter(448.0, 0), 1.0,
                224.0, 225.0, 1e-30, 3e38, 1e300, 2.0 ** -91, 448.0 * 2.0 ** -100,
                math.nextafter(448.0 * 2.0 ** -100, 1)]:
        e = -100
        while e < 119 and top > 448.0 * 2.0 ** e:
            e += 1
        assert host.t_scale_exponent(top) == e, top


def test_which_bits_are_a_scale(host):
    for x, want in ((0.0, 1), (1e-45, 1), (2.0 ** -100, 1), (1.0, 1), (2.0 ** 119, 1), (1.5 * 2.0 ** 119, 0),
                    (2.0 ** 120, 0), (2.0 ** 127, 0), (math.inf, 0), (math.nan, 0), (-1.0, 0), (-math.inf, 0)):
        bits = int(np.array([x], np.float32).view(np.uint32)[0])
        assert host.t_scale_ok(ctypes.c_uint32(bits)) == want, x


def test_every_tile_of_a_row_has_a_slot(host):
    for tile in (1, 2, 3, 16, 15, 64, 256):
        for start in (0, 1, tile - 1, tile, tile + 1, 1000):
            for count in list(range(0, 2 * tile + 3)) + [1000, 65537]:
                for first in (0, 1, tile - 1, tile, 12345):
                    assert host.t_missing_slots(start, count, first, tile) == 0


def test_every_block_of_columns_has_a_slot(host):
    for unit in (64, 128, 256):
        for group in (1, 3, 8, 17, 64):
            for start in (0, 1, 63, 64, 1000, 1048000):
                for count in list(range(0, 70)) + [255, 256, 257, 576]:
                    assert host.t_missing_blocks(start, count, group, unit) == 0


def test_units_are_shared_out_whole(host):
    host.t_units_shared.argtypes = [ctypes.c_int64, ctypes.c_int32]
    for groups in (1, 2, 3, 255, 256, 512):
        for total in (groups, groups + 1, 2 * groups - 1, 1000 * groups + 7, (1 << 43) + 5):
            assert host.t_units_shared(total, groups) == 1


def _share(host, d, kv, group, counts, lengths, room, window=0, ncu=256, spare=0):
    counts, lengths = np.asarray(counts, np.int32), np.asarray(lengths, np.int32)
    starts = bool((counts != 1).any()) or spare > 0
    host.t_rows_share.argtypes = [ctypes.c_int32] * 5 + [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p,
                                                         ctypes.c_int64, ctypes.c_int32, ctypes.c_int32]
    return host.t_rows_share(d, kv, group, len(counts), int(counts.sum()) + spare, counts.ctypes.data,
                             starts, lengths.ctypes.data, room, window, ncu)


@pytest.mark.parametrize("d, kv, group, new, length, room", [
    (256, 2, 4, 6, 8100, 8192), (256, 2, 4, 10, 3000, 8192), (256, 1, 8, 3, 8100, 8192),
    (512, 1, 8, 4, 8100, 8192), (256, 1, 4, 10, 64, 64), (256, 2, 4, 8, 5000, 8192),
    (256, 1, 1, 48, 128, 128), (512, 2, 4, 8, 500, 520)])
def test_rows_of_several_blocks_of_columns_are_shared_out_whole(host, d, kv, group, new, length, room):
    """One row of 17 to 48 columns in a table that it fills: three blocks go over its tokens."""
    assert _share(host, d, kv, group, [new], [length], room) == 0


def test_no_unit_is_left_to_workgroups_that_are_not_there(host):
    for d in (64, 128, 192, 256, 272, 512):
        for kv, group in ((1, 1), (1, 3), (2, 4), (1, 16), (3, 17), (8, 4), (1, 64), (64, 8)):
            for cols in (1, 15, 16, 17, 24, 31, 32, 33, 47, 48, 49, 200):
                new = max(1, cols // group)
                for room in (1, 16, 64, 127, 128, 129, 1024, 8192, 131072, 1 << 30):
                    for ncu in (1, 64, 256):
                        for rows in (1, 3, 40):
                            length = [max(0, room - r * 7 % (room + 1)) for r in range(rows)]
                            got = _share(host, d, kv, group, [new] * rows, length, room, ncu=ncu,
                                         window=0 if rows < 40 else 100)
                            assert got == 0, (d, kv, group, new, room, ncu, rows, got)
    rng = random.Random(2)
    for _ in range(3000):
        rows, room = rng.randrange(1, 70), int(2 ** rng.uniform(0, 14))
        got = _share(host, rng.randrange(1, 33) * 16, rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 4, 5, 16, 40]),
                     [rng.choice([0, 1, 1, 2, 5, 9, 17, 48, 90]) for _ in range(rows)],
                     [rng.randrange(room + 1) for _ in range(rows)], room,
                     rng.choice([0, 0, 1, 33, 512]), rng.choice([1, 32, 256]), rng.choice([0, 3]))
        assert got == 0


# ---------------------------------------------------- views that lie together


def _bytes_of(v):
    at, tokens, heads, ts, hs, vec = v
    return {at + i * ts + h * hs + x for i in range(tokens) for h in range(heads) for x in range(vec)}


def _meet(host, a, b):
    got = [host.t_vectors_meet((ctypes.c_int64 * 6)(*x), (ctypes.c_int64 * 6)(*y))
           for x, y in ((a, b), (b, a))]
    assert got[0] == got[1]
    return bool(got[0])


def test_parts_of_each_heads_record_are_apart(host):
    """Queries, keys, values and rotated queries of a head side by side, head by head."""
    d, heads, tokens = 8, 4, 5
    for order in ("tokens", "heads"):
        hs = 4 * d if order == "tokens" else 4 * d * tokens
        ts = 4 * d * heads if order == "tokens" else 4 * d
        parts = [(1000 + i * d, tokens, heads, ts, hs, d) for i in range(4)]
        for i, a in enumerate(parts):
            for j, b in enumerate(parts):
                assert _meet(host, a, b) == (i == j)
            assert _meet(host, a, (1000 + i * d + 4,) + a[1:])
    # keys of one head beside queries of several
    assert not _meet(host, (1000, 5, 4, 100, 16, 8), (1008, 5, 1, 100, 0, 8))
    assert not _meet(host, (1000, 1, 4, 0, 16, 8), (1008, 1, 4, 0, 16, 8))
    assert _meet(host, (1000, 1, 4, 0, 16, 8), (1012, 1, 4, 0, 16, 8))


def test_views_meet_where_their_bytes_do(host):
    """Views of the same strides: exactly.  Others: never apart where they are not."""
    rng = random.Random(3)
    exact = met = 0
    for _ in range(30000):
        vec, shape = 4, []
        tokens = rng.randrange(1, 5)
        strides = None
        for _ in range(2):
            heads = rng.randrange(1, 5)
            if strides is None or rng.random() < 0.4:
                inner = vec * rng.randrange(1, 4)
                if rng.random() < 0.5:
                    strides = ("tokens", inner, inner * 4 + vec * rng.randrange(3))
                else:
                    strides = ("heads", inner, inner * 4 + vec * rng.randrange(3))
            kind, s, big = strides
            ts, hs = (big, s) if kind == "tokens" else (s, big)
            shape.append((1000 + rng.randrange(60), tokens, heads, ts if tokens > 1 else 0,
                          hs if heads > 1 else 0, vec))
        a, b = shape
        want, got = bool(_bytes_of(a) & _bytes_of(b)), _meet(host, a, b)
        assert got or not want, (a, b)
        one = [(x[3], x[4]) for x in shape]
        if one[0] == one[1]:
            assert got == want, (a, b)
            exact += 1
            met += want
    assert exact > 5000 and 1000 < met < exact - 1000
    assert not _meet(host, (0, 1, 1, 0, 0, 4), (0, 1, 1, 0, 0, 4))  # (no view)
