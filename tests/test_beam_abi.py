"""Host side of the beam search and the page cache (include/gemma4_beam.h):
what the entry points refuse without a GPU, the Pascal unit against the
header, and the rules that the page kernels run, on the CPU."""
import ctypes
import gc
import os
import re
import subprocess
import weakref

import numpy as np
import pytest

from gemma4_sampler import beam, hip, native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "gemma4_beam.h")
UNIT = os.path.join(ROOT, "gemma4.pas_amd", "pascal", "Gemma4.Beam.pas")
HOST = os.path.join(ROOT, "tests", "native", "build", "libpages_host.so")
INVALID = native.G4S_ERR_INVALID_ARGUMENT


# ------------------------------------------------------------------ refusals


@pytest.mark.parametrize("args, code", [
    ((1, 1, 4, 30.0), INVALID), (((1 << 22) + 1, 1, 4, 30.0), native.G4S_ERR_UNSUPPORTED),
    ((100, 0, 4, 30.0), INVALID), ((100, 1, 0, 30.0), INVALID),
    ((100, 1, beam.MAX_BEAMS + 1, 30.0), INVALID), ((100, 1024, 64, 30.0), INVALID),
    ((100, 1, 4, float("nan")), INVALID), ((100, 1, 4, float("inf")), INVALID)])
def test_search_limits(args, code):
    with pytest.raises(native.SamplerError) as e:
        beam.BeamSearch(*args)
    assert e.value.code == code


GOOD = dict(page_tokens=16, n_pages=8, max_rows=4, max_slots=4, planes=2, parts=2, token_bytes=32)


@pytest.mark.parametrize("change", [
    dict(page_tokens=0), dict(page_tokens=65537), dict(n_pages=0),
    dict(n_pages=beam.PAGES_MAX_PAGES + 1), dict(max_rows=0),
    dict(max_rows=beam.PAGES_MAX_ROWS + 1), dict(max_slots=0),
    dict(page_tokens=65536, max_slots=32768),
    dict(page_tokens=1, max_slots=beam.PAGES_MAX_PAGES + 1), dict(planes=-1), dict(parts=0),
    dict(token_bytes=0), dict(token_bytes=-32), dict(token_bytes=1 << 30),
    dict(page_stride=1023), dict(page_stride=-1024), dict(plane_stride=1024 * 8 - 1),
    dict(page_stride=2048, plane_stride=1023), dict(page_stride=1 << 60)])
def test_page_geometry_limits(change):
    with pytest.raises(native.SamplerError) as e:
        beam.PageCache(**dict(GOOD, **change))
    assert e.value.code == INVALID


@pytest.mark.skipif(hip.device_count() > 0, reason="checks the no-device error path")
def test_creates_without_device():
    for make in (lambda: beam.BeamSearch(100), lambda: beam.PageCache(**GOOD)):
        with pytest.raises(native.SamplerError) as e:
            make()
        assert e.value.code == native.G4S_ERR_NO_DEVICE


def test_null_handles():
    L = beam.load()
    out = ctypes.c_void_p(7)
    assert L.g4s_beam_create(None, 100, 1, 4, 30.0, None) == INVALID
    assert L.g4s_pages_create(None, None, None) == INVALID
    assert L.g4s_pages_create(ctypes.byref(out), None, None) == INVALID and out.value is None
    assert L.g4s_beam_destroy(None) == 0 and L.g4s_pages_destroy(None) == 0
    assert L.g4s_beam_select(None, None, 0, 0, 1, 1, None, 1, None, None, None, None) == INVALID
    assert L.g4s_beam_reorder(None, None, None, 1, 0, 1, 1, 0, 0, None) == INVALID
    assert L.g4s_beam_last_error(None) == b"beam is NULL"
    assert L.g4s_pages_advance(None, None, 1, None, 1, None, None, None, None) == INVALID
    assert L.g4s_pages_compact(None, None, None, 1, None, None) == INVALID
    assert L.g4s_pages_copy(None, None, None, 1, None, None, None) == INVALID
    assert L.g4s_pages_last_error(None) == b"pages is NULL"
    assert L.g4s_beam_generate(None, 1, None, None, 0, 0, None, None,
                               ctypes.cast(None, beam.FORWARD_FN), None, None, None,
                               None) == INVALID


# ------------------------------------------------------------- Python binding


class FakeLibrary:
    """Calls forward once, as g4s_beam_generate would, and keeps its arguments."""

    def g4s_beam_generate(self, *args):
        self.args = args
        self.pages = args[7]._obj.pages if args[7] is not None else None
        self.status = args[8](None, ctypes.pointer(beam.BeamStep()))
        return native.G4S_OK if self.status == 0 else -9

    def g4s_beam_last_error(self, h):
        return b"the forward callback failed"


@pytest.fixture
def fake(monkeypatch):
    library = FakeLibrary()
    monkeypatch.setattr(beam, "load", lambda: library)
    library.search = beam.BeamSearch.__new__(beam.BeamSearch)
    library.search.h, library.search.vocab = ctypes.c_void_p(), 100
    library.destroyed = []
    library.g4s_pages_destroy = lambda h: library.destroyed.append(h.value)
    return library


@pytest.mark.parametrize("error", [ValueError, KeyboardInterrupt, SystemExit])
def test_an_exception_of_the_forward_ends_the_search(fake, error):
    def forward(step):
        raise error("stop")
    with pytest.raises(error):
        fake.search.Generate(1 << 20, 1, 1, 1, forward)
    assert fake.status != 0


def test_records_keep_what_they_name(fake):
    """A page cache, a state's arrays and a pool that only a record names live as
    long as it; a cache that was closed is not passed on."""
    class Array(hip.Buffer):
        def __init__(self, addr):
            self.nbytes, self.ptr = 8, ctypes.c_void_p(addr)

        def free(self):
            pass

    def cache():
        c = beam.PageCache.__new__(beam.PageCache)
        c.h = ctypes.c_void_p(77)
        return c
    arrays = [Array(i + 1) for i in range(8)]
    alive = [weakref.ref(a) for a in arrays]
    record = beam.BeamCache(cache(), [beam.PageState(*arrays[:3]), beam.PageState(*arrays[3:6])],
                            arrays[6])
    states = beam.BeamStates(arrays[7], 1, 0, 8, 8)
    del arrays
    gc.collect()
    assert fake.destroyed == [] and all(r() is not None for r in alive)
    fake.search.Generate(1 << 20, 1, 1, 1, lambda step: True, states=states, cache=record)
    assert fake.pages == 77 and [record.states[i].refs for i in range(2)] == [3, 6]
    record.cache.close()
    assert fake.destroyed == [77]
    fake.search.Generate(1 << 20, 1, 1, 1, lambda step: True, cache=record)
    assert fake.pages is None
    del record, states, fake.args
    gc.collect()
    assert all(r() is None for r in alive) and fake.destroyed == [77]


# ------------------------------------------------------------- Pascal unit


def _c(path):
    s = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    return re.sub(r"//[^\n]*", "", s)


def _pascal():
    s = re.sub(r"\{.*?\}", "", open(UNIT).read(), flags=re.S)
    return re.sub(r"//[^\n]*", "", s)


PAS2C = {"Integer": "int32_t", "Int64": "int64_t", "Single": "float", "Pointer": "void*",
         "PAnsiChar": "char*", "PInteger": "int32_t*", "PSingle": "float*",
         "PG4SBeam": "g4s_beam*", "PPG4SBeam": "g4s_beam**", "PG4SPages": "g4s_pages*",
         "PPG4SPages": "g4s_pages**", "PG4SPageGeometry": "g4s_page_geometry*",
         "PG4SPageState": "g4s_page_state*", "TG4SPageState": "g4s_page_state",
         "PG4SBeamConfig": "g4s_beam_config*", "PG4SBeamStates": "g4s_beam_states*",
         "PG4SBeamCache": "g4s_beam_cache*", "TG4SBeamForwardFn": "g4s_beam_forward_fn"}


def _canon(t):
    t = re.sub(r"\s*\*\s*", "*", t.replace("const", " "))
    t = re.sub(r"\s+", " ", t).strip()
    return "int32_t" if t == "int" else t


def test_pascal_externals_match_the_header():
    want = {}
    for ret, name, args in re.findall(r"([A-Za-z_][\w \*]*?)\s*\b(g4s_\w+)\s*\(([^)]*)\)\s*;",
                                      _c(HEADER)):
        want[name] = (_canon(ret), [_canon(re.match(r"(.*?)\w+$", a.strip()).group(1))
                                    for a in args.split(",")])
    got = {}
    for kind, name, args, ret in re.findall(
            r"\b(function|procedure)\s+(g4s_\w+)\s*\((.*?)\)\s*(?::\s*(\w+))?\s*;"
            r"\s*cdecl\s*;\s*external\s+CG4SLib\s*;", _pascal(), flags=re.S):
        params = []
        for group in [g.strip() for g in args.split(";") if g.strip()]:
            assert not re.match(r"(const|var|out)\b", group), (name, group)
            names, typ = group.split(":")
            params += [PAS2C[typ.strip()]] * len(names.split(","))
        got[name] = (PAS2C[ret], params)
    assert got == want
    assert set(want) < set(native.EXPORTS)


@pytest.mark.parametrize("c_name, p_name", [
    ("g4s_page_geometry", "TG4SPageGeometry"), ("g4s_page_state", "TG4SPageState"),
    ("g4s_beam_config", "TG4SBeamConfig"), ("g4s_beam_states", "TG4SBeamStates"),
    ("g4s_beam_cache", "TG4SBeamCache"), ("g4s_beam_step", "TG4SBeamStep")])
def test_pascal_records_match_the_structs(c_name, p_name):
    body = re.search(r"typedef struct %s \{(.*?)\}" % c_name, _c(HEADER), re.S).group(1)
    want = [(_canon(t) + (f"[{n}]" if n else ""), f.replace("_", "").lower()) for t, f, n in
            re.findall(r"([\w \*]+?)\s*\b(\w+)\s*(?:\[(\w+)\])?\s*;", body)]
    body = re.search(r"\b%s\s*=\s*record(.*?)\bend;" % p_name, _pascal(), re.S).group(1)
    got = []
    for line in [x.strip() for x in body.split(";") if x.strip()]:
        f, t = [x.strip() for x in line.split(":", 1)]
        arr = re.match(r"array\s*\[\s*0\s*\.\.\s*(\d+)\s*\]\s*of\s+(\w+)", t)
        got.append((PAS2C[arr.group(2)] + f"[{int(arr.group(1)) + 1}]" if arr else PAS2C[t],
                    f.lower()))
    assert got == want


def test_pascal_and_python_constants_match_the_header():
    want = {n: int(v) for n, v in re.findall(r"#define\s+(G4S_\w+)\s+(\d+)", _c(HEADER))}
    got = {n: int(v) for n, v in re.findall(r"\b(G4S_\w+)\s*=\s*(\d+)\s*;", _pascal())}
    assert got == want
    assert (beam.MAX_BEAMS, beam.MAX_ROWS, beam.PAGES_MAX_ROWS, beam.PAGES_MAX_PAGES) == tuple(
        want[n] for n in ("G4S_BEAM_MAX_BEAMS", "G4S_BEAM_MAX_ROWS", "G4S_PAGES_MAX_ROWS",
                          "G4S_PAGES_MAX_PAGES"))


def test_pascal_search_names_the_row_stride():
    """Rows of a vocabulary that does not fill whole 16-byte vectors are padded, and
    a search of more than one row is refused without their stride."""
    s = _pascal()
    intf, impl = s[:s.index("implementation")], s[s.index("implementation"):]
    at = intf.index("TGpuBeamSearch = class")
    method = re.search(r"function Generate\((.*?)\): Boolean", intf[at:], re.S).group(1)
    assert re.search(r"const ARowStride: Int64 = 0$", method.strip())
    body = impl[impl.index("function TGpuBeamSearch.Generate"):]
    call = re.search(r"g4s_beam_generate\((.*?)\)", body, re.S).group(1)
    external = re.search(r"function g4s_beam_generate\((.*?)\)", intf, re.S).group(1)
    names = [n.strip() for g in external.split(";") for n in g.split(":")[0].split(",")]
    stride = [a.strip() for a in call.split(",")][names.index("ARowStride")]
    before = body[:body.index("g4s_beam_generate")]
    assert re.search(r"\b%s := ARowStride;" % stride, before)
    assert re.search(r"if %s = 0 then\s+%s := FVocab;" % (stride, stride), before)


# ---------------------------------------------------------- the pages' rules


@pytest.fixture(scope="module")
def host():
    if not os.path.exists(HOST):
        subprocess.run(["make", "-s", "-C", os.path.join(ROOT, "tests", "native")], check=True)
    L = ctypes.CDLL(HOST)
    L.t_row_step.argtypes = [ctypes.c_int32] * 6 + [ctypes.c_void_p]
    L.t_geometry_ok.argtypes = [ctypes.c_void_p]
    L.t_page_offset.restype = ctypes.c_int64
    L.t_page_offset.argtypes = [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_uint32,
                                ctypes.c_uint32, ctypes.c_int32]

    def step(*a):
        out = np.zeros(5, np.int64)
        L.t_row_step(*a, out.ctypes.data_as(ctypes.c_void_p))
        return tuple(int(x) for x in out)
    L.step = step
    return L


BAD = (0, 0, 0, 0, 1)
MAX = (1 << 31) - 1


@pytest.mark.parametrize("args, want", [
    # parent, from_rows, length, grow, page_tokens, max_slots -> length, kept, fresh, tail, bad
    ((0, 1, 0, 0, 16, 4), (0, 0, 0, 0, 0)), ((0, 1, 0, 1, 16, 4), (1, 0, 1, 0, 0)),
    ((0, 1, 5, 0, 16, 4), (5, 1, 0, 0, 0)), ((0, 1, 5, 1, 16, 4), (6, 1, 0, 5, 0)),
    ((0, 1, 16, 1, 16, 4), (17, 1, 1, 0, 0)), ((0, 1, 15, 18, 16, 4), (33, 1, 2, 15, 0)),
    ((0, 1, 33, -1, 16, 4), (32, 2, 0, 0, 0)), ((0, 1, 33, -40, 16, 4), (0, 0, 0, 0, 0)),
    ((-1, 1, 9, 20, 16, 4), (20, 0, 2, 0, 0)), ((-1, 1, 9, -3, 16, 4), (0, 0, 0, 0, 0)),
    ((0, 1, 64, 0, 16, 4), (64, 4, 0, 0, 0)), ((0, 1, 64, 1, 16, 4), BAD),
    ((0, 1, 65, 0, 16, 4), BAD), ((0, 1, -1, 0, 16, 4), BAD), ((1, 1, 0, 0, 16, 4), BAD),
    ((-2, 1, 0, 0, 16, 4), BAD), ((0, 1, MAX, MAX, 65536, 32767), BAD),
    ((0, 1, 7, MAX, 1, MAX), BAD), ((0, 1, MAX, -MAX - 1, 1, MAX), (0, 0, 0, 0, 0)),
    ((0, 1, 3, 2, 1, 8), (5, 3, 2, 0, 0))])
def test_row_step(host, args, want):
    assert host.step(*args) == want


@pytest.mark.parametrize("tokens, page_tokens, want", [
    (0, 1, 0), (1, 16, 1), (16, 16, 1), (17, 16, 2), (MAX, 1, MAX), (MAX, 65536, 32768),
    (3000 * 715827, 3000, 715827), (3000 * 715827 - 2999, 3000, 715827)])
def test_used_slots(host, tokens, page_tokens, want):
    host.t_used_slots.argtypes = [ctypes.c_int64, ctypes.c_int32]
    assert host.t_used_slots(tokens, page_tokens) == want


def test_offsets_pass_32_bits(host):
    g = beam.PageGeometry(32, 1 << 20, 1, 1, 4, 2, 4096, (1 << 20) * 262144, 262144)
    assert host.t_geometry_ok(ctypes.byref(g)) == 1
    # the last 16 bytes of 7 tokens of the second part of the last page of plane 3
    per = 7 * 4096 // 16
    got = host.t_page_offset(ctypes.byref(g), 3, (1 << 20) - 1, 2 * per - 1, per, 16)
    assert got == 3 * (1 << 38) + ((1 << 20) - 1) * 262144 + 32 * 4096 + 7 * 4096 - 16
