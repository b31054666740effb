"""ctypes binding of include/gemma4_beam.h: beam search over device-resident
logits, and the cache pages its beams live in.

BeamSearch wraps a g4s_beam handle (select, reorder, Generate), PageCache a
g4s_pages handle (advance, compact, copy).  Device arrays are hip.Buffers or
addresses, as in native.py; a failing call raises native.SamplerError.
"""
import ctypes

import numpy as np

from . import native
from .native import DTYPE_F32, G4S_OK, SamplerError, _ptr

MAX_BEAMS = 64
MAX_ROWS = 65535
PAGES_MAX_ROWS = 2048
PAGES_MAX_PAGES = 1048576

# words of the status of PageCache.advance and compact
STATUS_CODE, STATUS_FREE, STATUS_TAKEN, STATUS_COPIED = range(4)


class PageGeometry(ctypes.Structure):
    """g4s_page_geometry"""
    _fields_ = [("page_tokens", ctypes.c_int32), ("n_pages", ctypes.c_int32),
                ("max_rows", ctypes.c_int32), ("max_slots", ctypes.c_int32),
                ("planes", ctypes.c_int32), ("parts", ctypes.c_int32),
                ("token_bytes", ctypes.c_int64), ("plane_stride", ctypes.c_int64),
                ("page_stride", ctypes.c_int64)]


class PageState(ctypes.Structure):
    """g4s_page_state: device arrays of a state (table, lengths, refs), which live as
    long as the record."""
    _fields_ = [("table", ctypes.c_void_p), ("lengths", ctypes.c_void_p),
                ("refs", ctypes.c_void_p)]

    def __init__(self, table=None, lengths=None, refs=None):
        super().__init__(_ptr(table), _ptr(lengths), _ptr(refs))
        self._owners = (table, lengths, refs)


class BeamConfig(ctypes.Structure):
    """g4s_beam_config"""
    _fields_ = [("beams", ctypes.c_int32), ("max_tokens", ctypes.c_int32),
                ("n_best", ctypes.c_int32), ("early_stop", ctypes.c_int32),
                ("length_penalty", ctypes.c_float)]


class BeamStates(ctypes.Structure):
    """g4s_beam_states"""
    _fields_ = [("d_state", ctypes.c_void_p), ("planes", ctypes.c_int64),
                ("plane_stride", ctypes.c_int64), ("row_stride", ctypes.c_int64),
                ("row_bytes", ctypes.c_int64)]

    def __init__(self, d_state, planes, plane_stride, row_stride, row_bytes):
        super().__init__(_ptr(d_state), int(planes), int(plane_stride), int(row_stride),
                         int(row_bytes))
        self._owners = (d_state,)


class BeamCache(ctypes.Structure):
    """g4s_beam_cache; the PageCache, its states and the pool live as long as
    the record."""
    _fields_ = [("pages", ctypes.c_void_p), ("states", PageState * 2),
                ("d_pool", ctypes.c_void_p)]

    def __init__(self, cache, states, d_pool):
        states = tuple(states)
        super().__init__(cache.h, (PageState * 2)(*states), _ptr(d_pool))
        self.cache = cache
        self._owners = (states, d_pool)


class BeamStep(ctypes.Structure):
    """g4s_beam_step"""
    _fields_ = [("tokens", ctypes.POINTER(ctypes.c_int32)),
                ("parents", ctypes.POINTER(ctypes.c_int32)), ("d_tokens", ctypes.c_void_p),
                ("d_parents", ctypes.c_void_p), ("rows", ctypes.c_int32),
                ("state", ctypes.c_int32)]

    def Tokens(self):
        return np.ctypeslib.as_array(self.tokens, (self.rows,)).copy()

    def Parents(self):
        return np.ctypeslib.as_array(self.parents, (self.rows,)).copy()


FORWARD_FN = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(BeamStep))

_bound = False


def load():
    """The library, with the argument types of gemma4_beam.h."""
    global _bound
    L = native.load()
    if not _bound:
        vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
        L.g4s_beam_create.argtypes = [ctypes.POINTER(vp), i32, i32, i32, f32, vp]
        L.g4s_beam_destroy.argtypes = [vp]
        L.g4s_beam_last_error.restype = ctypes.c_char_p
        L.g4s_beam_last_error.argtypes = [vp]
        L.g4s_beam_select.argtypes = [vp, vp, i32, i64, i32, i32, vp, i32, vp, vp, vp, vp]
        L.g4s_beam_reorder.argtypes = [vp, vp, vp, i64, i64, i32, i32, i64, i64, vp]
        L.g4s_pages_create.argtypes = [ctypes.POINTER(vp), vp, vp]
        L.g4s_pages_destroy.argtypes = [vp]
        L.g4s_pages_last_error.restype = ctypes.c_char_p
        L.g4s_pages_last_error.argtypes = [vp]
        L.g4s_pages_advance.argtypes = [vp, vp, i32, vp, i32, vp, vp, vp, vp]
        L.g4s_pages_compact.argtypes = [vp, vp, vp, i32, vp, vp]
        L.g4s_pages_copy.argtypes = [vp, vp, vp, i32, vp, vp, vp]
        L.g4s_beam_generate.argtypes = [vp, i32, vp, vp, i32, i64, vp, vp, FORWARD_FN, vp, vp, vp,
                                        vp]
        _bound = True
    return L


def _stream(stream):
    return stream.handle if stream is not None else None


def _ref(x):
    return ctypes.byref(x) if x is not None else None


class BeamSearch:
    """One g4s_beam handle."""

    def __init__(self, vocab, max_batch=1, max_beams=4, softcap=30.0, stream=None):
        self.h = None
        L = load()
        h = ctypes.c_void_p()
        rc = L.g4s_beam_create(ctypes.byref(h), int(vocab), int(max_batch), int(max_beams),
                               float(softcap), _stream(stream))
        if rc != G4S_OK:
            raise SamplerError(rc, L.g4s_beam_last_error(None).decode())
        self.h = h
        self.vocab, self.max_batch, self.max_beams = int(vocab), int(max_batch), int(max_beams)

    def last_error(self):
        return load().g4s_beam_last_error(self.h).decode()

    def _check(self, rc):
        if rc != G4S_OK:
            raise SamplerError(rc, self.last_error())

    def select(self, d_logits, batch, beams, d_scores, n_select, d_parents, d_tokens, d_out,
               d_lse=None, dtype=DTYPE_F32, row_stride=None):
        """g4s_beam_select (stream-ordered)"""
        stride = self.vocab if row_stride is None else int(row_stride)
        self._check(load().g4s_beam_select(
            self.h, _ptr(d_logits), int(dtype), stride, int(batch), int(beams), _ptr(d_scores),
            int(n_select), _ptr(d_parents), _ptr(d_tokens), _ptr(d_out), _ptr(d_lse)))

    def reorder(self, d_src, d_dst, planes, plane_stride, batch, beams, row_stride, row_bytes,
                d_parents):
        """g4s_beam_reorder (stream-ordered); d_dst = d_src moves in place"""
        self._check(load().g4s_beam_reorder(
            self.h, _ptr(d_src), _ptr(d_dst), int(planes), int(plane_stride), int(batch),
            int(beams), int(row_stride), int(row_bytes), _ptr(d_parents)))

    def Generate(self, d_logits, batch, beams, max_tokens, forward, n_best=1, early_stop=False,
                 length_penalty=1.0, states=None, cache=None, dtype=DTYPE_F32, row_stride=None):
        """g4s_beam_generate.  forward(BeamStep) -> bool (True = ok).  Returns,
        per sequence, a list of (tokens, score), the best first."""
        cfg = BeamConfig(int(beams), int(max_tokens), int(n_best), int(early_stop),
                         float(length_penalty))
        room = max(int(max_tokens), 0)
        count = max(int(batch) * int(n_best), 1)
        toks = np.zeros(max(count * room, 1), np.int32)
        lens = np.zeros(count, np.int32)
        scores = np.zeros(count, np.float32)
        errors = []

        def fwd(_, step):
            try:
                return 0 if forward(step.contents) else 1
            # an exception that left the callback would be printed and dropped, and the
            # search would go on over stale logits: an interrupt ends it too
            except BaseException as e:  # noqa: BLE001 -- raised again after the loop
                errors.append(e)
                return 1

        if cache is not None:
            cache.pages = cache.cache.h  # NULL, and so refused, once it is closed
        stride = self.vocab if row_stride is None else int(row_stride)
        rc = load().g4s_beam_generate(
            self.h, int(batch), ctypes.byref(cfg), _ptr(d_logits), int(dtype), stride,
            _ref(states), _ref(cache), FORWARD_FN(fwd), None,
            toks.ctypes.data_as(ctypes.c_void_p), lens.ctypes.data_as(ctypes.c_void_p),
            scores.ctypes.data_as(ctypes.c_void_p))
        if errors:
            raise errors[0]
        self._check(rc)
        out = []
        for b in range(batch):
            found = []
            for k in range(b * n_best, (b + 1) * n_best):
                if lens[k] > 0:
                    found.append((toks[k * room:k * room + lens[k]].copy(), float(scores[k])))
            out.append(found)
        return out

    def close(self):
        if self.h is not None and self.h.value:
            load().g4s_beam_destroy(self.h)
        self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PageCache:
    """One g4s_pages handle.  Planes lie outside the pages unless strides
    (bytes) say otherwise."""

    def __init__(self, page_tokens, n_pages, max_rows, max_slots, planes=0, parts=1,
                 token_bytes=0, plane_stride=None, page_stride=None, stream=None):
        self.h = None
        L = load()
        page = int(parts) * int(page_tokens) * int(token_bytes)
        page_stride = page if page_stride is None else int(page_stride)
        plane_stride = page_stride * int(n_pages) if plane_stride is None else int(plane_stride)
        self.geometry = PageGeometry(int(page_tokens), int(n_pages), int(max_rows),
                                     int(max_slots), int(planes), int(parts), int(token_bytes),
                                     plane_stride, page_stride)
        h = ctypes.c_void_p()
        rc = L.g4s_pages_create(ctypes.byref(h), ctypes.byref(self.geometry), _stream(stream))
        if rc != G4S_OK:
            raise SamplerError(rc, L.g4s_pages_last_error(None).decode())
        self.h = h

    def last_error(self):
        return load().g4s_pages_last_error(self.h).decode()

    def _check(self, rc):
        if rc != G4S_OK:
            raise SamplerError(rc, self.last_error())

    def advance(self, src, src_rows, dst, rows, d_parents, d_grow, d_pool, d_status):
        """g4s_pages_advance (stream-ordered) from PageState src to dst"""
        self._check(load().g4s_pages_advance(self.h, _ref(src), int(src_rows), _ref(dst),
                                             int(rows), _ptr(d_parents), _ptr(d_grow),
                                             _ptr(d_pool), _ptr(d_status)))

    def compact(self, src, dst, rows, d_pool, d_status):
        """g4s_pages_compact (stream-ordered) from PageState src to dst"""
        self._check(load().g4s_pages_compact(self.h, _ref(src), _ref(dst), int(rows),
                                             _ptr(d_pool), _ptr(d_status)))

    def copy(self, d_src_pool, d_dst_pool, n, d_src_pages, d_dst_pages, d_tokens=None):
        """g4s_pages_copy (stream-ordered)"""
        self._check(load().g4s_pages_copy(self.h, _ptr(d_src_pool), _ptr(d_dst_pool), int(n),
                                          _ptr(d_src_pages), _ptr(d_dst_pages), _ptr(d_tokens)))

    def close(self):
        if self.h is not None and self.h.value:
            load().g4s_pages_destroy(self.h)
        self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
