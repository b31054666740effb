"""ctypes binding of include/gemma4_cache.h: keys and values in 8 bits in the
pages of a cache, the append with its rotation, and the attention over them.

KvCache wraps a g4s_cache handle (append, attend) on the geometry of a
beam.PageCache.  Device arrays are hip.Buffers or addresses, as in native.py;
a failing call raises native.SamplerError.
"""
import ctypes

from . import native
from .beam import PageCache, PageGeometry, PageState, _stream  # noqa: F401
from .native import DTYPE_BF16, DTYPE_F32, G4S_OK, SamplerError, _ptr  # noqa: F401

MAX_HEADS = 512
MAX_KV_HEADS = 64
MAX_GROUP = 64
MAX_HEAD_DIM = 512
MAX_SCALE_TOKENS = 256
MAX_TOKENS = 1048576
MAX_CONTEXT = 1073741824

ROTARY = {"halves": 0, "neighbours": 1}


class CacheConfig(ctypes.Structure):
    """g4s_cache_config"""
    _fields_ = [("heads", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("scale_tokens", ctypes.c_int32),
                ("rotary_dims", ctypes.c_int32), ("rotary_pairs", ctypes.c_int32)]


class View(ctypes.Structure):
    """g4s_cache_view: data (which lives as long as the record) and its strides in elements."""
    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64)]

    def __init__(self, data, token_stride, head_stride):
        super().__init__(_ptr(data), int(token_stride), int(head_stride))
        self._owners = (data,)
        self._at = ctypes.addressof(self)


def geometry(page_tokens, n_pages, max_rows, max_slots, kv_heads, head_dim, planes=2,
             plane_stride=None, page_stride=None):
    """The page geometry of an 8-bit cache: a part per kv head, a scale behind
    each token's codes.  Its fields are what a PageCache of these pages takes."""
    token = int(head_dim) + 4
    page = int(kv_heads) * int(page_tokens) * token
    page_stride = page if page_stride is None else int(page_stride)
    plane_stride = page_stride * int(n_pages) if plane_stride is None else int(plane_stride)
    return PageGeometry(int(page_tokens), int(n_pages), int(max_rows), int(max_slots),
                        int(planes), int(kv_heads), token, plane_stride, page_stride)


def _address(x):
    """What a pointer argument takes, without a new object for most: a step's calls are as
    long on the host as on the GPU."""
    if x is None or type(x) is int:
        return x
    if type(x) is View:
        return x._at
    return ctypes.byref(x) if isinstance(x, ctypes.Structure) else _ptr(x)


_bound = False


def load():
    """The library, with the argument types of gemma4_cache.h."""
    global _bound
    L = native.load()
    if not _bound:
        vp, i32, f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_float
        L.g4s_cache_create.argtypes = [ctypes.POINTER(vp), vp, vp, vp]
        L.g4s_cache_destroy.argtypes = [vp]
        L.g4s_cache_last_error.restype = ctypes.c_char_p
        L.g4s_cache_last_error.argtypes = [vp]
        L.g4s_cache_append.argtypes = [vp, vp, i32, vp, i32, i32, vp, vp, vp, vp, vp, vp, vp, i32,
                                       i32]
        L.g4s_cache_attend.argtypes = [vp, vp, i32, vp, i32, i32, vp, vp, i32, i32, f32, i32, vp,
                                       vp]
        _bound = True
    return L


class KvCache:
    """One g4s_cache handle."""

    def __init__(self, geometry, heads, kv_heads, head_dim, scale_tokens=1, rotary_dims=None,
                 rotary_pairs="halves", stream=None):
        self.h = self._at = None
        L = load()
        rotary = int(head_dim) if rotary_dims is None else int(rotary_dims)
        self.geometry = geometry
        self.config = CacheConfig(int(heads), int(kv_heads), int(head_dim), int(scale_tokens),
                                  rotary, ROTARY.get(rotary_pairs, rotary_pairs))
        h = ctypes.c_void_p()
        rc = L.g4s_cache_create(ctypes.byref(h), ctypes.byref(self.geometry),
                                ctypes.byref(self.config), _stream(stream))
        if rc != G4S_OK:
            raise SamplerError(rc, L.g4s_cache_last_error(None).decode())
        self.h = h
        self._at, self._append, self._attend = h.value, L.g4s_cache_append, L.g4s_cache_attend

    def last_error(self):
        return load().g4s_cache_last_error(self.h).decode()

    def _check(self, rc):
        if rc != G4S_OK:
            raise SamplerError(rc, self.last_error())

    def append(self, state, rows, tokens, dtype, d_pool=None, k_plane=0, v_plane=1, q=None, k=None,
               v=None, q_out=None, d_starts=None, d_positions=None, d_freqs=None):
        """g4s_cache_append (stream-ordered); q, k, v and q_out are Views"""
        rc = self._append(self._at, _address(state), int(rows), _address(d_starts), int(tokens),
                          int(dtype), _address(q), _address(k), _address(v), _address(q_out),
                          _address(d_positions), _address(d_freqs), _address(d_pool),
                          int(k_plane), int(v_plane))
        if rc:
            self._check(rc)

    def attend(self, state, rows, tokens, dtype, d_pool, k_plane, v_plane, q, out, scale, window=0,
               d_starts=None, d_lse=None):
        """g4s_cache_attend (stream-ordered); q and out are Views"""
        rc = self._attend(self._at, _address(state), int(rows), _address(d_starts), int(tokens),
                          int(dtype), _address(q), _address(d_pool), int(k_plane), int(v_plane),
                          float(scale), int(window), _address(out), _address(d_lse))
        if rc:
            self._check(rc)

    def close(self):
        if self.h is not None and self.h.value:
            load().g4s_cache_destroy(self.h)
        self.h = self._at = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
