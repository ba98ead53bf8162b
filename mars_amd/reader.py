"""Reading retrieved memories: a paged cache of their tokens and the attention over it.

    r     = Reader(q_heads=32, kv_heads=8, head_dim=128, dtype="bfloat16", page_size=64,
                   rope_dim=128, rope_theta=1e6, rope_sections=(16, 24, 24))
    cache = PagedCache(k_pages, v_pages, times, episodes)
    r.plan(new_lens, cached_lens, block_table, free_pages, free_count, q_start=..., ...)   # once a step
    r.store(cache, q, k, v, positions, slots, q_out=q, times=..., episodes=...)            # once a layer
    r.attend(cache, q, out, q_start, kv_lens, block_table, decay=..., q_times=..., ...)
    r.release(done, next_lens, block_table, free_pages, free_count)                        # ended requests

The calls mirror mars_kv_* of include/mars_amd.h, which defines their results. They run on
`stream` (the integer of a hipStream_t; 0 is the null stream) and return without waiting.
Tensors are anything that holds device memory and has data_ptr(), shape, stride() and
dtype: a DeviceArray of this module, or a tensor of a framework that shares this library's HIP
runtime (imported before it). One that also has get_device() has to be on the reader's GPU, or pinned. Outputs
are the caller's.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np

from . import DeviceBuffer, _lib
from ._lib import check, lib

__all__ = ["Reader", "PagedCache", "DeviceArray"]

_DTYPES = {"float16": 0, "bfloat16": 1}
_ITEM = {"float16": 2, "bfloat16": 2, "float32": 4, "int32": 4, "int64": 8}
_NAMES: dict = {}


def _current_device() -> int:
    d = C.c_int32()
    check(lib.mars_device_current(C.byref(d)), "mars_device_current")
    return d.value


def _dtype(x) -> str:
    """The name of x's element type, without a framework's prefix."""
    d = x.dtype
    name = _NAMES.get(d)
    if name is None:
        name = _NAMES[d] = str(d).rsplit(".", 1)[-1]
    return name


class DeviceArray:
    """A device array of this library's own memory: dense, row-major."""

    def __init__(self, shape: Sequence[int], dtype: str, buffer: Optional[DeviceBuffer] = None):
        self.shape = tuple(int(s) for s in shape)
        self.dtype = dtype
        self.size = int(np.prod(self.shape, dtype=np.int64))
        self.buffer = buffer or DeviceBuffer(max(self.size, 1) * _ITEM[dtype])
        self._device = _current_device()
        strides, n = [], 1
        for s in reversed(self.shape):
            strides.append(n)
            n *= s
        self._strides = tuple(reversed(strides))

    @classmethod
    def from_numpy(cls, a: np.ndarray, dtype: Optional[str] = None) -> "DeviceArray":
        """dtype "bfloat16": `a` holds the bits as uint16."""
        a = np.ascontiguousarray(a)
        return cls(a.shape, dtype or str(a.dtype), DeviceBuffer.from_array(a) if a.size else None)

    def numpy(self) -> np.ndarray:
        """The contents once all work is done; bfloat16 as uint16 bits."""
        check(lib.mars_device_synchronize(), "mars_device_synchronize")
        dt = np.uint16 if self.dtype == "bfloat16" else np.dtype(self.dtype)
        return self.buffer.to_array(dt, self.size).reshape(self.shape)

    def data_ptr(self) -> int:
        return self.buffer.ptr

    def stride(self, i: int) -> int:
        return self._strides[i]

    def is_contiguous(self) -> bool:
        return True

    def get_device(self) -> int:
        return self._device


def _dense(x) -> bool:
    try:
        return x.is_contiguous()
    except AttributeError:
        n = 1
        for i in range(len(x.shape) - 1, -1, -1):
            if x.shape[i] != 1 and x.stride(i) != n:
                return False
            n *= x.shape[i]
        return True


def _device(x) -> Optional[int]:
    """The GPU that x is on, negative for host memory, None if x does not say."""
    try:
        return x.get_device()
    except AttributeError:
        return None


def _place(x, name: str, at: Optional[int], device: Optional[int]) -> None:
    """Refuses memory that a kernel on GPU `device` (None: any) must not be given."""
    if at is None or at == device or (device is None and at >= 0):
        return
    if at >= 0:
        raise ValueError(f"{name}: on GPU {at}, expected GPU {device}")
    if not (hasattr(x, "is_pinned") and x.is_pinned()):
        raise ValueError(f"{name}: in host memory")


def _arg(x, name: str, dtype: str, shape, device: Optional[int]) -> Optional[int]:
    """The address of a dense array of the given type and shape (None: any length) on that GPU."""
    if x is None:
        return None
    if _dtype(x) != dtype:
        raise ValueError(f"{name}: {_dtype(x)}, expected {dtype}")
    if shape is not None and x.shape != shape:
        raise ValueError(f"{name}: shape {tuple(x.shape)}, expected {shape}")
    if not _dense(x):
        raise ValueError(f"{name}: not dense")
    _place(x, name, _device(x), device)
    return x.data_ptr()


def _args(device: Optional[int], *specs) -> list:
    """_arg of every (array, name, type, shape), with one short check of an array that is as it should be."""
    known = _NAMES.get
    try:
        return [None if x is None else x.data_ptr() if known(x.dtype) == dtype and (shape is None or x.shape == shape) and x.is_contiguous()
                and x.get_device() == device else _arg(x, name, dtype, shape, device) for x, name, dtype, shape in specs]
    except AttributeError:                                  # one that does not say where it is, or whether it is dense
        return [_arg(*s, device) for s in specs]


def _rows(x, name: str, dtype: str, device: Optional[int], tokens: Optional[int], heads: int, dim: int):
    """Address and token stride of a (tokens, heads, dim) array with dense heads on that GPU."""
    if _NAMES.get(x.dtype) != dtype and _dtype(x) != dtype:
        raise ValueError(f"{name}: {_dtype(x)}, expected {dtype}")
    s = x.shape
    if len(s) != 3 or s[1] != heads or s[2] != dim or (tokens is not None and s[0] != tokens):
        raise ValueError(f"{name}: shape {tuple(s)}, expected ({'tokens' if tokens is None else tokens}, {heads}, {dim})")
    if x.stride(2) != 1 or (heads > 1 and x.stride(1) != dim):
        raise ValueError(f"{name}: a token's heads are not dense")
    try:
        at = x.get_device()
    except AttributeError:
        at = None
    if at != device:
        _place(x, name, at, device)
    return x.data_ptr(), (x.stride(0) if s[0] > 1 else heads * dim)


class PagedCache:
    """The pages of one layer (mars_kv_cache): k_pages (pages, kv_heads, page_size, head_dim), v_pages (pages,
    kv_heads, head_dim, page_size), each page dense; times (float32) and episodes (int32) one per slot."""

    def __init__(self, k_pages, v_pages, times=None, episodes=None):
        if len(k_pages.shape) != 4 or len(v_pages.shape) != 4:
            raise ValueError("k_pages, v_pages: 4 axes expected")
        n, h, p, d = (int(s) for s in k_pages.shape)
        if tuple(v_pages.shape) != (n, h, d, p):
            raise ValueError(f"v_pages: shape {tuple(v_pages.shape)}, expected {(n, h, d, p)}")
        if _dtype(k_pages) != _dtype(v_pages) or _dtype(k_pages) not in _DTYPES:
            raise ValueError(f"k_pages {_dtype(k_pages)}, v_pages {_dtype(v_pages)}")
        for name, x, inner in (("k_pages", k_pages, (p * d, d, 1)), ("v_pages", v_pages, (p * d, p, 1))):
            if any(x.shape[i + 1] != 1 and x.stride(i + 1) != inner[i] for i in range(3)):
                raise ValueError(f"{name}: a page is not dense")
        self.k_pages, self.v_pages, self.times, self.episodes = k_pages, v_pages, times, episodes
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = n, h, p, d
        self.dtype = _dtype(k_pages)
        self.geometry = (h, p, d, self.dtype)
        # the GPU of the arrays that are on one (pinned host memory is on none)
        self.device = next((at for at in map(_device, (k_pages, v_pages, times, episodes)) if at is not None and at >= 0), None)
        for name, x in (("k_pages", k_pages), ("v_pages", v_pages)):
            _place(x, name, _device(x), self.device)
        strides = [x.stride(0) if n > 1 else 0 for x in (k_pages, v_pages)]
        for name, x, want in (("times", times, "float32"), ("episodes", episodes, "int32")):
            if x is not None and int(np.prod(tuple(x.shape), dtype=np.int64)) != n * p:
                raise ValueError(f"{name}: shape {tuple(x.shape)}, expected one per slot, {n * p}")
            _arg(x, name, want, None, self.device)
        self.c = _lib.KvCacheC(k_pages.data_ptr(), v_pages.data_ptr(), times.data_ptr() if times is not None else None,
                               episodes.data_ptr() if episodes is not None else None, strides[0], strides[1], n, 0)
        self.ref = C.byref(self.c)


class Reader:
    """Geometry and scratch of the reading path (mars_reader), on the current GPU. One reader serves one stream at a time."""

    device: Optional[int] = None

    def __init__(self, q_heads: int = 12, kv_heads: Optional[int] = None, head_dim: int = 64, dtype: str = "float16",
                 page_size: int = 64, rope_dim: int = 0, rope_theta: float = 1e4,
                 rope_sections: Optional[Sequence[int]] = None, rope_adjacent: bool = False):
        if dtype not in _DTYPES:
            raise ValueError(f"dtype {dtype}: float16 or bfloat16")
        sections = tuple(rope_sections) if rope_sections is not None else (rope_dim // 2,)
        if len(sections) > 3:
            raise ValueError(f"{len(sections)} rope sections: at most 3 axes")
        self.q_heads, self.kv_heads = int(q_heads), int(q_heads if kv_heads is None else kv_heads)
        self.head_dim, self.dtype, self.page_size = int(head_dim), dtype, int(page_size)
        self.rope_dim, self.rope_axes = int(rope_dim), len(sections)
        self.geometry = (self.kv_heads, self.page_size, self.head_dim, self.dtype)
        desc = _lib.ReaderDescC(self.q_heads, self.kv_heads, self.head_dim, _DTYPES[dtype], self.page_size, self.rope_dim,
                                self.rope_axes, int(bool(rope_adjacent)),
                                (C.c_int32 * 3)(*(list(sections) + [0] * (3 - len(sections)))), 0, float(rope_theta))
        self.handle = C.c_void_p()
        check(lib.mars_reader_create(C.byref(desc), C.byref(self.handle)), "mars_reader_create")
        self.device = _current_device()

    def close(self) -> None:
        if self.handle:
            check(lib.mars_reader_destroy(self.handle), "mars_reader_destroy")
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _cache(self, cache: PagedCache):
        if cache.geometry != self.geometry:
            raise ValueError(f"cache of {cache.kv_heads} heads of {cache.head_dim}, pages of {cache.page_size}, {cache.dtype}; the reader has "
                             f"{self.kv_heads}, {self.head_dim}, {self.page_size}, {self.dtype}")
        if cache.device != self.device:
            _place(cache.k_pages, "cache", cache.device, self.device)
        return cache.ref

    def plan(self, new_lens, cached_lens, block_table, free_pages, free_count, *, q_start, kv_lens, slots, positions,
             free_count_out, next_lens=None, stream: int = 0) -> None:
        """Block table rows extended, and q_start, kv_lens, slots, positions of a step (mars_kv_plan). next_lens: the tokens
        in the cache after it, the next step's cached_lens (kv_lens is 0 for a request that pages did not suffice for)."""
        r, t = new_lens.shape[0], slots.shape[0]
        if len(block_table.shape) != 2:
            raise ValueError(f"block_table: shape {tuple(block_table.shape)}, expected (requests, pages)")
        width = block_table.shape[1]
        *head, next_lens = _args(
            self.device, (new_lens, "new_lens", "int32", (r,)), (cached_lens, "cached_lens", "int32", (r,)),
            (block_table, "block_table", "int32", (r, width)), (free_pages, "free_pages", "int32", None), (free_count, "free_count", "int32", (1,)),
            (q_start, "q_start", "int32", (r + 1,)), (kv_lens, "kv_lens", "int32", (r,)), (slots, "slots", "int64", (t,)),
            (positions, "positions", "int32", (t,)), (free_count_out, "free_count_out", "int32", (1,)), (next_lens, "next_lens", "int32", (r,)))
        a = _lib.KvPlanArgsC(*head, r, width, t, int(free_pages.shape[0]), next_lens)
        rc = lib.mars_kv_plan(self.handle, a, stream)
        if rc:
            check(rc, "mars_kv_plan")

    def release(self, done, kv_lens, block_table, free_pages, free_count, stream: int = 0) -> None:
        """The pages of requests with done != 0 pushed onto free_pages; their kv_lens (plan's next_lens) become 0 (mars_kv_release)."""
        r = int(done.shape[0])
        if len(block_table.shape) != 2:
            raise ValueError(f"block_table: shape {tuple(block_table.shape)}, expected (requests, pages)")
        width = int(block_table.shape[1])
        done, kv_lens, table, pages, count = _args(
            self.device, (done, "done", "int32", (r,)), (kv_lens, "kv_lens", "int32", (r,)), (block_table, "block_table", "int32", (r, width)),
            (free_pages, "free_pages", "int32", None), (free_count, "free_count", "int32", (1,)))
        check(lib.mars_kv_release(self.handle, done, kv_lens, table, r, width, pages, count, int(free_pages.shape[0]), stream), "mars_kv_release")

    def store(self, cache: Optional[PagedCache], q, k, v, positions, slots, *, q_out=None, times=None, episodes=None,
              inverse: bool = False, stream: int = 0) -> None:
        """q and k turned by their positions (axes, tokens), k, v, times, episodes written to `slots` (mars_kv_store).
        q_out: where the turned q goes (default q itself). k and v None: only q is turned; q None: only stores."""
        first = q if q is not None else k
        if first is None:
            raise ValueError("neither q nor k")
        t, g = int(first.shape[0]), self.device
        a = _lib.KvStoreArgsC(num_tokens=t, inverse=int(bool(inverse)))
        if q is not None:
            a.q, a.q_stride = _rows(q, "q", self.dtype, g, t, self.q_heads, self.head_dim)
            a.q_out, a.q_out_stride = (a.q, a.q_stride) if q_out is None else _rows(q_out, "q_out", self.dtype, g, t, self.q_heads, self.head_dim)
        ref = None
        if k is not None or v is not None:
            if k is None or v is None or cache is None or slots is None:
                raise ValueError("k, v, cache and slots come together")
            a.k, a.k_stride = _rows(k, "k", self.dtype, g, t, self.kv_heads, self.head_dim)
            a.v, a.v_stride = _rows(v, "v", self.dtype, g, t, self.kv_heads, self.head_dim)
            a.slots, a.times, a.episodes = _args(g, (slots, "slots", "int64", (t,)), (times, "times", "float32", (t,)),
                                                 (episodes, "episodes", "int32", (t,)))
            ref = self._cache(cache)
        if self.rope_dim:
            if positions is None:
                raise ValueError("positions are needed")
            want = (t,) if self.rope_axes == 1 and len(positions.shape) == 1 else (self.rope_axes, t)
            a.positions, = _args(g, (positions, "positions", "int32", want))
        rc = lib.mars_kv_store(self.handle, ref, a, stream)
        if rc:
            check(rc, "mars_kv_store")

    def attend(self, cache: PagedCache, q, out, q_start, kv_lens, block_table, *, lse=None, scale: float = 0.0,
               cap: float = 0.0, decay=None, q_times=None, q_episodes=None, prefix_lens=None, max_new: int = 0,
               stream: int = 0) -> None:
        """Attention of each request's rows of q over its cached tokens, into out (mars_kv_attend)."""
        t, r, g = q.shape[0], kv_lens.shape[0], self.device
        ref = self._cache(cache)
        qp, qs = _rows(q, "q", self.dtype, g, None, self.q_heads, self.head_dim)
        op, os_ = _rows(out, "out", self.dtype, g, t, self.q_heads, self.head_dim)
        if len(block_table.shape) != 2:
            raise ValueError(f"block_table: shape {tuple(block_table.shape)}, expected (requests, pages)")
        width = block_table.shape[1]
        a = _lib.KvAttendArgsC(
            qp, op, *_args(g, (lse, "lse", "float32", (t, self.q_heads)), (q_start, "q_start", "int32", (r + 1,)),
                           (kv_lens, "kv_lens", "int32", (r,)), (block_table, "block_table", "int32", (r, width)),
                           (decay, "decay", "float32", (self.q_heads,)), (q_times, "q_times", "float32", (t,)),
                           (q_episodes, "q_episodes", "int32", (t,)), (prefix_lens, "prefix_lens", "int32", (r,))),
            qs, os_, scale, cap, r, width, t, max_new)
        rc = lib.mars_kv_attend(self.handle, ref, a, stream)
        if rc:
            check(rc, "mars_kv_attend")
