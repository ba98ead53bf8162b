"""What the reading path refuses, before any device work: geometries, shapes, types, strides and missing arrays."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from mars_amd import _lib
from mars_amd._lib import MarsError, check, lib
from mars_amd.reader import PagedCache, Reader

INVALID, CAPACITY, UNSUPPORTED, NODEVICE = -1, -4, -5, -6


class Fake:
    """An array that is only described: `shape`, `stride`, `dtype` and an aligned address that nothing reads."""

    def __init__(self, *shape, dtype="float16", strides=None, ptr=1 << 20):
        self.shape, self.dtype, self._ptr = shape, dtype, ptr
        self._s = strides or tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))

    def data_ptr(self):
        return self._ptr

    def stride(self, i):
        return self._s[i]


@pytest.mark.parametrize("bad,code", [
    (dict(q_heads=5, kv_heads=2), INVALID), (dict(q_heads=0, kv_heads=0), INVALID), (dict(q_heads=2, kv_heads=4), INVALID),
    (dict(q_heads=65, kv_heads=1), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(page_size=8), UNSUPPORTED),
    (dict(page_size=48), UNSUPPORTED), (dict(page_size=512), UNSUPPORTED), (dict(rope_dim=66), INVALID), (dict(rope_dim=24), INVALID),
    (dict(rope_dim=64, rope_sections=(30,)), INVALID), (dict(rope_dim=64, rope_sections=(40, -8)), INVALID),
    (dict(rope_dim=64, rope_theta=1.0), INVALID), (dict(rope_dim=64, rope_theta=float("inf")), INVALID),
])
def test_reader_geometries(bad, code):
    with pytest.raises(MarsError) as e:
        Reader(**{**dict(q_heads=4, kv_heads=2, head_dim=64), **bad})
    assert e.value.code == code


def test_reader_types():
    with pytest.raises(ValueError):
        Reader(dtype="float32")
    with pytest.raises(ValueError):
        Reader(rope_dim=64, rope_sections=(8, 8, 8, 8))
    desc = _lib.ReaderDescC(4, 2, 64, 7, 16)
    out = C.c_void_p()
    assert lib.mars_reader_create(C.byref(desc), C.byref(out)) == UNSUPPORTED and not out
    assert lib.mars_reader_create(None, C.byref(out)) == INVALID
    assert lib.mars_reader_destroy(None) == 0


def test_caches():
    ok = dict(k=Fake(9, 2, 16, 64), v=Fake(9, 2, 64, 16))
    PagedCache(ok["k"], ok["v"])
    PagedCache(Fake(9, 2, 16, 64, strides=(4096, 1024, 64, 1)), Fake(9, 2, 64, 16, strides=(4096, 1024, 16, 1)))
    for k, v in ((Fake(9, 2, 16, 64), Fake(9, 2, 16, 64)), (Fake(9, 2, 64), ok["v"]), (ok["k"], Fake(9, 2, 64, 16, dtype="bfloat16")),
                 (Fake(9, 2, 16, 64, dtype="float32"), Fake(9, 2, 64, 16, dtype="float32")),
                 (Fake(9, 2, 16, 64, strides=(2048, 64, 128, 1)), ok["v"]), (ok["k"], Fake(8, 2, 64, 16))):
        with pytest.raises(ValueError):
            PagedCache(k, v)
    for t, e in ((Fake(9 * 16 - 1, dtype="float32"), None), (Fake(9, 16, dtype="float16"), None), (None, Fake(9, 16, dtype="float32"))):
        with pytest.raises(ValueError):
            PagedCache(ok["k"], ok["v"], t, e)


def a_reader(**kw):
    """A Reader without a device behind it: every call below is refused before its handle is used."""
    r = Reader.__new__(Reader)
    r.q_heads, r.kv_heads, r.head_dim, r.dtype, r.page_size, r.rope_dim, r.rope_axes = 4, 2, 64, "float16", 16, 64, 1
    r.geometry = (2, 16, 64, "float16")
    r.handle = C.c_void_p()
    for k, v in kw.items():
        setattr(r, k, v)
    return r


CACHE = (Fake(9, 2, 16, 64), Fake(9, 2, 64, 16))


def i32(*shape):
    return Fake(*shape, dtype="int32")


@pytest.mark.parametrize("change", [
    dict(q=Fake(7, 4, 32)), dict(q=Fake(7, 3, 64)), dict(q=Fake(7, 4, 64, dtype="bfloat16")), dict(q=Fake(7, 4, 64, strides=(256, 1, 4))),
    dict(out=Fake(6, 4, 64)), dict(q_start=i32(3)), dict(q_start=Fake(4, dtype="int64")), dict(kv_lens=Fake(3, dtype="float32")),
    dict(table=i32(2, 5)), dict(table=i32(3)), dict(lse=Fake(7, 4)), dict(decay=Fake(3, dtype="float32")), dict(q_times=Fake(6, dtype="float32")),
    dict(q_eps=i32(8)), dict(prefix=i32(2)), dict(cache=PagedCache(Fake(9, 4, 16, 64), Fake(9, 4, 64, 16))),
    dict(cache=PagedCache(Fake(9, 2, 32, 64), Fake(9, 2, 64, 32))), dict(table=Fake(3, 5, dtype="int32", strides=(1, 3))),
])
def test_attend_shapes(change):
    a = dict(cache=PagedCache(*CACHE), q=Fake(7, 4, 64), out=Fake(7, 4, 64), q_start=i32(4), kv_lens=i32(3), table=i32(3, 5), lse=None, decay=None,
             q_times=None, q_eps=None, prefix=None)
    a.update(change)
    with pytest.raises(ValueError):
        a_reader().attend(a["cache"], a["q"], a["out"], a["q_start"], a["kv_lens"], a["table"], lse=a["lse"], decay=a["decay"],
                          q_times=a["q_times"], q_episodes=a["q_eps"], prefix_lens=a["prefix"])


@pytest.mark.parametrize("change", [
    dict(q=None, k=None, v=None), dict(v=None), dict(slots=None), dict(slots=i32(7)), dict(positions=None), dict(positions=i32(2, 7)),
    dict(positions=Fake(7, dtype="float32")), dict(k=Fake(7, 4, 64)), dict(k=Fake(6, 2, 64)), dict(times=Fake(6, dtype="float32")),
    dict(episodes=Fake(7, dtype="float32")), dict(cache=None), dict(q_out=Fake(7, 4, 32)),
])
def test_store_shapes(change):
    a = dict(cache=PagedCache(*CACHE), q=Fake(7, 4, 64), k=Fake(7, 2, 64), v=Fake(7, 2, 64), positions=i32(7), slots=Fake(7, dtype="int64"),
             q_out=None, times=None, episodes=None)
    a.update(change)
    with pytest.raises(ValueError):
        a_reader().store(a.pop("cache"), a.pop("q"), a.pop("k"), a.pop("v"), a.pop("positions"), a.pop("slots"), **a)


@pytest.mark.parametrize("change", [dict(cached=i32(4)), dict(table=i32(2, 5)), dict(count=i32(2)), dict(q_start=i32(3)), dict(slots=i32(7)),
                                    dict(positions=i32(8)), dict(left=i32(0))])
def test_plan_shapes(change):
    a = dict(cached=i32(3), table=i32(3, 5), count=i32(1), q_start=i32(4), slots=Fake(7, dtype="int64"), positions=i32(7), left=i32(1))
    a.update(change)
    with pytest.raises(ValueError):
        a_reader().plan(i32(3), a["cached"], a["table"], i32(20), a["count"], q_start=a["q_start"], kv_lens=i32(3), slots=a["slots"],
                        positions=a["positions"], free_count_out=a["left"])


class On(Fake):
    """The same that also says where it lies: a GPU's number, or -1 for host memory."""

    def __init__(self, x, device, pinned=False):
        super().__init__(*x.shape, dtype=x.dtype, strides=x._s)
        self._device, self._pinned = device, pinned

    def get_device(self):
        return self._device

    def is_pinned(self):
        return self._pinned


def f32(*shape):
    return Fake(*shape, dtype="float32")


def calls():
    """Every call with all its arrays by name."""
    k, v, times, eps = Fake(9, 2, 16, 64), Fake(9, 2, 64, 16), f32(9 * 16), i32(9 * 16)
    cache = dict(k_pages=k, v_pages=v, c_times=times, c_episodes=eps)

    def paged(a):
        return PagedCache(a["k_pages"], a["v_pages"], a["c_times"], a["c_episodes"])

    def plan(r, a):
        r.plan(a["new"], a["cached"], a["table"], a["free"], a["count"], q_start=a["q_start"], kv_lens=a["kv_lens"], slots=a["slots"],
               positions=a["positions"], free_count_out=a["left"], next_lens=a["next_lens"])

    def store(r, a):
        r.store(paged(a), a["q"], a["k"], a["v"], a["positions"], a["slots"], q_out=a["q_out"], times=a["times"], episodes=a["episodes"])

    def attend(r, a):
        r.attend(paged(a), a["q"], a["out"], a["q_start"], a["kv_lens"], a["table"], lse=a["lse"], decay=a["decay"], q_times=a["q_times"],
                 q_episodes=a["q_eps"], prefix_lens=a["prefix"])

    def release(r, a):
        r.release(a["done"], a["kv_lens"], a["table"], a["free"], a["count"])

    slots = Fake(7, dtype="int64")
    return [(plan, dict(new=i32(3), cached=i32(3), table=i32(3, 5), free=i32(20), count=i32(1), q_start=i32(4), kv_lens=i32(3), slots=slots,
                        positions=i32(7), left=i32(1), next_lens=i32(3))),
            (store, dict(cache, q=Fake(7, 4, 64), k=Fake(7, 2, 64), v=Fake(7, 2, 64), positions=i32(7), slots=slots, q_out=Fake(7, 4, 64),
                         times=f32(7), episodes=i32(7))),
            (attend, dict(cache, q=Fake(7, 4, 64), out=Fake(7, 4, 64), q_start=i32(4), kv_lens=i32(3), table=i32(3, 5), lse=f32(7, 4),
                          decay=f32(4), q_times=f32(7), q_eps=i32(7), prefix=i32(3))),
            (release, dict(done=i32(3), kv_lens=i32(3), table=i32(3, 5), free=i32(20), count=i32(1)))]


@pytest.mark.parametrize("call,arrays", calls(), ids=["plan", "store", "attend", "release"])
def test_arrays_on_the_host_or_another_gpu(call, arrays):
    """An address in host memory, or in another GPU's, never reaches a kernel; pinned memory, which kernels read, may."""
    here = {n: On(x, 1) for n, x in arrays.items()}

    def reaches_c(a, r):
        with pytest.raises(MarsError) as e:              # no handle: refused there, before any device work
            call(r, a)
        assert e.value.code == INVALID

    reaches_c(arrays, a_reader())                        # arrays that do not say where they are
    reaches_c(arrays, a_reader(device=1))
    reaches_c(here, a_reader(device=1))
    for n, x in arrays.items():
        for at in (-1, 0, 2):
            with pytest.raises(ValueError):
                call(a_reader(device=1), dict(here, **{n: On(x, at)}))
        reaches_c(dict(here, **{n: On(x, -1, pinned=True)}), a_reader(device=1))
    with pytest.raises(ValueError):
        call(a_reader(device=0), here)


def test_release_shapes():
    for kw in (dict(kv_lens=i32(2)), dict(table=i32(3)), dict(table=i32(2, 5)), dict(count=i32(2)), dict(free=f32(20))):
        a = dict(kv_lens=i32(3), table=i32(3, 5), free=i32(20), count=i32(1))
        a.update(kw)
        with pytest.raises(ValueError):
            a_reader().release(i32(3), a["kv_lens"], a["table"], a["free"], a["count"])


def test_null_arguments():
    """The C entries report a missing handle or argument block, and touch nothing."""
    for name, args in (("mars_kv_plan", (None, None, None)), ("mars_kv_store", (None, None, None, None)),
                       ("mars_kv_attend", (None, None, None, None)), ("mars_kv_release", (None, None, None, None, 1, 1, None, None, 1, None))):
        with pytest.raises(MarsError) as e:
            check(getattr(lib, name)(*args), name)
        assert e.value.code == INVALID


@pytest.mark.gpu
def test_refusals_of_live_arrays():
    """The refusals of the tests below on arrays that are there, zeros of a size that any of these calls stays in: where a check
    is lost, this test fails, and nothing is touched that is not its own."""
    import mars_amd
    from mars_amd.reader import DeviceArray
    mars_amd.init(0)
    r = Reader(4, 2, 64, "float16", 16, rope_dim=64)
    names = ("q", "k", "v", "out", "q_out", "k_pages", "v_pages", "times", "episodes", "q_start", "kv_lens", "block_table", "slots", "positions",
             "new_lens", "cached_lens", "free_pages", "free_count", "free_count_out", "other")
    zeros = {n: DeviceArray.from_numpy(np.zeros(1 << 16, np.int64)) for n in names}
    p = {n: x.data_ptr() for n, x in zeros.items()}

    def cache(**kw):
        return _lib.KvCacheC(**{**dict(k_pages=p["k_pages"], v_pages=p["v_pages"], num_pages=9), **kw})

    def some(keys, **kw):
        return {**{n: p[n] for n in keys.split()}, **kw}

    attend = some("q out q_start kv_lens block_table", q_stride=256, out_stride=256, num_requests=3, max_pages=5, num_tokens=7)
    for kw, code in ((dict(q=None), INVALID), (dict(num_requests=0), INVALID), (dict(num_requests=4097), CAPACITY), (dict(max_pages=0), INVALID),
                     (dict(max_pages=2 ** 28), CAPACITY), (dict(num_tokens=-1), INVALID), (dict(num_tokens=2 ** 30), CAPACITY),
                     (dict(q_stride=248), INVALID), (dict(q_stride=260), INVALID), (dict(q=p["q"] + 2), INVALID), (dict(out_stride=12), INVALID),
                     (dict(cap=-1.0), INVALID), (dict(cap=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(decay=p["other"]), INVALID),
                     (dict(q_episodes=p["other"]), INVALID), (dict(max_new=-1), INVALID)):
        assert lib.mars_kv_attend(r.handle, C.byref(cache()), C.byref(_lib.KvAttendArgsC(**{**attend, **kw})), None) == code, kw
    for kw in (dict(k_pages=None), dict(num_pages=0), dict(k_page_stride=8), dict(v_page_stride=4097), dict(k_pages=p["k_pages"] + 8),
               dict(times=p["times"] + 4)):
        assert lib.mars_kv_attend(r.handle, C.byref(cache(**kw)), C.byref(_lib.KvAttendArgsC(**attend)), None) == INVALID, kw
    store = some("q k v q_out positions slots", q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, num_tokens=7)
    for kw in (dict(q=None, k=None, v=None), dict(v=None), dict(q_out=None), dict(slots=None), dict(positions=None), dict(k_stride=120),
               dict(v_stride=130), dict(q_out=p["q"], q_out_stride=512), dict(times=p["other"]), dict(episodes=p["other"]), dict(num_tokens=-1),
               dict(k=p["k"] + 2)):
        assert lib.mars_kv_store(r.handle, C.byref(cache()), C.byref(_lib.KvStoreArgsC(**{**store, **kw})), None) == INVALID, kw
    plan = some("new_lens cached_lens block_table free_pages free_count q_start kv_lens slots positions free_count_out", num_requests=3, max_pages=5,
                num_tokens=7, free_capacity=9)
    for kw, code in ((dict(new_lens=None), INVALID), (dict(slots=None), INVALID), (dict(free_count_out=p["free_count"]), INVALID),
                     (dict(num_requests=0), INVALID), (dict(num_requests=4097), CAPACITY), (dict(max_pages=0), INVALID), (dict(free_capacity=-1), INVALID),
                     (dict(num_tokens=-1), INVALID), (dict(kv_lens=p["cached_lens"]), INVALID), (dict(kv_lens=p["new_lens"]), INVALID),
                     (dict(q_start=p["cached_lens"]), INVALID), (dict(q_start=p["new_lens"]), INVALID)):
        assert lib.mars_kv_plan(r.handle, C.byref(_lib.KvPlanArgsC(**{**plan, **kw})), None) == code, kw
    for name, x in zeros.items():
        assert not x.numpy().any(), name


@pytest.mark.gpu
def test_c_refusals():
    """Arguments that only the C entries can check, on a live reader; nothing is launched."""
    import mars_amd
    mars_amd.init(0)
    r = Reader(4, 2, 64, "float16", 16, rope_dim=64)
    p = 1 << 20

    def cache(**kw):
        return _lib.KvCacheC(**{**dict(k_pages=p, v_pages=p, num_pages=9), **kw})

    good = dict(q=p, out=p, q_start=p, kv_lens=p, block_table=p, q_stride=256, out_stride=256, num_requests=3, max_pages=5, num_tokens=7)

    def attend(c=None, **kw):
        a = _lib.KvAttendArgsC(**{**good, **kw})
        return lib.mars_kv_attend(r.handle, C.byref(c or cache()), C.byref(a), None)

    for kw, code in ((dict(q=None), INVALID), (dict(num_requests=0), INVALID), (dict(num_requests=4097), CAPACITY), (dict(max_pages=0), INVALID),
                     (dict(max_pages=2 ** 28), CAPACITY), (dict(num_tokens=-1), INVALID), (dict(num_tokens=2 ** 30), CAPACITY), (dict(q_stride=248), INVALID),
                     (dict(q_stride=260), INVALID), (dict(q=p + 2), INVALID), (dict(out_stride=12), INVALID), (dict(cap=-1.0), INVALID),
                     (dict(cap=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(decay=p), INVALID), (dict(q_episodes=p), INVALID),
                     (dict(max_new=-1), INVALID)):
        assert attend(**kw) == code, kw
    for c in (cache(k_pages=None), cache(num_pages=0), cache(k_page_stride=8), cache(v_page_stride=4097), cache(k_pages=p + 8), cache(times=p + 4)):
        assert attend(c) == INVALID
    assert attend(num_tokens=0) == 0                     # nothing to do
    store = dict(q=p, k=p, v=p, q_out=p, positions=p, slots=p, q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, num_tokens=7)
    for kw in (dict(q=None, k=None, v=None), dict(v=None), dict(q_out=None), dict(slots=None), dict(positions=None), dict(k_stride=120), dict(v_stride=130),
               dict(q_out_stride=512), dict(times=p), dict(episodes=p), dict(num_tokens=-1), dict(k=p + 2)):
        a = _lib.KvStoreArgsC(**{**store, **kw})
        assert lib.mars_kv_store(r.handle, C.byref(cache()), C.byref(a), None) == INVALID, kw
    plan = dict(new_lens=p, cached_lens=p, block_table=p, free_pages=p, free_count=p, q_start=p, kv_lens=p, slots=p, positions=p,
                free_count_out=p + 64, num_requests=3, max_pages=5, num_tokens=7, free_capacity=9)
    for kw, code in ((dict(new_lens=None), INVALID), (dict(slots=None), INVALID), (dict(free_count_out=p), INVALID), (dict(num_requests=0), INVALID),
                     (dict(num_requests=4097), CAPACITY), (dict(max_pages=0), INVALID), (dict(free_capacity=-1), INVALID), (dict(num_tokens=-1), INVALID)):
        a = _lib.KvPlanArgsC(**{**plan, **kw})
        assert lib.mars_kv_plan(r.handle, C.byref(a), None) == code, kw


@pytest.mark.gpu
def test_plan_refuses_lengths_in_place():
    """kv_lens and q_start are written while other workgroups still read the lengths; nothing is launched."""
    import mars_amd
    mars_amd.init(0)
    r = Reader(4, 2, 64, "float16", 16)
    at = [(1 << 20) + 256 * i for i in range(10)]
    names = ("new_lens", "cached_lens", "block_table", "free_pages", "free_count", "q_start", "kv_lens", "slots", "positions", "free_count_out")
    plan = dict(zip(names, at), num_requests=3, max_pages=5, num_tokens=7, free_capacity=9)
    for out in ("kv_lens", "q_start"):
        for lens in ("cached_lens", "new_lens"):
            a = _lib.KvPlanArgsC(**{**plan, out: plan[lens]})
            assert lib.mars_kv_plan(r.handle, C.byref(a), None) == INVALID, (out, lens)


@pytest.mark.gpu
def test_plan_refuses_next_lens_in_place():
    """next_lens is written while other workgroups still read the lengths, and beside kv_lens and q_start."""
    import mars_amd
    from mars_amd.reader import DeviceArray
    mars_amd.init(0)
    r = Reader(4, 2, 64, "float16", 16)
    names = ("new_lens", "cached_lens", "block_table", "free_pages", "free_count", "q_start", "kv_lens", "slots", "positions", "free_count_out",
             "next_lens")
    arrays = {n: DeviceArray.from_numpy(np.zeros(64, np.int64)) for n in names}
    plan = dict({n: x.data_ptr() for n, x in arrays.items()}, num_requests=3, max_pages=5, num_tokens=7, free_capacity=9)
    for other in ("cached_lens", "new_lens", "kv_lens", "q_start"):
        a = _lib.KvPlanArgsC(**{**plan, "next_lens": plan[other]})
        assert lib.mars_kv_plan(r.handle, C.byref(a), None) == INVALID, other
    for more in (plan, dict(plan, next_lens=None)):      # three requests without tokens
        assert lib.mars_kv_plan(r.handle, C.byref(_lib.KvPlanArgsC(**more)), None) == 0
    assert not any(arrays[n].numpy().any() for n in ("q_start", "kv_lens", "next_lens", "free_count_out"))
