"""What the calls over 8-bit caches and shared prefixes refuse, before any device work; and the restatement's own e4m3 against torch's."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import reader8_ref as ref8
from mars_amd import _lib
from mars_amd._lib import MarsError, check, lib
from mars_amd.reader import PagedCache
from test_reader_args import CAPACITY, INVALID, Fake, On, a_reader, f32, i32

U8 = "uint8"


def cache8(n=9, h=2, p=16, d=64, dtype=U8, **kw):
    a = dict(k_pages=Fake(n, h, p, d, dtype=dtype), v_pages=Fake(n, h, d, p, dtype=dtype), k_scales=Fake(n, h, p, dtype=U8), v_scales=Fake(n, h, p, dtype=U8))
    a.update(kw)
    return PagedCache(**a)


def test_restatement():
    """Every e4m3 value, and the rounding of values between, as torch's float8_e4m3fn has them."""
    torch = pytest.importorskip("torch")
    b = np.arange(256, dtype=np.uint8)
    t = torch.from_numpy(b.copy()).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(ref8.VALUES, t)
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(50_000) * 2.0 ** rng.integers(-14, 7, 50_000), (ref8._POSITIVE[1:] + ref8._POSITIVE[:-1]) / 2, -ref8._POSITIVE])
    x = x.astype(np.float32).astype(np.float64)
    x = x[np.abs(x) <= 448]
    np.testing.assert_array_equal(ref8.to_e4m3(x), torch.from_numpy(x).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    for top in (448.0, 448.1, 1.0, 1.75, 1.7500001, 2.0 ** -30, 6e4):
        e = int(ref8.exponent(np.array([top]), "bfloat16"))
        assert 224 * 2.0 ** (e - 127) < top <= 448 * 2.0 ** (e - 127)
    assert ref8.exponent(np.zeros(4), "float16") == 112 and ref8.exponent(np.array([np.nan, np.inf, 7.0]), "float16") == 121


@pytest.mark.parametrize("kw", [
    dict(k_scales=None), dict(v_scales=None), dict(k_scales=Fake(9, 2, 16, dtype="float32")), dict(v_scales=Fake(9, 16, 2, dtype=U8)),
    dict(k_scales=Fake(8, 2, 16, dtype=U8)), dict(k_scales=Fake(9, 2, 16, dtype=U8, strides=(64, 32, 1))), dict(k_pages=Fake(9, 2, 16, 64, dtype="float16")),
    dict(k_pages=Fake(9, 2, 16, 64), v_pages=Fake(9, 2, 64, 16)), dict(v_pages=Fake(9, 2, 16, 64, dtype=U8)), dict(times=f32(8)),
    dict(k_pages=Fake(9, 2, 16, 64, dtype=U8, strides=(2048, 64, 128, 1))),
])
def test_caches(kw):
    cache8()
    cache8(dtype="float8_e4m3fn")
    cache8(k_pages=Fake(9, 2, 16, 64, dtype=U8, strides=(4096, 1024, 64, 1)))
    with pytest.raises(ValueError):
        cache8(**kw)
    with pytest.raises(ValueError):
        PagedCache(Fake(9, 2, 16, 64, dtype=U8), Fake(9, 2, 64, 16, dtype=U8))


LOAD = dict(slots=Fake(7, dtype="int64"), k=Fake(7, 2, 64), v=Fake(7, 2, 64), times=f32(7), episodes=i32(7))
ATTEND = dict(q=Fake(7, 4, 64), out=Fake(7, 4, 64), q_start=i32(4), kv_lens=i32(3), block_table=i32(3, 5), group_start=i32(3), shared_lens=i32(2))


@pytest.mark.parametrize("change", [dict(slots=i32(7)), dict(k=None), dict(v=None), dict(k=Fake(7, 4, 64)), dict(v=Fake(6, 2, 64)), dict(k=Fake(7, 2, 64, dtype="bfloat16")),
                                    dict(v=Fake(7, 2, 64, strides=(128, 1, 2))), dict(times=i32(7)), dict(times=f32(8)), dict(episodes=i32(6))])
def test_load_shapes(change):
    a = {**LOAD, **change}
    for c in (cache8(times=f32(144), episodes=i32(144)), PagedCache(Fake(9, 2, 16, 64), Fake(9, 2, 64, 16), f32(144), i32(144))):
        with pytest.raises(ValueError):
            a_reader().load(c, a["slots"], a["k"], a["v"], times=a["times"], episodes=a["episodes"])


@pytest.mark.parametrize("change", [dict(group_start=None), dict(shared_lens=None), dict(group_start=i32(2)), dict(shared_lens=f32(2)), dict(group_start=Fake(3, dtype="int64")),
                                    dict(shared_lens=i32(3)), dict(q=Fake(7, 4, 32))])
def test_shared_shapes(change):
    for c in (cache8(), PagedCache(Fake(9, 2, 16, 64), Fake(9, 2, 64, 16))):
        with pytest.raises(ValueError):
            a_reader().attend(c, **{**ATTEND, **change})
    if "q" not in change:
        g = {n: {**ATTEND, **change}[n] for n in ("group_start", "shared_lens")}
        with pytest.raises(ValueError):
            a_reader().release(i32(3), i32(3), i32(3, 5), i32(20), i32(1), **g)


@pytest.mark.parametrize("c", [cache8(h=4), cache8(p=32), cache8(d=128)])
def test_caches_of_another_geometry(c):
    for call in (lambda r: r.attend(c, **ATTEND), lambda r: r.load(c, **LOAD),
                 lambda r: r.store(c, None, Fake(7, 2, 64), Fake(7, 2, 64), i32(7), Fake(7, dtype="int64"))):
        with pytest.raises(ValueError):
            call(a_reader())


def calls():
    c = dict(k_pages=Fake(9, 2, 16, 64, dtype=U8), v_pages=Fake(9, 2, 64, 16, dtype=U8), k_scales=Fake(9, 2, 16, dtype=U8), v_scales=Fake(9, 2, 16, dtype=U8),
             c_times=f32(144), c_episodes=i32(144))

    def paged(a):
        return PagedCache(a["k_pages"], a["v_pages"], a["c_times"], a["c_episodes"], a["k_scales"], a["v_scales"])

    def store(r, a):
        r.store(paged(a), None, a["k"], a["v"], a["positions"], a["slots"])

    def load(r, a):
        r.load(paged(a), a["slots"], a["k"], a["v"], times=a["times"], episodes=a["episodes"])

    def attend(r, a):
        r.attend(paged(a), a["q"], a["out"], a["q_start"], a["kv_lens"], a["block_table"], group_start=a["group_start"], shared_lens=a["shared_lens"])

    def release(r, a):
        r.release(a["done"], a["kv_lens"], a["block_table"], a["free"], a["count"], a["group_start"], a["shared_lens"])

    return [(store, dict(c, k=LOAD["k"], v=LOAD["v"], positions=i32(7), slots=LOAD["slots"])), (load, dict(c, **LOAD)), (attend, dict(c, **ATTEND)),
            (release, dict(done=i32(3), kv_lens=i32(3), block_table=i32(3, 5), free=i32(20), count=i32(1), group_start=i32(3), shared_lens=i32(2)))]


@pytest.mark.parametrize("call,arrays", calls(), ids=["store", "load", "attend", "release"])
def test_arrays_on_the_host_or_another_gpu(call, arrays):
    here = {n: On(x, 1) for n, x in arrays.items()}

    def reaches_c(a, r):
        with pytest.raises(MarsError) as e:              # no handle: refused there, before any device work
            call(r, a)
        assert e.value.code == INVALID

    reaches_c(arrays, a_reader())
    reaches_c(here, a_reader(device=1))
    for n, x in arrays.items():
        for at in (-1, 0, 2):
            with pytest.raises(ValueError):
                call(a_reader(device=1), dict(here, **{n: On(x, at)}))
        reaches_c(dict(here, **{n: On(x, -1, pinned=True)}), a_reader(device=1))
    with pytest.raises(ValueError):
        call(a_reader(device=0), here)


def test_null_arguments():
    for name, args in (("mars_kv_store8", (None,) * 4), ("mars_kv_load", (None,) * 4), ("mars_kv_load8", (None,) * 4), ("mars_kv_attend8", (None,) * 5),
                       ("mars_kv_attend_shared", (None,) * 5), ("mars_kv_release_shared", (None, None, None, None, 1, 1, None, None, None, 1, None))):
        with pytest.raises(MarsError) as e:
            check(getattr(lib, name)(*args), name)
        assert e.value.code == INVALID


def test_release_stream_and_groups(monkeypatch):
    """The stream stands sixth, as it does without groups, or behind the groups, or by name."""
    from mars_amd import reader
    seen = []

    class Calls:
        def mars_kv_release(self, handle, done, lens, table, r, width, free, count, capacity, stream):
            seen.append((r, width, capacity, None, stream))
            return 0

        def mars_kv_release_shared(self, handle, done, lens, table, r, width, shared, free, count, capacity, stream):
            seen.append((r, width, capacity, shared.num_groups, stream))
            return 0

    monkeypatch.setattr(reader, "lib", Calls())
    r, a = a_reader(), (i32(3), i32(3), i32(3, 5), i32(20), i32(1))
    g = i32(3), i32(2)
    named = dict(group_start=g[0], shared_lens=g[1])
    for args, kw, want in (((), {}, (None, 0)), ((77,), {}, (None, 77)), ((0,), {}, (None, 0)), ((), dict(stream=77), (None, 77)), (g, {}, (2, 0)), ((*g, 77), {}, (2, 77)),
                           (g, dict(stream=77), (2, 77)), ((g[0],), dict(shared_lens=g[1], stream=77), (2, 77)), ((), dict(named, stream=77), (2, 77)), ((77,), named, (2, 77)),
                           ((None, None, 77), {}, (None, 77))):
        r.release(*a, *args, **kw)
        assert seen.pop() == (3, 5, 20, *want), (args, kw)
    for args, kw, error in (((g[0],), {}, ValueError), ((77,), dict(group_start=g[0]), ValueError), ((77, 78), {}, TypeError), ((77,), dict(stream=78), TypeError),
                            (g, named, TypeError), ((*g, 77, 78), {}, TypeError)):
        with pytest.raises(error):
            r.release(*a, *args, **kw)
    assert not seen


@pytest.mark.gpu
def test_c_refusals():
    """Arguments that only the C entries can check, on arrays that are there; nothing is launched, nothing written."""
    import mars_amd
    from mars_amd.reader import DeviceArray, Reader
    mars_amd.init(0)
    r = Reader(4, 2, 64, "float16", 16, rope_dim=64)
    names = ("q", "k", "v", "out", "q_out", "k_pages", "v_pages", "k_scales", "v_scales", "times", "episodes", "q_start", "kv_lens", "block_table", "slots", "positions",
             "free_pages", "free_count", "other", "group_start", "shared_lens", "done")
    zeros = {n: DeviceArray.from_numpy(np.zeros(1 << 16, np.int64)) for n in names}
    p = {n: x.data_ptr() for n, x in zeros.items()}

    def some(keys, **kw):
        return {**{n: p[n] for n in keys.split()}, **kw}

    pages = some("k_pages v_pages", num_pages=9)
    eight = some("k_scales v_scales", **pages)
    shared = some("group_start shared_lens", num_groups=2)
    attend = some("q out q_start kv_lens block_table", q_stride=256, out_stride=256, num_requests=3, max_pages=5, num_tokens=7)
    store = some("k v slots positions", k_stride=128, v_stride=128, num_tokens=7)
    load = some("k v slots", k_stride=128, v_stride=128, num_tokens=7)

    def calls8(c):
        c = C.byref(_lib.KvCache8C(**c))
        return [lib.mars_kv_attend8(r.handle, c, C.byref(_lib.KvAttendArgsC(**attend)), None, None),
                lib.mars_kv_attend8(r.handle, c, C.byref(_lib.KvAttendArgsC(**attend)), C.byref(_lib.KvSharedC(**shared)), None),
                lib.mars_kv_store8(r.handle, c, C.byref(_lib.KvStoreArgsC(**store)), None),
                lib.mars_kv_load8(r.handle, c, C.byref(_lib.KvLoadArgsC(**load)), None)]

    for kw in (dict(k_pages=None), dict(num_pages=0), dict(k_scales=None), dict(v_scales=None), dict(k_scales=p["k_scales"] + 8), dict(k_page_stride=8),
               dict(v_page_stride=2056), dict(v_pages=p["v_pages"] + 8), dict(times=p["times"] + 4)):
        assert calls8({**eight, **kw}) == [INVALID] * 4, kw
    for kw, code in ((dict(q=None), INVALID), (dict(num_requests=0), INVALID), (dict(num_requests=4097), CAPACITY), (dict(max_pages=2 ** 28), CAPACITY),
                     (dict(num_tokens=-1), INVALID), (dict(q_stride=260), INVALID), (dict(cap=-1.0), INVALID), (dict(scale=float("inf")), INVALID),
                     (dict(decay=p["other"]), INVALID), (dict(q_episodes=p["other"]), INVALID)):
        a = C.byref(_lib.KvAttendArgsC(**{**attend, **kw}))
        g = C.byref(_lib.KvSharedC(**shared))
        assert lib.mars_kv_attend8(r.handle, C.byref(_lib.KvCache8C(**eight)), a, None, None) == code, kw
        assert lib.mars_kv_attend_shared(r.handle, C.byref(_lib.KvCacheC(**pages)), a, g, None) == code, kw
    for kw in (dict(group_start=None), dict(shared_lens=None), dict(num_groups=0), dict(num_groups=4097)):
        g, a = C.byref(_lib.KvSharedC(**{**shared, **kw})), C.byref(_lib.KvAttendArgsC(**attend))
        assert lib.mars_kv_attend8(r.handle, C.byref(_lib.KvCache8C(**eight)), a, g, None) == INVALID, kw
        assert lib.mars_kv_attend_shared(r.handle, C.byref(_lib.KvCacheC(**pages)), a, g, None) == INVALID, kw
        assert lib.mars_kv_release_shared(r.handle, p["done"], p["kv_lens"], p["block_table"], 3, 5, g, p["free_pages"], p["free_count"], 9, None) == INVALID, kw
    assert lib.mars_kv_attend_shared(r.handle, C.byref(_lib.KvCacheC(**pages)), C.byref(_lib.KvAttendArgsC(**attend)), None, None) == INVALID
    assert lib.mars_kv_release_shared(r.handle, p["done"], p["kv_lens"], p["block_table"], 3, 5, None, p["free_pages"], p["free_count"], 9, None) == INVALID
    for kw in (dict(slots=None), dict(k=None), dict(v=None), dict(k=None, v=None), dict(k_stride=120), dict(v_stride=130), dict(k=p["k"] + 2), dict(times=p["other"]),
               dict(episodes=p["other"]), dict(num_tokens=-1)):
        a = C.byref(_lib.KvLoadArgsC(**{**load, **kw}))
        assert lib.mars_kv_load8(r.handle, C.byref(_lib.KvCache8C(**eight)), a, None) == INVALID, kw
        assert lib.mars_kv_load(r.handle, C.byref(_lib.KvCacheC(**pages)), a, None) == INVALID, kw
    for kw in (dict(slots=None), dict(positions=None), dict(v=None), dict(times=p["other"]), dict(k_stride=120)):
        assert lib.mars_kv_store8(r.handle, C.byref(_lib.KvCache8C(**eight)), C.byref(_lib.KvStoreArgsC(**{**store, **kw})), None) == INVALID, kw
    # nothing to do
    assert lib.mars_kv_load8(r.handle, C.byref(_lib.KvCache8C(**eight)), C.byref(_lib.KvLoadArgsC(**{**load, "num_tokens": 0})), None) == 0
    assert lib.mars_kv_attend8(r.handle, C.byref(_lib.KvCache8C(**eight)), C.byref(_lib.KvAttendArgsC(**{**attend, "num_tokens": 0})), None, None) == 0
    for name, x in zeros.items():
        assert not x.numpy().any(), name
