"""Caches of 8 bits and shared prefixes on the GPU (mars_kv_store8, load, load8, attend8, attend_shared, release_shared) against
their 64-bit restatement: layouts, lengths around pages and steps, values at the ends of the types, NaN, groups of every kind."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import mars_amd
import reader8_ref as ref8
import reader_ref as ref
from mars_amd import _lib
from mars_amd.reader import DeviceArray, PagedCache, Reader
from test_gpu_reader import LAYOUTS, _As, dev, make_cache, options, poison

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    mars_amd.init(0)


class View:
    """A view of a device array at an element offset."""

    def __init__(self, base, shape, strides, offset=0):
        self.base, self.shape, self.dtype, self._s = base, shape, base.dtype, strides
        self._o = offset * {"float16": 2, "bfloat16": 2}.get(base.dtype, 1)

    def data_ptr(self):
        return self.base.data_ptr() + self._o

    def stride(self, i):
        return self._s[i]


def bits_of(shape, dtype):
    return np.zeros(shape, np.uint16 if dtype == "bfloat16" else np.float16)


# ---- store ----------------------------------------------------------------------------
def run_store(tokens, hq, hkv, D, dtype, page, rope, sections, adjacent=False, interleaved=False, in_place=False, inverse=False, parts=False, seed=0, x=None):
    rng = np.random.default_rng(seed)
    theta = 1e4 if D == 64 else 1e6
    r = Reader(hq, hkv, D, dtype, page, rope_dim=rope, rope_theta=theta, rope_sections=sections if rope else None, rope_adjacent=adjacent)
    H = hq + 2 * hkv
    if x is None:                                        # heads whose sizes differ by many octaves
        x = rng.standard_normal((tokens, H, D)) * 2.0 ** rng.integers(-9, 4, (tokens, H, 1))
    qkv = ref.to_bits(x, dtype)
    pages = -(-tokens // page) + 3
    slots = rng.permutation(pages)[:, None] * page + np.arange(page)[None]
    slots = slots.reshape(-1)[page // 2 + 1:][:tokens].astype(np.int64)
    slots[rng.random(tokens) < 0.1] = -1
    if tokens > 2:
        slots[0] = pages * page                          # outside the cache: stores nothing
    pos = rng.integers(0, 40_000, (max(len(sections), 1), tokens)).astype(np.int32)
    pos[0, 0], pos[-1, -1] = 2 ** 31 - 1, -70_001
    times, eps = rng.random(tokens).astype(np.float32) * 600, rng.integers(-1, 9, tokens).astype(np.int32)
    d = dev(qkv, dtype)
    q, k, v = (View(d, (tokens, h, D), (H * D, D, 1), o * D) for h, o in ((hq, 0), (hkv, hq), (hkv, hq + hkv)))
    layers, layer = (3, 1) if interleaved else (1, 0)
    n = hkv * page * D
    before = [rng.integers(0, 256, (pages, layers, hkv, page * D)).astype(np.uint8) for _ in range(2)]
    sc = [rng.integers(0, 256, (pages, hkv, page)).astype(np.uint8) for _ in range(2)]
    kb, vb, ks, vs = dev(before[0]), dev(before[1]), dev(sc[0]), dev(sc[1])
    kp = View(kb, (pages, hkv, page, D), (layers * n, page * D, D, 1), layer * n)
    vp = View(vb, (pages, hkv, D, page), (layers * n, page * D, page, 1), layer * n)
    kt, ke = dev(np.full(pages * page, -3, np.float32)), dev(np.full(pages * page, -3, np.int32))
    cache = PagedCache(kp, vp, kt, ke, ks, vs)
    q_out = None if in_place else dev(bits_of((tokens, hq, D), dtype), dtype)
    p = dev(pos) if rope else None
    if parts:
        r.store(cache, None, k, v, p, dev(slots), times=dev(times), inverse=inverse)
        r.store(cache, None, k, v, p, dev(slots), episodes=dev(eps), inverse=inverse)
        r.store(None, q, None, None, p, None, q_out=q_out, inverse=inverse)
    else:
        r.store(cache, q, k, v, p, dev(slots), q_out=q_out, times=dev(times), episodes=dev(eps), inverse=inverse)

    xx = ref.from_bits(qkv, dtype)
    with np.errstate(invalid="ignore"):
        want, size = ref.rotate(xx[:, :hq + hkv], pos, theta, rope, sections, adjacent, inverse)
    err = 2.0 ** -19 * size
    turned = want[:, hq:].copy()
    want = np.concatenate([want[:, :hq], ref8.limited(turned, dtype)], 1)
    got_q = ref.from_bits((d if in_place else q_out).numpy(), dtype)[:, :hq]
    fine = np.isfinite(want[:, :hq])
    off = np.where(size == 0, 0, ref.U[dtype] * np.abs(want) + err + 2.0 ** -25)[:, :hq]
    with np.errstate(invalid="ignore"):
        assert np.all((np.abs(got_q - want[:, :hq]) <= off)[fine])
    ok = (slots >= 0) & (slots < pages * page)
    pg, at = slots[ok] // page, slots[ok] % page
    k_now, v_now = kb.numpy().reshape(pages, layers, hkv, page, D), vb.numpy().reshape(pages, layers, hkv, D, page)
    # v: the bytes themselves
    wb, we = ref8.hold(xx[ok, hq + hkv:], dtype)
    ge = vs.numpy()[pg, :, at]
    np.testing.assert_array_equal(ge, we)
    gb = v_now[pg, layer, :, :, at]
    nan = (wb & 0x7F) == 0x7F
    np.testing.assert_array_equal((gb & 0x7F) == 0x7F, nan)
    np.testing.assert_array_equal(np.where(nan, 0, gb), np.where(nan, 0, wb))
    # k: within half a step of the turned value; the exponent is the reference's wherever the largest element is not at the border
    kw, ks_err = want[ok, hq:], err[ok, hq:]
    ge = ks.numpy()[pg, :, at]
    top = np.max(np.where(np.isfinite(kw), np.abs(kw), 0), -1)
    lo, hi = (ref8.exponent(np.stack([top + s * np.max(np.where(np.isfinite(ks_err), ks_err, 0), -1)], -1).clip(min=0), dtype) for s in (-1, 1))
    assert np.all((lo <= ge) & (ge <= hi))
    got = ref8.held(k_now[pg, layer, :, at], ge[..., None])
    assert np.array_equal(np.isnan(got), ~np.isfinite(kw))
    fine = np.isfinite(kw)
    with np.errstate(invalid="ignore"):
        assert np.all((np.abs(got - kw) <= ref8.half_step(np.where(fine, kw, 0), ge, np.where(fine, ks_err, 0)) + ks_err)[fine])
    same = (size[ok, hq:] == 0) & (ge == ref8.exponent(kw, dtype))[..., None]          # elements that do not turn
    np.testing.assert_array_equal(got[same & fine], ref8.held(*[y if y.ndim == 3 else y[..., None] for y in ref8.hold(kw, dtype)])[same & fine])
    # nothing else is written
    hit = np.zeros((pages, page), bool)
    hit[pg, at] = True
    kw8, vw8 = before[0].reshape(k_now.shape), before[1].reshape(v_now.shape)
    for i in range(layers):
        keep = ~hit if i == layer else np.ones_like(hit)
        np.testing.assert_array_equal(k_now[:, i].transpose(0, 2, 1, 3)[keep], kw8[:, i].transpose(0, 2, 1, 3)[keep])
        np.testing.assert_array_equal(v_now[:, i].transpose(0, 3, 1, 2)[keep], vw8[:, i].transpose(0, 3, 1, 2)[keep])
    for now, old in ((ks, sc[0]), (vs, sc[1])):
        np.testing.assert_array_equal(now.numpy().transpose(0, 2, 1)[~hit], old.transpose(0, 2, 1)[~hit])
    tw, ew = np.full(pages * page, -3, np.float32), np.full(pages * page, -3, np.int32)
    tw[slots[ok]], ew[slots[ok]] = times[ok], eps[ok]
    np.testing.assert_array_equal(kt.numpy(), tw)
    np.testing.assert_array_equal(ke.numpy(), ew)


STORES = [(12, 12, 64, "float16", 16), (8, 2, 128, "bfloat16", 64), (3, 1, 256, "float16", 128), (10, 5, 64, "bfloat16", 256), (7, 7, 128, "float16", 32),
          (4, 2, 256, "bfloat16", 16)]


@pytest.mark.parametrize("tokens", [1, 2, 17, 64, 130, 1029, 2101])
@pytest.mark.parametrize("hq,hkv,D,dtype,page", STORES)
def test_store(tokens, hq, hkv, D, dtype, page):
    run_store(tokens, hq, hkv, D, dtype, page, D, (D // 8, D // 4, D // 8), seed=tokens)


@pytest.mark.parametrize("D,rope,sections,adjacent", [(64, 64, (32,), False), (64, 64, (32,), True), (64, 48, (4, 20, 0), True), (64, 16, (0, 3, 5), False),
                                                      (128, 64, (32,), True), (128, 128, (64,), False), (256, 32, (16,), False), (64, 0, (), False)])
@pytest.mark.parametrize("tokens", [5, 200, 2089])
def test_store_rotations(tokens, D, rope, sections, adjacent):
    run_store(tokens, 4, 2, D, "bfloat16", 32, rope, sections, adjacent, seed=rope)


@pytest.mark.parametrize("tokens", [3, 150, 2100])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_store_layouts(tokens, D):
    run_store(tokens, 6, 2, D, "float16", 16, 64, (32,), interleaved=True, seed=1)
    run_store(tokens, 6, 2, D, "float16", 16, 64, (32,), in_place=True, seed=2)
    run_store(tokens, 6, 2, D, "float16", 16, 64, (16, 16), inverse=True, adjacent=True, seed=3)
    run_store(tokens, 6, 2, D, "bfloat16", 16, 64, (32,), parts=True, seed=4)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("tokens", [40, 2060])
def test_store_values_of_any_size(tokens, dtype):
    """Heads of zeros, of the types' largest and least values, at the borders of an exponent, with infinities and NaN."""
    rng = np.random.default_rng(5)
    hq, hkv, D = 2, 2, 64
    most, least = (65504.0, 2.0 ** -24) if dtype == "float16" else (2.0 ** 127 * (2 - 2.0 ** -7), 2.0 ** -133)
    x = rng.standard_normal((tokens, hq + 2 * hkv, D))
    kinds = [0.0, most, least, 448.0, 449.0, 450.0, 7.0, 7.03125, 2.0 ** -14, np.inf, -np.inf, np.nan, 1.75 * 2.0 ** -10]
    for t in range(tokens):
        k = kinds[t % len(kinds)]
        if np.isfinite(k):
            x[t] = k * rng.uniform(-1, 1, x[t].shape) if t % 2 else 0.0
            x[t, :, t % D] = k * (-1) ** t
        else:
            x[t, :, t % D] = k
    x[0] = np.nan                                        # no finite value at all
    run_store(tokens, hq, hkv, D, dtype, 16, 0, (), x=x)


def test_store_past_32_bits():
    """Pages whose bytes lie past 2^32: stored there, read back and attended there."""
    hq, hkv, D, page, dtype = 4, 2, 128, 256, "float16"
    n = hkv * page * D
    pages = 2 ** 32 // n + 40
    kb, vb = (DeviceArray((pages, hkv, page, D), "uint8") for _ in range(2))
    ks, vs = (DeviceArray((pages, hkv, page), "uint8") for _ in range(2))
    cache = PagedCache(kb, _As(vb, (pages, hkv, D, page)), k_scales=ks, v_scales=vs)
    rng = np.random.default_rng(12)
    L = 2500
    table = np.array([[pages - 1, 2, pages - 17, pages - 3, 5, pages - 30, 7, pages - 12, pages - 13, 9]], np.int32)
    j = np.arange(L)
    slots = table[0][j // page].astype(np.int64) * page + j % page
    x = ref.to_bits(rng.standard_normal((L, hq + 2 * hkv, D)), dtype)
    r = Reader(hq, hkv, D, dtype, page)
    k, v = (dev(np.ascontiguousarray(x[:, hq + i * hkv:hq + (i + 1) * hkv]), dtype) for i in range(2))
    for a, b in ((0, 400), (400, L)):                      # both forms
        part = [View(y, (b - a, hkv, D), (hkv * D, D, 1), a * hkv * D) for y in (k, v)]
        r.store(cache, None, *part, None, dev(slots[a:b]))
    back = [DeviceArray((L, hkv, D), dtype) for _ in range(2)]
    r.load(cache, dev(slots), *back)
    small = []
    for i in range(2):
        b, e = ref8.hold(ref.from_bits(x[:, hq + i * hkv:hq + (i + 1) * hkv], dtype), dtype)
        small.append(ref8.held(b, e[..., None]))
        np.testing.assert_array_equal(back[i].numpy().astype(np.float64), small[i])
    pad = np.zeros((2, 10 * page, hkv, D))
    pad[0, :L], pad[1, :L] = small
    want, _, tol, _ = ref.attend(ref.from_bits(x[-40:, :hq], dtype), pad[0].reshape(10, page, hkv, D).transpose(0, 2, 1, 3),
                                 pad[1].reshape(10, page, hkv, D).transpose(0, 2, 3, 1), [0, 40], [L], np.arange(10)[None], dtype)
    q = dev(np.ascontiguousarray(x[-40:, :hq]), dtype)
    for m in (0, 1):
        out = DeviceArray((40, hq, D), dtype)
        r.attend(cache, q, out, dev(np.array([0, 40], np.int32)), dev(np.array([L], np.int32)), dev(table), max_new=m)
        assert np.all(np.abs(out.numpy().astype(np.float64) - want) <= tol)


# ---- load -----------------------------------------------------------------------------
def make_cache8(rng, shape, dtype):
    """Random finite bytes and exponents that the type's values have."""
    n, h, p, d = shape
    k, v = rng.integers(0, 256, shape).astype(np.uint8), rng.integers(0, 256, (n, h, d, p)).astype(np.uint8)
    k[(k & 0x7F) == 0x7F] ^= 1
    v[(v & 0x7F) == 0x7F] ^= 1
    s = [rng.integers(112, 136, (n, h, p)).astype(np.uint8) for _ in range(2)]
    return k, v, *s


@pytest.mark.parametrize("tokens", [1, 7, 64, 65, 300])
@pytest.mark.parametrize("held8", [True, False])
@pytest.mark.parametrize("hkv,D,dtype,page", [(12, 64, "float16", 16), (2, 128, "bfloat16", 64), (1, 256, "float16", 256), (3, 64, "bfloat16", 32), (2, 256, "bfloat16", 16),
                                              (5, 128, "float16", 128)])
def test_load(hkv, D, dtype, page, held8, tokens):
    """Slots in order, in runs from anywhere, at random, named twice, outside the cache; rows with room between them."""
    rng = np.random.default_rng(tokens + D)
    pages = 9
    N = pages * page
    if held8:
        k, v, ks, vs = make_cache8(rng, (pages, hkv, page, D), dtype)
        with np.errstate(over="ignore"):                                 # 448 2^8 is more than float16 has: rows are of the type
            kx, vx = (ref.rounded(x, dtype) for x in ref8.pages_held(k, v, ks, vs))
    else:
        k, v = ref.to_bits(rng.standard_normal((pages, hkv, page, D)), dtype), ref.to_bits(rng.standard_normal((pages, hkv, D, page)), dtype)
        kx, vx = ref.from_bits(k, dtype), ref.from_bits(v, dtype)
    kt, ke = rng.random(N).astype(np.float32), rng.integers(-1, 99, N).astype(np.int32)
    at = "uint8" if held8 else dtype
    cache = PagedCache(dev(k, at), dev(v, at), dev(kt), dev(ke), *((dev(ks), dev(vs)) if held8 else ()))
    r = Reader(hkv, hkv, D, dtype, page)
    runs = (rng.integers(0, N, -(-tokens // 11))[:, None] + np.arange(11)).reshape(-1)[:tokens] % N
    for slots in (np.arange(tokens) % N + (3 if tokens < 60 else 0), runs, rng.integers(0, N, tokens), np.full(tokens, N - 1)):
        slots = np.array(slots, np.int64)
        bad = rng.random(tokens) < 0.15
        slots[bad] = rng.choice([-1, N, -2 ** 40, 2 ** 40], bad.sum())
        bad = (slots < 0) | (slots >= N)
        rows = [dev(ref.to_bits(np.full((tokens, hkv + 1, D), 77.0), dtype), dtype) for _ in range(2)]
        views = [View(x, (tokens, hkv, D), ((hkv + 1) * D, D, 1)) for x in rows]
        t, e = dev(np.full(tokens, -7, np.float32)), dev(np.full(tokens, -7, np.int32))
        r.load(cache, dev(slots), *views, times=t, episodes=e)
        s = np.where(bad, 0, slots)
        for x, want in zip(rows, (kx[s // page, :, s % page], vx[s // page, :, :, s % page])):
            got = ref.from_bits(x.numpy(), dtype)
            np.testing.assert_array_equal(got[:, :hkv], np.where(bad[:, None, None], 77.0, want))
            assert np.all(got[:, hkv] == 77.0)
        np.testing.assert_array_equal(t.numpy(), np.where(bad, np.float32(-7), kt[s]))
        np.testing.assert_array_equal(e.numpy(), np.where(bad, -7, ke[s]))
    t2 = dev(np.full(tokens, -7, np.float32))                            # times alone
    r.load(cache, dev(slots), times=t2)
    np.testing.assert_array_equal(t2.numpy(), t.numpy())


def test_load_special_values():
    """Every byte under exponents at the ends of the types: rounded to the type where it has no such value; NaN; bytes 0 and 255."""
    for dtype in ("float16", "bfloat16"):
        k = np.tile(np.arange(256, dtype=np.uint8).reshape(1, 4, 1, 64), (1, 1, 16, 1))
        e = np.array([0, 1, 10, 60, 100, 112, 119, 127, 130, 135, 136, 140, 200, 247, 254, 255], np.uint8)
        ks = np.tile(e[None, None], (1, 4, 1))
        v = np.ascontiguousarray(k.transpose(0, 1, 3, 2))
        cache = PagedCache(dev(k), dev(v), k_scales=dev(ks), v_scales=dev(ks))
        kk, vv = (DeviceArray((16, 4, 64), dtype) for _ in range(2))
        Reader(4, 4, 64, dtype, 16).load(cache, dev(np.arange(16)), kk, vv)
        want = ref8.held(k[0], ks[0][..., None]).transpose(1, 0, 2)
        with np.errstate(over="ignore"):
            want = ref.rounded(want, dtype)
        for got in (kk, vv):
            g = ref.from_bits(got.numpy(), dtype)
            sure = np.isnan(want) | (np.abs(want) < 6e4) if dtype == "float16" else np.isnan(want) | (np.abs(want) < 1e38)
            np.testing.assert_array_equal(g[sure & (np.abs(np.nan_to_num(want)) >= 2.0 ** -120)], want[sure & (np.abs(np.nan_to_num(want)) >= 2.0 ** -120)])
            np.testing.assert_array_equal(np.isnan(g), np.isnan(want))


def test_moved_tokens():
    """Tokens read back from 8 bits and stored anew at other places and in a 16-bit cache: rotations add up."""
    rng = np.random.default_rng(3)
    T, h, D, page, dtype = 130, 2, 64, 16, "float16"
    r = Reader(h, h, D, dtype, page, rope_dim=D)
    x = ref.to_bits(rng.standard_normal((T, h, D)), dtype)
    k8 = PagedCache(DeviceArray((12, h, page, D), "uint8"), DeviceArray((12, h, D, page), "uint8"), k_scales=DeviceArray((12, h, page), "uint8"),
                    v_scales=DeviceArray((12, h, page), "uint8"))
    k16 = PagedCache(DeviceArray((12, h, page, D), dtype), DeviceArray((12, h, D, page), dtype))
    slots = rng.permutation(12 * page)[:T].astype(np.int64)
    p0 = rng.integers(0, 5000, T).astype(np.int32)
    r.store(k8, None, dev(x), dev(x), dev(p0), dev(slots))
    kk, vv = (DeviceArray((T, h, D), dtype) for _ in range(2))
    r.load(k8, dev(slots), kk, vv)
    move = np.full(T, -777, np.int32)
    r.store(k16, None, kk, vv, dev(move), dev(slots))
    k2, v2 = (DeviceArray((T, h, D), dtype) for _ in range(2))
    r.load(k16, dev(slots), k2, v2)
    held = kk.numpy().astype(np.float64)
    want, size = ref.rotate(held, move[None], 1e4, D, (D // 2,), False)
    assert np.all(np.abs(k2.numpy() - want) <= ref.U[dtype] * np.abs(want) + 2.0 ** -19 * size + 2.0 ** -25)
    np.testing.assert_array_equal(v2.numpy(), vv.numpy())
    there, size = ref.rotate(ref.from_bits(x, dtype), (p0 + move)[None], 1e4, D, (D // 2,), False)
    # the whole way: e4m3's rounding of both of a pair (2^-4 each, and the subnormals'), then float16's
    assert np.all(np.abs(k2.numpy() - there) <= (2.0 ** -4 + 2.0 ** -10) * size + 2.0 ** -9)


# ---- attend ---------------------------------------------------------------------------
def quantise(kbits, vbits, dtype):
    """A cache of 16 bits as one of 8: bytes, exponents, and the 64-bit pages that it stands for."""
    k, ks = ref8.hold(ref.from_bits(kbits, dtype), dtype)
    v, vs = ref8.hold(ref.from_bits(vbits, dtype).transpose(0, 1, 3, 2), dtype)
    v = np.ascontiguousarray(v.transpose(0, 1, 3, 2))
    return (k, v, ks, vs), ref8.pages_held(k, v, ks, vs)


def poison8(table, lens, c, page):
    """NaN and exponents of any kind in every slot that holds no token."""
    k, v, ks, vs = c
    hit = np.zeros((k.shape[0], page), bool)
    for r, n in enumerate(lens):
        j = np.arange(n)
        hit[table[r][j // page], j % page] = True
    for pg, off in zip(*np.nonzero(~hit)):
        k[pg, :, off] = 0x7F
        v[pg, :, :, off] = (0x7F, 0xFF, 0x7E)[(pg + off) % 3]
        ks[pg, :, off] = vs[pg, :, off] = (255, 254, 0)[(pg + off) % 3]


def widened(table, page, hkv, D):
    """The table with room for 128 MiB of 8-bit slots, as a server's rows have: only then prefixes are read apart. Garbage in what no row uses."""
    width = max(table.shape[1], -(-(128 << 20) // (len(table) * page * hkv * D * 2)))
    return np.concatenate([table, np.full((len(table), width - table.shape[1]), 10 ** 6, np.int32)], 1)


def check(r, dtype, q, cache, pages, q_start, lens, table, max_new=(0,), groups=None, stream=0, wide=True, **opt):
    """One call, twice for each max_new (the same bits), held to the restatement over 64-bit pages."""
    T, hq, D = q.shape
    kt, ke = opt.pop("k_times", None), opt.pop("k_eps", None)
    if len(cache) == 4:
        c = PagedCache(dev(cache[0]), dev(cache[1]), None if kt is None else dev(kt), None if ke is None else dev(ke), dev(cache[2]), dev(cache[3]))
    else:
        c = PagedCache(dev(cache[0], dtype), dev(cache[1], dtype), None if kt is None else dev(kt), None if ke is None else dev(ke))
    d = {n: (dev(opt[s]) if opt.get(s) is not None else None)
         for n, s in (("decay", "decay"), ("q_times", "q_times"), ("q_episodes", "q_eps"), ("prefix_lens", "prefix"))}
    if groups:
        d.update(group_start=dev(np.asarray(groups[0], np.int32)), shared_lens=dev(np.asarray(groups[1], np.int32)))
    want, wlse, tol, ltol = ref.attend(ref.from_bits(q, dtype), *pages, q_start, lens, table, dtype, k_times=kt, k_eps=ke, **opt)
    owned = np.isin(np.arange(T), np.concatenate([np.arange(a, b) for a, b in zip(q_start[:-1], q_start[1:])] or [[]]))
    if groups and wide:
        table = widened(table, r.page_size, r.kv_heads, D)
    for m in max_new:
        bits = None
        for _ in range(2):
            out = dev(ref.to_bits(np.full((T, hq, D), 77.0), dtype), dtype)
            lse = dev(np.full((T, hq), 77.0, np.float32))
            r.attend(c, dev(q, dtype), out, dev(np.asarray(q_start, np.int32)), dev(np.asarray(lens, np.int32)), dev(table), lse=lse,
                     scale=opt.get("scale") or 0.0, cap=opt.get("cap", 0.0), max_new=m, stream=stream, **d)
            gb, gl = out.numpy(), lse.numpy()
            got = ref.from_bits(gb, dtype)
            assert np.all(got[~owned] == 77.0) and np.all(gl[~owned] == 77.0)
            assert np.array_equal(np.isnan(got[owned]), np.isnan(want[owned]))
            fine = np.isfinite(want) & owned[:, None, None]
            with np.errstate(invalid="ignore"):
                err = np.abs(got - want) - tol
                lerr = np.abs(gl - wlse) - ltol
            assert np.all(err[fine] <= 0), (m, float(np.max(err[fine])), np.argwhere((err > 0) & fine)[:5])
            lf = np.isfinite(wlse) & owned[:, None]
            assert np.all(lerr[lf] <= 0), float(np.max(lerr[lf]))
            odd = ~np.isfinite(wlse) & owned[:, None]
            assert np.array_equal(gl[odd], wlse[odd].astype(np.float32), equal_nan=True)
            if bits is not None:
                np.testing.assert_array_equal(gb.view(np.uint16), bits[0].view(np.uint16))
                np.testing.assert_array_equal(gl.view(np.uint32), bits[1].view(np.uint32))
            bits = (gb, gl)
    return got


@pytest.mark.parametrize("which", ["", "cap decay", "decay", "episode prefix", "cap decay episode prefix"])
@pytest.mark.parametrize("hq,hkv,D,dtype,page", LAYOUTS)
def test_attend_single_tokens(hq, hkv, D, dtype, page, which):
    """One new token a request; one request without any, one whose first token it is, lengths around pages and steps."""
    rng = np.random.default_rng(hq + D)
    lens = [1, 15, 16, 17, 33, 0, 63, 64, 65, 127, 128, 129, 300, 1000]
    new = [0 if n == 0 else 1 for n in lens]
    q_start = np.concatenate([[0], np.cumsum(new)])
    table, k, v = make_cache(rng, lens, hkv, D, dtype, page)
    c, pages = quantise(k, v, dtype)
    poison8(table, lens, c, page)
    T = int(q_start[-1])
    q = ref.to_bits(rng.standard_normal((T, hq, D)), dtype)
    check(Reader(hq, hkv, D, dtype, page), dtype, q, c, pages, q_start, lens, table, max_new=(0, 1),
          **options(rng, which, T, hq, k.shape[0] * page, len(lens)))


@pytest.mark.parametrize("which", ["", "cap decay", "decay", "episode prefix", "cap decay episode prefix"])
@pytest.mark.parametrize("hq,hkv,D,dtype,page", LAYOUTS)
def test_attend_chunks(hq, hkv, D, dtype, page, which):
    """Chunks of new tokens of many lengths beside single tokens, with and without tokens cached before."""
    rng = np.random.default_rng(hq * D)
    new = [5, 1, 33, 0, 64, 97, 1, 140]
    lens = [5, 44, 40, 9, 64, 300, 1, 141]
    q_start = np.concatenate([[0], np.cumsum(new)])
    table, k, v = make_cache(rng, lens, hkv, D, dtype, page)
    c, pages = quantise(k, v, dtype)
    poison8(table, lens, c, page)
    T = int(q_start[-1]) + 3                             # rows that no request owns
    q = ref.to_bits(rng.standard_normal((T, hq, D)), dtype)
    check(Reader(hq, hkv, D, dtype, page), dtype, q, c, pages, q_start, lens, table, max_new=(0, 140, 1),
          **options(rng, which, T, hq, k.shape[0] * page, len(lens)))


@pytest.mark.parametrize("n,length", [(1, 4099), (1, 20_001), (4, 9_000), (13, 5_000), (70, 6_007), (200, 3_333)])
@pytest.mark.parametrize("hq,hkv,D,dtype,page", [(8, 2, 128, "bfloat16", 64), (6, 6, 64, "float16", 16), (2, 1, 256, "float16", 32)])
def test_attend_long(n, length, hq, hkv, D, dtype, page):
    """Few rows over many keys, split over workgroups and joined; heads whose sizes differ by octaves from token to token."""
    rng = np.random.default_rng(n)
    table, k, v = make_cache(rng, [length], hkv, D, dtype, page)
    s = [2.0 ** rng.integers(-3, 3, (k.shape[0], hkv, page)) for _ in range(2)]
    c, pages = quantise(ref.to_bits(ref.from_bits(k, dtype) * s[0][..., None], dtype), ref.to_bits(ref.from_bits(v, dtype) * s[1][:, :, None], dtype), dtype)
    q = ref.to_bits(rng.standard_normal((n, hq, D)), dtype)
    check(Reader(hq, hkv, D, dtype, page), dtype, q, c, pages, [0, n], [length], table, max_new=(0, n))


@pytest.mark.parametrize("requests,spread", [(3, 0), (40, 400), (200, 37), (450, 150), (600, 300)])
def test_attend_spans(requests, spread):
    """Lengths dealt out to workgroups: pieces that begin and end inside requests, at their edges, and requests too short to cut."""
    rng = np.random.default_rng(requests)
    hq, hkv, D, page, dtype = 2, 1, 64, 16, "bfloat16"
    L = 2_600
    one, k, v = make_cache(rng, [L], hkv, D, dtype, page)
    lens = [int(x) for x in np.clip(rng.integers(0, spread + 1, requests) * rng.integers(0, 12, requests) + (L if requests == 3 else 0), 0, L)]
    table = np.repeat(one, requests, 0)
    c, pages = quantise(k, v, dtype)
    q = ref.to_bits(rng.standard_normal((requests, hq, D)), dtype)
    check(Reader(hq, hkv, D, dtype, page), dtype, q, c, pages, np.arange(requests + 1), lens, table, max_new=(0, 1))


@pytest.mark.parametrize("n,requests", [(1, 300), (20, 96), (40, 300)])
def test_attend_long_lists(n, requests):
    """Requests over one long context, each within an episode of its own: lists of steps longer than a window."""
    rng = np.random.default_rng(n)
    L, hq, hkv, D, page, dtype = (8_900 if n == 20 else 700), 4, 4, 64, 16, "float16"
    one, k, v = make_cache(rng, [L], hkv, D, dtype, page)
    table = np.repeat(one, requests, 0)
    k_eps = np.full(k.shape[0] * page, -9, np.int32)
    j = np.arange(L)
    k_eps[table[0][j // page] * page + j % page] = np.where(j < 30, -1, j // 50)
    q_eps = np.repeat(rng.integers(-1, L // 50, requests), n).astype(np.int32)
    q_eps[0] = L // 50 - 1
    c, pages = quantise(k, v, dtype)
    q = ref.to_bits(rng.standard_normal((n * requests, hq, D)), dtype)
    opt = dict(q_eps=q_eps, k_eps=k_eps)
    r = Reader(hq, hkv, D, dtype, page)
    check(r, dtype, q, c, pages, np.arange(requests + 1) * n, [L] * requests, table, max_new=(0, n), **opt)
    shared = (L - n) // page * page                      # and the context as a prefix that all have in common
    check(r, dtype, q, c, pages, np.arange(requests + 1) * n, [L] * requests, table, max_new=(n,), groups=([0, requests], [shared]), **opt)


@pytest.mark.parametrize("n", [1, 40])
def test_attend_rows_that_see_nothing(n):
    rng = np.random.default_rng(2)
    lens, new = [0, 200, 90], [n, n, n]
    q_start = np.concatenate([[0], np.cumsum(new)])
    table, k, v = make_cache(rng, lens, 2, 64, "float16", 16)
    c, pages = quantise(k, v, "float16")
    poison8(table, lens, c, 16)
    q = ref.to_bits(rng.standard_normal((3 * n, 4, 64)), "float16")
    q_eps = np.repeat(np.array([1, 2, 55], np.int32), n)                 # 55: no key has it
    out = check(Reader(4, 2, 64, "float16", 16), "float16", q, c, pages, q_start, lens, table, max_new=(0, n), q_eps=q_eps,
                k_eps=np.full(k.shape[0] * 16, 2, np.int32))
    assert not out[:n].any() and not out[2 * n:].any()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n", [3, 50, 150])
def test_attend_nan(n, dtype):
    """NaN in keys and values reach the rows that see them and no other, keys split and not, through prefixes and not."""
    rng = np.random.default_rng(n)
    for L in (150 + n, 3_000):
        hq, hkv, D, page = 4, 2, 64, 16
        table, k, v = make_cache(rng, [L], hkv, D, dtype, page)
        c, _ = quantise(k, v, dtype)
        for j, g, d in ((L - 1, 0, 5), (L - 2, 0, 63), (L - n // 2 - 1, 1, 20), (40, 1, 33)):
            c[1][table[0][j // page], g, d, j % page] = 0xFF if d == 63 else 0x7F
        c[0][table[0][(L - 1) // page], 0, (L - 1) % page, 3] = 0x7F     # a score of NaN for the last row alone
        pages = ref8.pages_held(*c)
        q = ref.to_bits(rng.standard_normal((n, hq, D)), dtype)
        k_eps, q_eps = np.full(k.shape[0] * page, 1, np.int32), np.ones(n, np.int32)
        other = table[0][0] * page + np.arange(8)                        # another episode's keys, all NaN
        k_eps[other] = 2
        c[0][table[0][0], :, :8] = 0x7F
        c[1][table[0][0], :, :, :8] = 0x7F
        pages = ref8.pages_held(*c)
        r = Reader(hq, hkv, D, dtype, page)
        for g in (None, ([0, 1], [L - n]), ([0, 1], [64])):
            check(r, dtype, q, c, pages, [0, n], [L], table, max_new=(0, n), groups=g, q_eps=q_eps, k_eps=k_eps)


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("n", [1, 40])
def test_attend_scores_of_nan(n, D, page):
    """A row of q that holds NaN, alone and through a shared prefix: that row is NaN, the others are not."""
    rng = np.random.default_rng(7 * n + D)
    for L in (n, 400 + n, 3_000):
        table, k, v = make_cache(rng, [L], 2, D, "float16", page)
        c, pages = quantise(k, v, "float16")
        q = rng.standard_normal((n, 4, D))
        q[n // 2, 1, 3] = np.nan
        q = ref.to_bits(q, "float16")
        for g in (None, ([0, 1], [L - n])):
            check(Reader(4, 2, D, "float16", page), "float16", q, c, pages, [0, n], [L], table, max_new=(0, n), groups=g)
            check(Reader(4, 2, D, "float16", page), "float16", q, (k, v), (ref.from_bits(k, "float16"), ref.from_bits(v, "float16")), [0, n], [L], table,
                  max_new=(0, n), groups=g)


# ---- shared prefixes ------------------------------------------------------------------
def make_shared(rng, groups, hkv, D, dtype, page):
    """groups: (shared tokens, [(own cached tokens, new tokens), ...]). Returns the table, lengths and a cache of 16 bits in which a group's
    requests name the same pages for the shared tokens (rounded up to pages; the rest of such a page would hold their own)."""
    lens, new, starts, shared = [], [], [0], []
    for s, members in groups:
        shared.append(s)
        for own, n in members:
            lens.append(s // page * page + own + n)
            new.append(n)
        starts.append(len(lens))
    width = max(max(-(-n // page) for n in lens), 1)
    total = sum(-(-n // page) for n in lens)
    ids = list(rng.permutation(total + 3))
    table = np.full((len(lens), width), -5, np.int32)
    for (s, members), a, b in zip(groups, starts, starts[1:]):
        common = [ids.pop() for _ in range(s // page)]
        for r in range(a, b):
            mine = -(-lens[r] // page) - len(common)
            table[r, :len(common) + mine] = common + [ids.pop() for _ in range(mine)]
    k = ref.to_bits(rng.standard_normal((total + 3, hkv, page, D)), dtype)
    v = ref.to_bits(rng.standard_normal((total + 3, hkv, D, page)), dtype)
    q_start = np.concatenate([[0], np.cumsum(new)])
    return table, k, v, q_start, lens, starts, shared


GROUPS = {"one": [(515, [(0, 1), (33, 1), (1, 1), (700, 1), (64, 1)])],
          "several": [(129, [(3, 1)]), (0, [(40, 1), (0, 5)]), (1000, [(10, 1), (0, 1), (20, 7)]), (15, [(100, 2)]), (300, [(0, 0), (5, 1)])],
          "wide": [(777, [(i % 50, 1) for i in range(40)])],
          "chunks": [(260, [(0, 70), (100, 1), (3, 140)]), (600, [(9, 1), (0, 30)])],
          "long": [(6_100, [(200, 1), (1, 3)])],
          # the prefix in pieces that the second phase joins while its own are written, and more rows than that takes in one tile
          "own": [(3_100, [(5_000, 1), (30, 2)]), (2_000, [(4_000, 12), (3, 1)])]}


@pytest.mark.parametrize("held8", [False, True])
@pytest.mark.parametrize("which", ["", "decay", "cap decay episode prefix"])
@pytest.mark.parametrize("kind,wide", [(k, True) for k in sorted(GROUPS)] + [("several", False)])
@pytest.mark.parametrize("hq,hkv,D,dtype,page", [(12, 12, 64, "float16", 16), (8, 2, 128, "bfloat16", 64), (7, 1, 128, "float16", 32), (4, 2, 256, "bfloat16", 16)])
def test_shared(hq, hkv, D, dtype, page, kind, wide, which, held8):
    rng = np.random.default_rng(hq + len(kind))
    table, k, v, q_start, lens, starts, shared = make_shared(rng, GROUPS[kind], hkv, D, dtype, page)
    T = int(q_start[-1]) + 2
    if held8:
        c, pages = quantise(k, v, dtype)
        poison8(table, lens, c, page)
    else:
        pages = (ref.from_bits(k, dtype), ref.from_bits(v, dtype))
        poison(table, lens, k, v, page, dtype)
        c = (k, v)
    q = ref.to_bits(rng.standard_normal((T, hq, D)), dtype)
    check(Reader(hq, hkv, D, dtype, page), dtype, q, c, pages, q_start, lens, table, max_new=(0, max(1, int(np.diff(q_start).max())), 1), groups=(starts, shared), wide=wide,
          **options(rng, which, T, hq, k.shape[0] * page, len(lens)))


@pytest.mark.parametrize("held8", [False, True])
def test_shared_of_every_kind(held8):
    """Requests in no group, groups without requests, prefixes longer than what a request has cached or than the table, negative ones, requests
    that were not served, starts past the requests: each request's result is the one without groups."""
    rng = np.random.default_rng(21)
    hq, hkv, D, page, dtype = 4, 2, 64, 16, "bfloat16"
    table, k, v, q_start, lens, _, _ = make_shared(rng, [(160, [(3, 1), (40, 2), (0, 1), (17, 3), (5, 1), (60, 1)])], hkv, D, dtype, page)
    lens[4] = 0                                          # not served
    q = ref.to_bits(rng.standard_normal((int(q_start[-1]), hq, D)), dtype)
    c, pages = quantise(k, v, dtype) if held8 else ((k, v), (ref.from_bits(k, dtype), ref.from_bits(v, dtype)))
    r = Reader(hq, hkv, D, dtype, page)
    for groups in (([0, 6], [160]), ([1, 3], [160]), ([0, 0, 2, 2, 6], [999, 144, 7, 100]), ([0, 6], [10 ** 9]), ([0, 6], [2 ** 31 - 1]), ([0, 6], [-5]),
                   ([0, 3, 6], [165, 31]), ([2, 5], [175]), ([0, 100], [160]), ([6, 6], [160]), ([0, 1, 2, 3, 4, 5, 6], [160] * 6)):
        check(r, dtype, q, c, pages, q_start, lens, table, max_new=(0, 3), groups=groups)


def test_shared_values_that_tables_should_not_hold():
    """Starts that fall, negative ones, pages outside the cache: nothing outside the arrays is touched and requests in no such group are as before."""
    rng = np.random.default_rng(22)
    hq, hkv, D, page, dtype = 2, 1, 64, 16, "float16"
    table, k, v, q_start, lens, _, _ = make_shared(rng, [(64, [(3, 1), (40, 2)]), (0, [(30, 20)])], hkv, D, dtype, page)
    q = ref.to_bits(rng.standard_normal((int(q_start[-1]), hq, D)), dtype)
    want, _, tol, _ = ref.attend(ref.from_bits(q, dtype), ref.from_bits(k, dtype), ref.from_bits(v, dtype), q_start, lens, table, dtype)
    r = Reader(hq, hkv, D, dtype, page)
    cache = PagedCache(dev(k, dtype), dev(v, dtype))
    table = widened(table, page, hkv, D)
    for starts, shared, bad in (([1, 0, 2], [64, 64], None), ([-7, 2], [64], None), ([2 ** 31 - 1, -2 ** 31, 2], [64, 64], None), ([0, 2], [64], [10 ** 9, -4, 3, 2 ** 31 - 1])):
        t = table.copy()
        if bad:
            t[0, :4] = bad
        for m in (0, 20, 1):
            out = dev(np.zeros(q.shape, np.float16), dtype)
            r.attend(cache, dev(q, dtype), out, dev(np.asarray(q_start, np.int32)), dev(np.asarray(lens, np.int32)), dev(t), max_new=m,
                     group_start=dev(np.array(starts, np.int32)), shared_lens=dev(np.array(shared, np.int32)))
            assert np.all((np.abs(out.numpy().astype(np.float64) - want) <= tol)[3:])


def test_shared_many_requests_and_rows():
    """More requests than a workgroup looks at together, in many groups; and more rows than the sums of a prefix are kept for."""
    rng = np.random.default_rng(23)
    hq, hkv, D, page, dtype = 2, 1, 64, 16, "float16"
    r = Reader(hq, hkv, D, dtype, page)
    table, k, v, q_start, lens, starts, shared = make_shared(
        rng, [(16 * (g % 7), [(int(rng.integers(0, 30)), int(rng.integers(0, 3))) for _ in range(1 + g % 5)]) for g in range(300)], hkv, D, dtype, page)
    pages = (ref.from_bits(k, dtype), ref.from_bits(v, dtype))
    q = ref.to_bits(rng.standard_normal((int(q_start[-1]), hq, D)), dtype)
    check(r, dtype, q, (k, v), pages, q_start, lens, table, max_new=(0, 2), groups=(starts, shared))
    table, k, v, q_start, lens, starts, shared = make_shared(rng, [(16 * (g % 3 + 1), [(g % 5, 1), (0, g % 2)]) for g in range(2048)], hkv, D, dtype, page)
    assert len(lens) == 4096                             # the most that a call takes
    q = ref.to_bits(rng.standard_normal((int(q_start[-1]), hq, D)), dtype)
    c, pages = quantise(k, v, dtype)
    check(r, dtype, q, c, pages, q_start, lens, table, max_new=(0, 1), groups=(starts, shared))
    hq = 64                                              # 600 tokens of 64 heads are more than 2^15 rows
    table, k, v, q_start, lens, starts, shared = make_shared(rng, [(96, [(5, 300), (0, 300)])], hkv, D, dtype, page)
    pages = (ref.from_bits(k, dtype), ref.from_bits(v, dtype))
    q = ref.to_bits(rng.standard_normal((600, hq, D)), dtype)
    check(Reader(hq, hkv, D, dtype, page), dtype, q, (k, v), pages, q_start, lens, table, max_new=(300,), groups=(starts, shared))
    q, q_start, lens = q[:512], [0, 212, 512], [96 + 5 + 212, 96 + 300]          # 2^15 rows: the most that are
    check(Reader(hq, hkv, D, dtype, page), dtype, q, (k, v), pages, q_start, lens, table, max_new=(300,), groups=(starts, shared))


@pytest.mark.parametrize("n,dtype", [(1, "float16"), (1, "bfloat16"), (40, "float16")])
def test_shared_scores_of_any_size(n, dtype):
    """A prefix whose scores lie far above or below those of the requests' own keys: either side's weights may all but vanish."""
    rng = np.random.default_rng(24)
    hq, hkv, D, page = 2, 1, 64, 16
    for low, high in ((0.05, 6.0), (6.0, 0.05), (4.0, 4.0)):
        table, k, v, q_start, lens, starts, shared = make_shared(rng, [(320, [(100, n), (0, n)])], hkv, D, dtype, page)
        f = np.full(k.shape[0], high)
        f[table[0, :20]] = low
        k = ref.to_bits(ref.from_bits(k, dtype) * f[:, None, None, None], dtype)
        q = ref.to_bits(rng.standard_normal((2 * n, hq, D)), dtype)
        check(Reader(hq, hkv, D, dtype, page), dtype, q, (k, v), (ref.from_bits(k, dtype), ref.from_bits(v, dtype)), q_start, lens, table, max_new=(0, n),
              groups=(starts, shared))


@pytest.mark.parametrize("held8", [False, True])
@pytest.mark.parametrize("n,own", [(1, 30), (3, 700), (40, 30), (40, 700)])
def test_shared_not_finite(n, own, held8):
    """NaN in a shared prefix's keys and values, and in a request's own, the prefix ending inside a tile, in pieces and not: they reach the rows
    that see them and no other."""
    rng = np.random.default_rng(25 + n)
    hq, hkv, D, page, dtype = 4, 2, 64, 16, "float16"
    for S in (144, 3_024):                               # 16 tokens more than steps of 32, 64
        table, k, v, q_start, lens, starts, shared = make_shared(rng, [(S, [(own, n), (0, n), (5, 1)]), (48, [(9, n)])], hkv, D, dtype, page)
        T = int(q_start[-1])
        nan = 0x7E00
        v[table[0, 2], 0, 7, 5] = nan                    # of the first group, head 0: all its rows' element 7 of query heads 0 and 1
        v[table[0, S // page - 1], 1, 20, page - 1] = nan
        v[table[1, S // page], 1, 33, 0] = nan           # the second request's own first key
        other = table[0, 3] * page + np.arange(page)     # another episode's keys, all NaN
        k[table[0, 3]] = nan
        v[table[0, 3]] = nan
        k_eps, q_eps = np.full(k.shape[0] * page, 1, np.int32), np.ones(T, np.int32)
        k_eps[other] = 2
        q = ref.to_bits(rng.standard_normal((T, hq, D)), dtype)
        c, pages = quantise(k, v, dtype) if held8 else ((k, v), (ref.from_bits(k, dtype), ref.from_bits(v, dtype)))
        check(Reader(hq, hkv, D, dtype, page), dtype, q, c, pages, q_start, lens, table, max_new=(0, n), groups=(starts, shared), q_eps=q_eps, k_eps=k_eps)
        k[table[0, 3]] = v[table[0, 3]] = 0              # without episodes, and one score of NaN
        k[table[0, 1], 1, 3, 9] = nan
        c, pages = quantise(k, v, dtype) if held8 else ((k, v), (ref.from_bits(k, dtype), ref.from_bits(v, dtype)))
        check(Reader(hq, hkv, D, dtype, page), dtype, q, c, pages, q_start, lens, table, max_new=(0, n), groups=(starts, shared))


@pytest.mark.parametrize("page", [16, 64])
def test_release_shared(page):
    """The pages behind the prefixes come back, in request order; those of the prefixes stay."""
    rng = np.random.default_rng(page)
    for R, G in ((1, 1), (7, 2), (600, 40)):
        width, cap = 9, 4096 * 9
        starts = np.sort(rng.integers(0, R + 1, G + 1)).astype(np.int32)
        shared = rng.integers(0, 5 * page, G).astype(np.int32)
        lens = rng.integers(0, 8 * page, R).astype(np.int32)
        done = rng.integers(0, 2, R).astype(np.int32)
        table = rng.permutation(R * width).reshape(R, width).astype(np.int32)
        free = np.full(cap, -1, np.int32)
        free[:5] = -7
        want, at, left = free.copy(), 5, lens.copy()
        for q in range(R):
            if not done[q]:
                continue
            left[q] = 0
            g = [x for x in range(G) if starts[x] <= q < starts[x + 1]]
            for j in range(int(shared[g[0]]) // page if g else 0, -(-int(lens[q]) // page)):
                want[at] = table[q, j]
                at += 1
        r = Reader(page_size=page)
        d_lens, d_free, d_count = dev(lens), dev(free), dev(np.array([5], np.int32))
        r.release(dev(done), d_lens, dev(table), d_free, d_count, group_start=dev(starts), shared_lens=dev(shared))
        np.testing.assert_array_equal(d_lens.numpy(), left)
        np.testing.assert_array_equal(d_free.numpy(), want)
        assert d_count.numpy()[0] == at


# ---- together -------------------------------------------------------------------------
@pytest.mark.parametrize("held8", [True, False])
def test_answers_from_one_memory(held8):
    """As a server uses them: a memory is stored once, requests begin behind it, plan, store and attend step by step (eagerly, then as a
    captured step that is replayed with eager work between), and their own pages come back."""
    hip = C.CDLL("libamdhip64.so.7")
    stream = C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    rng = np.random.default_rng(31)
    hq, hkv, D, page, dtype, R, width, pages = 8, 2, 64, 16, "float16", 5, 6_600, 120
    S, T = 200, 12                                       # the memory's tokens: 12 whole pages are shared
    r = Reader(hq, hkv, D, dtype, page, rope_dim=D)
    if held8:
        cache = PagedCache(*(DeviceArray(s, "uint8") for s in ((pages, hkv, page, D), (pages, hkv, D, page))),
                           k_scales=DeviceArray((pages, hkv, page), "uint8"), v_scales=DeviceArray((pages, hkv, page), "uint8"))
    else:
        cache = PagedCache(DeviceArray((pages, hkv, page, D), dtype), DeviceArray((pages, hkv, D, page), dtype))
    shared = S // page * page

    def up(a):
        return dev(np.asarray(a, np.int32))

    def put(a, values):
        _lib.check(_lib.lib.mars_copy_to_device(C.c_void_p(a.data_ptr()), C.c_void_p(values.ctypes.data), values.nbytes), "copy")

    # the memory, as a request of its own
    free = rng.permutation(pages).astype(np.int32)
    d_free, left = dev(free), [up([pages]), up([0])]
    row, start1, kv1, slots1, pos1 = up(np.zeros((1, width))), up([0, 0]), up([0]), DeviceArray((shared,), "int64"), DeviceArray((shared,), "int32")
    r.plan(up([shared]), up([0]), row, d_free, left[0], q_start=start1, kv_lens=kv1, slots=slots1, positions=pos1, free_count_out=left[1])
    mem = [ref.to_bits(rng.standard_normal((shared, h, D)), dtype) for h in (hkv, hkv)]
    r.store(cache, None, *(dev(m) for m in mem), pos1, slots1)
    left.reverse()
    # the requests begin with its pages
    table = dev(np.repeat(row.numpy(), R, 0))
    lens = np.full(R, shared, np.int32)
    group_start, shared_lens = up([0, R]), up([shared])
    new, cached = DeviceArray((R,), "int32"), DeviceArray((R,), "int32")
    q_start, kv, slots, pos, count = (DeviceArray((n,), d) for n, d in ((R + 1, "int32"), (R, "int32"), (T, "int64"), (T, "int32"), (1, "int32")))
    x = [DeviceArray((T, h, D), dtype) for h in (hq, hkv, hkv)]
    qr, out = DeviceArray((T, hq, D), dtype), DeviceArray((T, hq, D), dtype)
    free_now = int(left[0].numpy()[0])
    assert free_now == pages - shared // page

    def inputs(n):
        put(new, np.array(n, np.int32))
        put(cached, lens)
        put(count, np.array([free_now], np.int32))
        for a in x:
            put(a, ref.to_bits(rng.standard_normal(a.shape), dtype))

    def step():
        s = stream.value
        r.plan(new, cached, table, d_free, count, q_start=q_start, kv_lens=kv, slots=slots, positions=pos, free_count_out=left[1], stream=s)
        r.store(cache, *x, pos, slots, q_out=qr, stream=s)
        r.attend(cache, qr, out, q_start, kv, table, group_start=group_start, shared_lens=shared_lens, stream=s)

    def verify(n):
        nonlocal free_now
        assert hip.hipStreamSynchronize(stream) == 0
        if held8:
            held = ref8.pages_held(*(y.numpy() for y in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)))
        else:
            held = [y.numpy().astype(np.float64) for y in (cache.k_pages, cache.v_pages)]
        lens[:] += np.array(n, np.int32)
        assert np.array_equal(kv.numpy(), lens)
        t = sum(n)                                       # rows behind them are nobody's
        want, _, tol, _ = ref.attend(qr.numpy()[:t].astype(np.float64), *held, q_start.numpy(), lens, table.numpy(), dtype)
        assert np.all(np.abs(out.numpy().astype(np.float64)[:t] - want) <= tol)
        free_now = int(left[1].numpy()[0])

    for n in ([3, 0, 5, 1, 2], [1] * R):
        inputs(n)
        step()
        verify(n)
    graph, exe = C.c_void_p(), C.c_void_p()
    inputs([1] * R)
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    step()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
    for i, n in enumerate(([1] * R, [1, 0, 7, 1, 0], [1] * R, [2, 2, 2, 2, 2])):
        if i:
            inputs(n)
        assert hip.hipGraphLaunch(exe, stream) == 0
        verify(n)
        if i == 1:                                       # eager work between replays
            inputs([1] * R)
            step()
            verify([1] * R)
    assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0 and hip.hipStreamDestroy(stream) == 0
    # the answers end: their own pages come back, the memory's stay until it is released itself
    d_lens, d_count = dev(lens), up([free_now])
    r.release(up([1] * R), d_lens, table, d_free, d_count, group_start, shared_lens)
    assert d_count.numpy()[0] == pages - shared // page and not d_lens.numpy().any()
    r.release(up([1]), kv1, row, d_free, d_count)
    assert np.array_equal(np.sort(d_free.numpy()), np.arange(pages))
