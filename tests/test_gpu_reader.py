"""The reading path on the GPU (mars_kv_plan, store, attend, release) against its 64-bit restatement: every head layout,
page size and type; requests without tokens, of one token, of chunks that end inside pages and tiles; empty rows; NaN
where no row looks; strides, streams and offsets past 32 bits."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import mars_amd
import reader_ref as ref
from mars_amd import _lib
from mars_amd.reader import DeviceArray, PagedCache, Reader

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    mars_amd.init(0)


def dev(a, dtype=None):
    return DeviceArray.from_numpy(a, dtype)


# ---- plan ---------------------------------------------------------------------------
def run_plan(new, cached, width, page, free_count, extra_tokens=0, missing_tokens=0, seed=0):
    rng = np.random.default_rng(seed)
    new, cached = np.asarray(new, np.int32), np.asarray(cached, np.int32)
    R, T = len(new), max(int(np.maximum(new, 0).sum()) + extra_tokens - missing_tokens, 0)
    ids = rng.permutation(4 * (R * width + free_count + 8)).astype(np.int32)
    table = rng.integers(10 ** 6, 2 * 10 ** 6, (R, width)).astype(np.int32)
    at = 0
    for r in range(R):
        have = min(-(-max(int(cached[r]), 0) // page), width)
        table[r, :have] = ids[at:at + have]
        at += have
    free = ids[at:at + free_count + 5]
    want = ref.plan(new, cached, table, free, free_count, T, page)
    r = Reader(page_size=page)
    d_table, q_start, kv = dev(table), dev(np.full(R + 1, -7, np.int32)), dev(np.full(R, -7, np.int32))
    slots, pos, out = dev(np.full(T, -7, np.int64)), dev(np.full(T, -7, np.int32)), dev(np.full(1, -7, np.int32))
    for _ in range(2):                                   # the same call again gives the same
        r.plan(dev(new), dev(cached), d_table, dev(free), dev(np.array([free_count], np.int32)), q_start=q_start, kv_lens=kv,
               slots=slots, positions=pos, free_count_out=out)
        for name, g, w in zip(("table", "q_start", "kv_lens", "slots", "positions"), (d_table, q_start, kv, slots, pos), want):
            np.testing.assert_array_equal(g.numpy(), w, err_msg=name)
        assert out.numpy()[0] == want[5]


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("requests", [1, 2, 63, 64, 65, 511, 513, 1025])
def test_plan(requests, page):
    rng = np.random.default_rng(requests + page)
    new = rng.integers(0, 4, requests) + (rng.random(requests) < 0.1) * rng.integers(0, 300, requests)
    cached = rng.integers(0, 5 * page, requests)
    width = int(max(-(-(cached + new) // page).max(), 1))
    run_plan(new, cached, width, page, free_count=int((-(-(cached + new) // page) - -(-cached // page)).sum()) + 3)


def test_plan_most_requests():
    rng = np.random.default_rng(3)
    run_plan(rng.integers(0, 5, 4096), rng.integers(0, 40, 4096), 3, 16, free_count=5000)


def test_plan_short_of_pages_rows_and_tokens():
    # pages run out in the middle: requests that need none are still served, later ones that need some are not
    run_plan([1, 40, 1, 17, 1, 1], [5, 0, 16, 3, 31, 32], 4, 16, free_count=4)
    run_plan([1, 40, 1], [16, 0, 15], 4, 16, free_count=0)
    # a request longer than its table row takes nothing; the ones after it do
    run_plan([1, 90, 20], [16, 0, 15], 4, 16, free_count=9)
    # more rows than tokens (padding), and fewer
    run_plan([3, 0, 20], [16, 7, 15], 4, 16, free_count=9, extra_tokens=77)
    run_plan([3, 0, 20, 1], [16, 7, 15, 0], 4, 16, free_count=9, missing_tokens=5)
    run_plan([0, 0], [0, 0], 1, 16, free_count=0)
    run_plan([-3, 2], [-5, 4], 1, 16, free_count=1)


def test_plan_long_chunks():
    run_plan([9001, 1, 12345], [0, 77, 500], 60, 256, free_count=200)
    run_plan([4095, 1, 4097], [1, 15, 0], 300, 32, free_count=400)


def test_release_and_plan_again():
    page, width, R = 16, 6, 9
    rng = np.random.default_rng(4)
    kv = np.array([0, 1, 16, 17, 90, 96, 500, 33, 5], np.int32)          # 500: longer than its row
    done = np.array([1, 1, 0, 1, 0, 1, 1, 0, 7], np.int32)
    table = rng.permutation(R * width).astype(np.int32).reshape(R, width)
    free = np.concatenate([np.arange(1000, 1004), np.full(20, -1)]).astype(np.int32)
    d = [dev(x) for x in (done, kv, table, free, np.array([4], np.int32))]
    r = Reader(page_size=page)
    r.release(*d)
    back = [x for i in range(R) if done[i] for x in table[i, :min(-(-int(kv[i]) // page), width)]]
    want = np.concatenate([free[:4], back])
    assert d[4].numpy()[0] == len(want)
    np.testing.assert_array_equal(d[3].numpy()[:len(want)], want)
    np.testing.assert_array_equal(d[1].numpy(), np.where(done != 0, 0, kv))
    np.testing.assert_array_equal(d[2].numpy(), table)
    small = dev(free[:6])                                # no room for all: the rest is dropped
    d = [dev(done), dev(kv), dev(table), small, dev(np.array([4], np.int32))]
    r.release(*d)
    assert d[4].numpy()[0] == 6
    np.testing.assert_array_equal(small.numpy(), want[:6])


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_plan_again_after_a_shortage(seed):
    """Step after step from a pool that runs out: a request that was not served keeps its tokens, positions and pages, goes on
    where it stood once others have ended, and every page is back exactly once at the end."""
    rng = np.random.default_rng(seed)
    R, page, width, pool = 6, 16, 6, 14
    r = Reader(page_size=page)
    table, free = dev(np.full((R, width), -1, np.int32)), dev(rng.permutation(pool).astype(np.int32))
    lens = [dev(np.zeros(R, np.int32)) for _ in range(2)]
    left = [dev(np.array([pool], np.int32)) for _ in range(2)]
    have, short, again = np.zeros(R, np.int64), np.zeros(R, bool), 0
    where = [{} for _ in range(R)]                       # slot of each of a request's tokens
    for step in range(40):
        new = rng.integers(0, 20, R).astype(np.int32)
        T = int(new.sum())
        q_start, kv, slots, pos = (DeviceArray((n,), d) for n, d in ((R + 1, "int32"), (R, "int32"), (T, "int64"), (T, "int32")))
        r.plan(dev(new), lens[0], table, free, left[0], q_start=q_start, kv_lens=kv, slots=slots, positions=pos, free_count_out=left[1],
               next_lens=lens[1])
        want = ref.plan(new, have.astype(np.int32), table.numpy(), free.numpy(), int(left[0].numpy()[0]), T, page)
        kv, slots, pos, start = kv.numpy(), slots.numpy(), pos.numpy(), q_start.numpy()
        np.testing.assert_array_equal(kv, want[2])
        served = (kv == have + new)
        np.testing.assert_array_equal(kv[~served], 0)
        for i in range(R):
            rows = slice(start[i], start[i + 1])
            np.testing.assert_array_equal(pos[rows], have[i] + np.arange(new[i]))
            if served[i]:
                where[i].update(zip(pos[rows].tolist(), slots[rows].tolist()))
                again += bool(short[i] and have[i] and new[i])
            else:
                assert np.all(slots[rows] == -1)
        short = ~served
        have = np.where(served, have + new, have)
        np.testing.assert_array_equal(lens[1].numpy(), have)
        now = table.numpy()
        held = [now[i, :-(-int(have[i]) // page)].tolist() for i in range(R)]
        pages = sum(held, [])
        assert len(set(pages)) == len(pages) == pool - int(left[1].numpy()[0]) and all(0 <= x < pool for x in pages)
        for i in range(R):                               # every token lies where its table row says, those of earlier steps too
            assert where[i] == {p: held[i][p // page] * page + p % page for p in range(int(have[i]))}
        lens.reverse()
        left.reverse()
        done = rng.random(R) < (0.25 if step < 39 else 2)
        r.release(dev(done.astype(np.int32)), lens[0], table, free, left[0])
        have[done] = 0
        for i in np.nonzero(done)[0]:
            where[i] = {}
        np.testing.assert_array_equal(lens[0].numpy(), have)
    assert again > 0                                     # the case that this is about did occur
    np.testing.assert_array_equal(left[0].numpy(), [pool])
    np.testing.assert_array_equal(np.sort(free.numpy()), np.arange(pool))


# ---- store --------------------------------------------------------------------------
def run_store(tokens, hq, hkv, D, dtype, page, rope, sections, adjacent=False, packed=True, interleaved=False, in_place=False, inverse=False,
              seed=0, slots=None, pages=None, big=False):
    rng = np.random.default_rng(seed)
    r = Reader(hq, hkv, D, dtype, page, rope_dim=rope, rope_theta=1e4 if D == 64 else 1e6, rope_sections=sections if rope else None,
               rope_adjacent=adjacent)
    theta = 1e4 if D == 64 else 1e6
    qkv = ref.to_bits(rng.standard_normal((tokens, hq + 2 * hkv, D)), dtype)
    pages = pages or -(-tokens // page) + 3
    if slots is None:
        slots = rng.permutation(pages)[:, None] * page + np.arange(page)[None]
        slots = slots.reshape(-1)[page // 2 + 1:][:tokens].astype(np.int64)
        slots[rng.random(tokens) < 0.1] = -1
    if rng.random() < 0.5 and tokens > 2:
        slots[0] = pages * page                          # outside the cache: stores nothing
    axes = max(len(sections), 1)
    pos = rng.integers(0, 40_000, (axes, tokens)).astype(np.int32)
    pos[0, 0] = 2 ** 31 - 1
    pos[-1, -1] = -70_001
    times, eps = rng.random(tokens).astype(np.float32) * 600, rng.integers(-1, 9, tokens).astype(np.int32)

    class View:                                          # a view of a device array at an element offset
        def __init__(self, base, shape, strides, offset=0):
            self.base, self.shape, self.dtype, self._s, self._o = base, shape, base.dtype, strides, offset

        def data_ptr(self):
            return self.base.data_ptr() + 2 * self._o

        def stride(self, i):
            return self._s[i]

    H = hq + 2 * hkv
    if packed:                                           # q, k and v of a token side by side
        x = dev(qkv, dtype)
        q, k, v = (View(x, (tokens, h, D), (H * D, D, 1), o * D) for h, o in ((hq, 0), (hkv, hq), (hkv, hq + hkv)))
    else:
        q, k, v = (dev(np.ascontiguousarray(qkv[:, a:b]), dtype) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, H)))
    before = [ref.to_bits(rng.standard_normal((pages, 2 if interleaved else 1, hkv, page * D)), dtype) for _ in range(2)]
    kb, vb = (dev(b, dtype) for b in before)
    n = hkv * page * D
    stride, layer = (2 * n, 1) if interleaved else (n, 0)
    kp = View(kb, (pages, hkv, page, D), (stride, page * D, D, 1), layer * n)
    vp = View(vb, (pages, hkv, D, page), (stride, page * D, page, 1), layer * n)
    kt, ke = dev(np.full(pages * page, -3, np.float32)), dev(np.full(pages * page, -3, np.int32))
    cache = PagedCache(kp, vp, kt, ke)
    q_out = None if in_place else dev(np.zeros((tokens, hq, D), np.uint16 if dtype == "bfloat16" else np.float16), dtype)
    r.store(cache, q, k, v, dev(pos) if rope else None, dev(slots), q_out=q_out, times=dev(times), episodes=dev(eps), inverse=inverse)

    x = ref.from_bits(qkv, dtype)
    want, size = ref.rotate(x[:, :hq + hkv], pos, theta, rope, sections, adjacent, inverse)
    u = ref.U[dtype]
    tol = u * np.abs(want) + 2.0 ** -19 * size + 2.0 ** -25
    exact = size == 0                                    # elements that do not turn are copied
    if in_place:
        got_q = ref.from_bits(x0 := (x_dev := (q.base if packed else q)).numpy(), dtype)[:, :hq]
        assert x0 is not None and x_dev is not None
    else:
        got_q = ref.from_bits(q_out.numpy(), dtype)
    assert np.all(np.abs(got_q - want[:, :hq]) <= np.where(exact, 0, tol)[:, :hq])
    ok = (slots >= 0) & (slots < pages * page)
    pg, off = slots[ok] // page, slots[ok] % page
    got_k = ref.from_bits(kb.numpy(), dtype).reshape(pages, -1, hkv, page, D)[:, layer]
    got_v = vb.numpy().reshape(pages, -1, hkv, D, page)[:, layer]
    assert np.all(np.abs(got_k[pg, :, off] - want[ok, hq:]) <= np.where(exact, 0, tol)[ok, hq:])
    np.testing.assert_array_equal(got_v[pg, :, :, off], qkv[ok, hq + hkv:])
    # nothing else is written
    hit = np.zeros((pages, page), bool)
    hit[pg, off] = True
    kw, vw = before[0].reshape(pages, -1, hkv, page, D), before[1].reshape(pages, -1, hkv, D, page)
    k_now, v_now = kb.numpy().reshape(kw.shape), vb.numpy().reshape(vw.shape)
    np.testing.assert_array_equal(np.where(hit[:, None, :, None], 0, k_now[:, layer]), np.where(hit[:, None, :, None], 0, kw[:, layer]))
    np.testing.assert_array_equal(np.where(hit[:, None, None, :], 0, v_now[:, layer]), np.where(hit[:, None, None, :], 0, vw[:, layer]))
    if interleaved:
        np.testing.assert_array_equal(k_now[:, 0], kw[:, 0])
        np.testing.assert_array_equal(v_now[:, 0], vw[:, 0])
    tw, ew = np.full(pages * page, -3, np.float32), np.full(pages * page, -3, np.int32)
    tw[slots[ok]], ew[slots[ok]] = times[ok], eps[ok]
    np.testing.assert_array_equal(kt.numpy(), tw)
    np.testing.assert_array_equal(ke.numpy(), ew)


@pytest.mark.parametrize("tokens", [1, 2, 17, 64, 130, 1029])
@pytest.mark.parametrize("hq,hkv,D,dtype,page", [(12, 12, 64, "float16", 16), (8, 2, 128, "bfloat16", 64), (3, 1, 256, "float16", 128),
                                                 (10, 5, 64, "bfloat16", 256), (7, 7, 128, "float16", 32)])
def test_store(tokens, hq, hkv, D, dtype, page):
    run_store(tokens, hq, hkv, D, dtype, page, D, (D // 8, D // 8 + 3, D // 4 - 3), seed=tokens)


@pytest.mark.parametrize("rope,sections,adjacent", [(64, (32,), False), (64, (32,), True), (32, (16,), False), (48, (4, 20, 0), True),
                                                    (16, (0, 3, 5), False), (0, (), False)])
@pytest.mark.parametrize("tokens", [5, 200])
def test_store_rotations(rope, sections, adjacent, tokens):
    run_store(tokens, 6, 3, 64, "float16", 32, rope, sections, adjacent, packed=tokens == 5, seed=rope)


@pytest.mark.parametrize("tokens", [3, 150])
def test_store_layouts(tokens):
    run_store(tokens, 4, 2, 128, "bfloat16", 64, 128, (64,), interleaved=True, seed=1)
    run_store(tokens, 4, 2, 128, "float16", 16, 128, (20, 40, 4), in_place=True, seed=2)
    run_store(tokens, 4, 2, 128, "float16", 16, 128, (64,), inverse=True, packed=False, seed=3)
    # slots in no order, one page for each token, and chunks that go on at slots that are not multiples of 8
    rng = np.random.default_rng(5)
    run_store(tokens, 2, 1, 64, "float16", 16, 64, (32,), slots=rng.permutation(tokens * 3)[:tokens].astype(np.int64), pages=-(-tokens * 3 // 16))
    run_store(tokens, 2, 1, 64, "bfloat16", 16, 64, (32,), slots=np.arange(tokens, dtype=np.int64)[::-1].copy() + 3, pages=-(-tokens // 16) + 1)


def test_store_rotation_is_a_gradient():
    """d(sum g . rotate(x)) / dx = inverse rotation of g: against the formula, and against differences of the forward call."""
    rng = np.random.default_rng(8)
    t, h, D = 3, 2, 64
    r = Reader(h, h, D, "float16", 16, rope_dim=48, rope_sections=(8, 8, 8))
    pos = rng.integers(0, 50, (3, t)).astype(np.int32)
    x, g = (ref.rounded(rng.standard_normal((t, h, D)), "float16") for _ in range(2))

    def turned(y, inverse):
        out = dev(np.zeros((t, h, D), np.float16))
        r.store(None, dev(y.astype(np.float16)), None, None, dev(pos), None, q_out=out, inverse=inverse)
        return out.numpy().astype(np.float64)

    grad = turned(g, True)
    want, size = ref.rotate(g, pos, 1e4, 48, (8, 8, 8), False, inverse=True)
    assert np.all(np.abs(grad - want) <= ref.U["float16"] * np.abs(want) + 2.0 ** -19 * size + 2.0 ** -25)
    # the map is linear, so a difference over a step of any size is exact but for the two outputs' roundings
    step, base = 4.0, turned(x, False)
    for e in rng.choice(t * h * D, 24, replace=False):
        y = x.reshape(-1).copy()
        y[e] += step
        y = ref.rounded(y, "float16")
        moved = y[e] - x.reshape(-1)[e]
        up = turned(y.reshape(x.shape), False)
        tol = 2.0 ** -11 * (np.abs(up) + np.abs(base)).reshape(-1) @ np.abs(g).reshape(-1) / abs(moved) + 1e-3
        assert abs(((up - base) * g).sum() / moved - want.reshape(-1)[e]) <= tol


# ---- attend -------------------------------------------------------------------------
def make_cache(rng, lens, hkv, D, dtype, page, spare=3, width=None):
    width = width or max(max(-(-n // page) for n in lens), 1)
    total = sum(-(-n // page) for n in lens)
    ids = rng.permutation(total + spare).astype(np.int32)
    table = np.full((len(lens), width), -5, np.int32)
    at = 0
    for r, n in enumerate(lens):
        table[r, :-(-n // page)] = ids[at:at + -(-n // page)]
        at += -(-n // page)
    k = ref.to_bits(rng.standard_normal((total + spare, hkv, page, D)), dtype)
    v = ref.to_bits(rng.standard_normal((total + spare, hkv, D, page)), dtype)
    return table, k, v


def poison(table, lens, k, v, page, dtype):
    """NaN and infinities in every slot that holds no token: spare pages and the ends of last pages."""
    held = np.zeros((k.shape[0], page), bool)
    for r, n in enumerate(lens):
        j = np.arange(n)
        held[table[r][j // page], j % page] = True
    bad = {"float16": np.array([0x7E00, 0x7C00, 0xFC00], np.uint16), "bfloat16": np.array([0x7FC0, 0x7F80, 0xFF80], np.uint16)}[dtype]
    kb, vb = k.view(np.uint16), v.view(np.uint16)
    for pg, off in zip(*np.nonzero(~held)):
        kb[pg, :, off] = bad[0]
        vb[pg, :, :, off] = bad[(pg + off) % 3]


def check_attend(r, dtype, q, kbits, vbits, q_start, lens, table, rows=None, stream=0, max_new=(0,), q_view=None, **opt):
    """One call, twice for each max_new (the same bits), held to the restatement."""
    T, hq, D = q.shape
    kt, ke = opt.pop("k_times", None), opt.pop("k_eps", None)
    cache = PagedCache(dev(kbits, dtype), dev(vbits, dtype), None if kt is None else dev(kt), None if ke is None else dev(ke))
    dq = dev(q, dtype) if q_view is None else q_view
    d = {n: (dev(opt[s]) if opt.get(s) is not None else None)
         for n, s in (("decay", "decay"), ("q_times", "q_times"), ("q_episodes", "q_eps"), ("prefix_lens", "prefix"))}
    want, wlse, tol, ltol = ref.attend(ref.from_bits(q, dtype), ref.from_bits(kbits, dtype), ref.from_bits(vbits, dtype), q_start, lens, table,
                                       dtype, k_times=kt, k_eps=ke, **opt)
    owned = ~np.isnan(wlse[:, 0]) | np.isin(np.arange(T), np.concatenate([np.arange(a, b) for a, b in zip(q_start[:-1], q_start[1:])] or [[]]))
    bits = None
    for m in max_new:
        for _ in range(2):
            out = dev(ref.to_bits(np.full((T, hq, D), 77.0), dtype), dtype)
            lse = dev(np.full((T, hq), 77.0, np.float32))
            r.attend(cache, dq, out, dev(np.asarray(q_start, np.int32)), dev(np.asarray(lens, np.int32)), dev(table), lse=lse,
                     scale=opt.get("scale") or 0.0, cap=opt.get("cap", 0.0), max_new=m, stream=stream, **d)
            gb, gl = out.numpy(), lse.numpy()
            got = ref.from_bits(gb, dtype)
            assert np.all(got[~owned] == 77.0) and np.all(gl[~owned] == 77.0)
            fine = np.isfinite(want) & owned[:, None, None]
            assert np.array_equal(np.isnan(got[owned]), np.isnan(want[owned]))
            inf = np.isinf(want) & owned[:, None, None]
            assert np.array_equal(got[inf], want[inf])
            err = np.abs(got - want) - tol
            assert np.all(err[fine] <= 0), (m, float(np.max(err[fine])), np.argwhere((err > 0) & fine)[:5])
            lf = np.isfinite(wlse)
            assert np.array_equal(gl[owned & ~lf.all(1)][~lf[owned & ~lf.all(1)]], wlse[owned & ~lf.all(1)][~lf[owned & ~lf.all(1)]], equal_nan=True)
            assert np.all(np.abs(gl - wlse)[lf] <= ltol[lf]), float(np.max((np.abs(gl - wlse) - ltol)[lf]))
            if _ == 0:
                bits = (gb, gl)
            else:
                np.testing.assert_array_equal(gb, bits[0])
                np.testing.assert_array_equal(gl.view(np.uint32), bits[1].view(np.uint32))
    return got


LAYOUTS = [(12, 12, 64, "float16", 16), (12, 4, 64, "bfloat16", 32), (8, 2, 128, "bfloat16", 64), (7, 1, 128, "float16", 16),
           (3, 1, 256, "float16", 128), (4, 2, 256, "bfloat16", 256), (20, 1, 64, "float16", 64), (40, 2, 128, "bfloat16", 16)]


def options(rng, which, T, hq, slots, requests, episodes=4):
    o = {}
    if "cap" in which:
        o["cap"] = 3.0                                   # low enough to bend scores of a few units
    if "decay" in which:
        o.update(decay=(0.01 * 2.0 ** -np.arange(hq)).astype(np.float32), q_times=rng.uniform(300, 600, T).astype(np.float32),
                 k_times=rng.uniform(0, 620, slots).astype(np.float32))
    if "episode" in which:
        o.update(q_eps=rng.integers(-1, episodes, T).astype(np.int32), k_eps=rng.integers(-1, episodes, slots).astype(np.int32))
    if "prefix" in which:
        o["prefix"] = rng.integers(0, 40, requests).astype(np.int32)
    return o


@pytest.mark.parametrize("which", ["", "cap decay", "episode prefix", "cap decay episode prefix"])
@pytest.mark.parametrize("hq,hkv,D,dtype,page", LAYOUTS)
def test_attend_single_tokens(hq, hkv, D, dtype, page, which):
    """One new token a request; one request without any, one whose first token it is, lengths around pages and steps."""
    rng = np.random.default_rng(hq + D)
    lens = [1, 15, 16, 17, 33, 0, 127, 128, 129, 300, 1000]
    new = [1, 1, 1, 1, 1, 0, 1, 1, 1, 1, 1]
    q_start = np.concatenate([[0], np.cumsum(new)])
    table, k, v = make_cache(rng, lens, hkv, D, dtype, page)
    poison(table, lens, k, v, page, dtype)
    T = int(q_start[-1])
    q = ref.to_bits(rng.standard_normal((T, hq, D)), dtype)
    check_attend(Reader(hq, hkv, D, dtype, page), dtype, q, k, v, q_start, lens, table, max_new=(0, 1),
                 **options(rng, which, T, hq, k.shape[0] * page, len(lens)))


@pytest.mark.parametrize("which", ["", "cap decay", "episode prefix", "cap decay episode prefix"])
@pytest.mark.parametrize("hq,hkv,D,dtype,page", LAYOUTS)
def test_attend_chunks(hq, hkv, D, dtype, page, which):
    """Chunks of new tokens of many lengths beside single tokens, with and without tokens cached before."""
    rng = np.random.default_rng(hq * D)
    new = [5, 1, 33, 0, 64, 97, 1, 140]
    lens = [5, 44, 40, 9, 64, 300, 1, 141]
    q_start = np.concatenate([[0], np.cumsum(new)])
    table, k, v = make_cache(rng, lens, hkv, D, dtype, page)
    poison(table, lens, k, v, page, dtype)
    T = int(q_start[-1]) + 3                             # rows that no request owns
    q = ref.to_bits(rng.standard_normal((T, hq, D)), dtype)
    check_attend(Reader(hq, hkv, D, dtype, page), dtype, q, k, v, q_start, lens, table, max_new=(0, 140, 1),
                 **options(rng, which, T, hq, k.shape[0] * page, len(lens)))


@pytest.mark.parametrize("n,length", [(1, 4099), (1, 20_001), (4, 9_000), (13, 5_000), (70, 6_007), (200, 3_333)])
@pytest.mark.parametrize("hq,hkv,D,dtype,page", [(8, 2, 128, "bfloat16", 64), (6, 6, 64, "float16", 16), (2, 1, 256, "float16", 32)])
def test_attend_long(n, length, hq, hkv, D, dtype, page):
    """Few rows over many keys: the keys split over workgroups and joined."""
    rng = np.random.default_rng(n)
    table, k, v = make_cache(rng, [length], hkv, D, dtype, page)
    q = ref.to_bits(rng.standard_normal((n, hq, D)), dtype)
    # scores that rise along the keys: the running reference moves again and again
    k = ref.to_bits(ref.from_bits(k, dtype) * 2.0, dtype)
    check_attend(Reader(hq, hkv, D, dtype, page), dtype, q, k, v, [0, n], [length], table, max_new=(0, n))


def test_attend_many_requests():
    rng = np.random.default_rng(11)
    for R in (257, 700):
        new = rng.integers(0, 3, R)
        lens = [int(n + c) for n, c in zip(new, rng.integers(0, 40, R))]
        q_start = np.concatenate([[0], np.cumsum(new)])
        table, k, v = make_cache(rng, lens, 1, 64, "float16", 16)
        q = ref.to_bits(rng.standard_normal((int(q_start[-1]), 2, 64)), "float16")
        check_attend(Reader(2, 1, 64, "float16", 16), "float16", q, k, v, q_start, lens, table, max_new=(0, 2))


@pytest.mark.parametrize("n,requests", [(1, 300), (20, 96), (40, 300)])
def test_attend_shared_pages_and_long_lists(n, requests):
    """Requests that share the pages of one long context, each within an episode of its own: lists of steps longer than a
    window, more requests than a workgroup looks at together, tiles enough that no keys are split."""
    rng = np.random.default_rng(n)
    L, hq, hkv, D, page, dtype = (8_300 if n == 20 else 700), 4, 4, 64, 16, "float16"
    one, k, v = make_cache(rng, [L], hkv, D, dtype, page)
    table = np.repeat(one, requests, 0)
    k_eps = np.full(k.shape[0] * page, -9, np.int32)
    j = np.arange(L)
    k_eps[table[0][j // page] * page + j % page] = np.where(j < 30, -1, j // 50)
    q_eps = np.repeat(rng.integers(-1, L // 50, requests), n).astype(np.int32)
    q_eps[0] = L // 50 - 1
    q = ref.to_bits(rng.standard_normal((n * requests, hq, D)), dtype)
    check_attend(Reader(hq, hkv, D, dtype, page), dtype, q, k, v, np.arange(requests + 1) * n, [L] * requests, table, max_new=(0, n),
                 q_eps=q_eps, k_eps=k_eps)


@pytest.mark.parametrize("requests,spread", [(3, 0), (40, 400), (200, 37), (600, 300)])
def test_attend_spans(requests, spread):
    """Lengths dealt out to workgroups: pieces that begin and end inside requests, at their edges, and requests too short to cut."""
    rng = np.random.default_rng(requests)
    hq, hkv, D, page, dtype = 2, 1, 64, 16, "bfloat16"
    L = 2_600
    one, k, v = make_cache(rng, [L], hkv, D, dtype, page)
    lens = [int(x) for x in np.clip(rng.integers(0, spread + 1, requests) * rng.integers(0, 12, requests) + (L if requests == 3 else 0), 0, L)]
    table = np.repeat(one, requests, 0)
    q = ref.to_bits(rng.standard_normal((requests, hq, D)), dtype)
    check_attend(Reader(hq, hkv, D, dtype, page), dtype, q, k, v, np.arange(requests + 1), lens, table, max_new=(1,),
                 decay=np.full(hq, 0.01, np.float32), q_times=np.full(requests, 600, np.float32),
                 k_times=rng.uniform(0, 600, k.shape[0] * page).astype(np.float32))
    check_attend(Reader(hq, hkv, D, dtype, page), dtype, q, k, v, np.arange(requests + 1), lens, table, max_new=(0, 1))


@pytest.mark.parametrize("n", [1, 40])
def test_attend_rows_that_see_nothing(n):
    """Requests that were not served (kv_lens 0), episodes without a token, ages that leave no weight: rows of zeros, lse -inf."""
    rng = np.random.default_rng(2)
    lens, new = [0, 200, 90], [n, n, n]
    q_start = np.concatenate([[0], np.cumsum(new)])
    table, k, v = make_cache(rng, lens, 2, 64, "float16", 16)
    poison(table, lens, k, v, 16, "float16")
    q = ref.to_bits(rng.standard_normal((3 * n, 4, 64)), "float16")
    q_eps = np.repeat(np.array([1, 2, 55], np.int32), n)                 # 55: no key has it
    k_eps = np.full(k.shape[0] * 16, 2, np.int32)
    out = check_attend(Reader(4, 2, 64, "float16", 16), "float16", q, k, v, q_start, lens, table, max_new=(0, n), q_eps=q_eps, k_eps=k_eps)
    assert not out[:n].any() and not out[2 * n:].any() and out[n:2 * n].any()
    # a key stamped -inf is infinitely old: no weight, in a row of such keys none at all
    kt = np.full(k.shape[0] * 16, -np.inf, np.float32)
    out = check_attend(Reader(4, 2, 64, "float16", 16), "float16", q, k, v, q_start, lens, table, max_new=(0, n),
                       decay=np.full(4, 0.5, np.float32), q_times=np.full(3 * n, 600, np.float32), k_times=kt)
    assert not out.any()
    kt[rng.random(kt.size) < 0.5] = 590.0
    check_attend(Reader(4, 2, 64, "float16", 16), "float16", q, k, v, q_start, lens, table, max_new=(0, n),
                 decay=np.full(4, 0.5, np.float32), q_times=np.full(3 * n, 600, np.float32), k_times=kt)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n", [3, 50, 150])
def test_attend_not_finite_values(n, dtype):
    """Infinities and NaN in keys and values reach the rows that see them and no other."""
    rng = np.random.default_rng(n)
    L, hq, hkv, D, page = 150 + n, 4, 2, 64, 16
    table, k, v = make_cache(rng, [L], hkv, D, dtype, page)
    nan, pinf, ninf = {"float16": (0x7E00, 0x7C00, 0xFC00), "bfloat16": (0x7FC0, 0x7F80, 0xFF80)}[dtype]
    kb, vb = k.view(np.uint16), v.view(np.uint16)
    for j, g, d, x in ((L - 1, 0, 5, nan), (L - 1, 1, 6, pinf), (L - 2, 0, 63, ninf), (L - 2, 0, 0, pinf), (L - 1, 0, 0, ninf), (L - n // 2 - 1, 1, 20, nan)):
        vb[table[0][j // page], g, d, j % page] = x
    kb[table[0][(L - 1) // page], 0, (L - 1) % page, 3] = nan            # a score of NaN for the last row alone
    q = ref.to_bits(rng.standard_normal((n, hq, D)), dtype)
    k_eps, q_eps = np.full(k.shape[0] * page, 1, np.int32), np.ones(n, np.int32)
    other = table[0][0] * page + np.arange(8)                            # another episode's keys, all NaN
    k_eps[other] = 2
    kb[table[0][0], :, :8] = nan
    vb[table[0][0], :, :, :8] = nan
    check_attend(Reader(hq, hkv, D, dtype, page), dtype, q, k, v, [0, n], [L], table, max_new=(0, n), q_eps=q_eps, k_eps=k_eps)


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("n", [1, 40])
def test_attend_not_finite_values_that_all_rows_see(n, D, page):
    """Infinities and NaN in the middle of what every row sees, keys split and not."""
    rng = np.random.default_rng(n + D)
    for L in (400 + n, 3_000):
        table, k, v = make_cache(rng, [L], 2, D, "float16", page)
        vb = v.view(np.uint16)
        for j, g, d, x in ((70, 0, 5, 0x7C00), (71, 0, 6, 0xFC00), (200, 1, 7, 0x7E00), (201, 1, 9, 0x7C00), (300, 1, 9, 0xFC00), (330, 0, 5, 0x7C00)):
            vb[table[0][j // page], g, d, j % page] = x
        q = ref.to_bits(rng.standard_normal((n, 4, D)), "float16")
        check_attend(Reader(4, 2, D, "float16", page), "float16", q, k, v, [0, n], [L], table, max_new=(0, n))


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("n", [1, 40])
def test_attend_scores_that_are_not_numbers(n, D, page):
    """A row of q that holds NaN, and NaN in the only key that a row sees: the row is NaN, the others are not."""
    rng = np.random.default_rng(7 * n + D)
    for L in (n, 400 + n, 3_000):
        table, k, v = make_cache(rng, [L], 2, D, "float16", page)
        q = rng.standard_normal((n, 4, D))
        q[n // 2, 1, 3] = np.nan
        q = ref.to_bits(q, "float16")
        check_attend(Reader(4, 2, D, "float16", page), "float16", q, k, v, [0, n], [L], table, max_new=(0, n))
    table, k, v = make_cache(rng, [n], 2, D, "float16", page)
    k.view(np.uint16)[table[0][0], 1, 0, 5] = 0x7E00
    check_attend(Reader(4, 2, D, "float16", page), "float16", ref.to_bits(rng.standard_normal((n, 4, D)), "float16"), k, v, [0, n], [n], table,
                 max_new=(0, n))


def test_attend_scores_of_any_size():
    """Scores far from zero: rows whose largest score is very low, very high, and rising by more than the weights' range."""
    rng = np.random.default_rng(6)
    L, D = 700, 64
    table, k, v = make_cache(rng, [L, L], 1, D, "bfloat16", 16)
    q = ref.to_bits(rng.standard_normal((2, 2, D)), "bfloat16")
    for scale in (-40.0, 1e-6, 30.0, 1e30):
        kk = ref.to_bits(np.sign(ref.from_bits(k, "bfloat16")), "bfloat16") if scale == 1e30 else k
        qq = ref.to_bits(np.sign(ref.from_bits(q, "bfloat16")) * np.arange(1, 3)[:, None, None], "bfloat16") if scale == 1e30 else q
        check_attend(Reader(2, 1, D, "bfloat16", 16), "bfloat16", qq, kk, v, [0, 1, 2], [L, L], table, max_new=(0, 1), scale=scale)


def test_attend_strides():
    """q as a part of a packed projection, out with room between tokens, the cache's layers interleaved."""
    rng = np.random.default_rng(9)
    hq, hkv, D, page, dtype = 4, 2, 128, 32, "float16"
    lens, new = [90, 41], [37, 2]
    table, k, v = make_cache(rng, lens, hkv, D, dtype, page)
    T = 39
    packed = ref.to_bits(rng.standard_normal((T, hq + 2 * hkv + 1, D)), dtype)
    want, _, tol, _ = ref.attend(ref.from_bits(packed[:, 1:1 + hq], dtype), ref.from_bits(k, dtype), ref.from_bits(v, dtype), [0, 37, 39], lens, table, dtype)
    layers = 3
    kl, vl = (ref.to_bits(rng.standard_normal((x.shape[0], layers) + x.shape[1:]), dtype) for x in (k, v))
    kl[:, 2], vl[:, 2] = k, v
    dk, dv, dq = dev(kl, dtype), dev(vl, dtype), dev(packed, dtype)
    out = dev(np.full((T, hq + 5, D), 9.0, np.float16), dtype)
    start, lens_d, table_d = dev(np.array([0, 37, 39], np.int32)), dev(np.array(lens, np.int32)), dev(table)
    n = hkv * page * D
    r = Reader(hq, hkv, D, dtype, page)
    c = _lib.KvCacheC(dk.data_ptr() + 2 * 2 * n, dv.data_ptr() + 2 * 2 * n, None, None, layers * n, layers * n, k.shape[0], 0)
    a = _lib.KvAttendArgsC(q=dq.data_ptr() + 2 * D, out=out.data_ptr() + 2 * 2 * D, q_start=start.data_ptr(), kv_lens=lens_d.data_ptr(),
                           block_table=table_d.data_ptr(), q_stride=(hq + 2 * hkv + 1) * D, out_stride=(hq + 5) * D, num_requests=2,
                           max_pages=table.shape[1], num_tokens=T)
    _lib.check(_lib.lib.mars_kv_attend(r.handle, C.byref(c), C.byref(a), None), "mars_kv_attend")
    got = out.numpy().astype(np.float64)
    assert np.all(np.abs(got[:, 2:2 + hq] - want) <= tol)
    assert np.all(got[:, :2] == 9.0) and np.all(got[:, 2 + hq:] == 9.0)


def test_offsets_past_32_bits():
    """Pages whose elements lie past 2^31, and bytes past 2^32: stored there, read from there."""
    hq, hkv, D, page, dtype = 4, 2, 128, 256, "float16"
    n = hkv * page * D
    pages = 2 ** 31 // n + 40
    kb, vb = (DeviceArray((pages, hkv, page, D), dtype) for _ in range(2))
    cache = PagedCache(kb, _As(vb, (pages, hkv, D, page)))
    rng = np.random.default_rng(12)
    L = 700
    table = np.array([[pages - 1, 2, pages - 17]], np.int32)
    j = np.arange(L)
    slots = table[0][j // page].astype(np.int64) * page + j % page
    assert slots.max() * hkv * D > 2 ** 31
    x = ref.to_bits(rng.standard_normal((L, hq + 2 * hkv, D)), dtype)
    r = Reader(hq, hkv, D, dtype, page)
    q = dev(np.ascontiguousarray(x[-40:, :hq]), dtype)
    r.store(cache, None, dev(np.ascontiguousarray(x[:, hq:hq + hkv]), dtype), dev(np.ascontiguousarray(x[:, hq + hkv:]), dtype), None, dev(slots))
    small = [ref.from_bits(x[:, hq + i * hkv:hq + (i + 1) * hkv], dtype) for i in range(2)]
    pad = np.zeros((3 * page, hkv, D))
    pad[:L] = small[0]
    kp = pad.reshape(3, page, hkv, D).transpose(0, 2, 1, 3)
    pad = np.zeros((3 * page, hkv, D))
    pad[:L] = small[1]
    vp = pad.reshape(3, page, hkv, D).transpose(0, 2, 3, 1)
    want, _, tol, _ = ref.attend(ref.from_bits(x[-40:, :hq], dtype), kp, vp, [0, 40], [L], np.array([[0, 1, 2]]), dtype)
    for m in (0, 1):
        out = DeviceArray((40, hq, D), dtype)
        r.attend(cache, q, out, dev(np.array([0, 40], np.int32)), dev(np.array([L], np.int32)), dev(table), max_new=m)
        assert np.all(np.abs(out.numpy().astype(np.float64) - want) <= tol)


class _As:
    """A device array under another dense shape."""

    def __init__(self, base, shape):
        self.base, self.shape, self.dtype = base, shape, base.dtype
        self._s = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]

    def data_ptr(self):
        return self.base.data_ptr()

    def stride(self, i):
        return self._s[i]


def test_values_that_a_table_should_not_hold():
    """Pages outside the cache, lengths past the table, negative ones: nothing outside the arrays is touched, other requests are as before."""
    rng = np.random.default_rng(13)
    hq, hkv, D, page, dtype = 2, 1, 64, 16, "float16"
    lens, new = [60, 50], [2, 30]
    table, k, v = make_cache(rng, lens, hkv, D, dtype, page)
    q = ref.to_bits(rng.standard_normal((32, hq, D)), dtype)
    want, _, tol, _ = ref.attend(ref.from_bits(q, dtype), ref.from_bits(k, dtype), ref.from_bits(v, dtype), [0, 2, 32], lens, table, dtype)
    r = Reader(hq, hkv, D, dtype, page)
    cache = PagedCache(dev(k, dtype), dev(v, dtype))
    for bad_table, bad_lens, bad_start, good in (([10 ** 9, -4, 2 ** 31 - 1, -2 ** 31], [60, 50], [0, 2, 32], slice(2, 32)),
                                                 (table[0], [10 ** 9, 50], [0, 2, 32], slice(2, 32)),
                                                 (table[0], [-9, 50], [0, 2, 32], slice(2, 32)),
                                                 (table[0], [60, 50], [0, 2, 10 ** 9], slice(0, 2)),
                                                 (table[0], [60, 50], [-50, 2, 32], slice(2, 32))):
        t = table.copy()
        t[0] = bad_table
        for m in (0, 30, 1):
            out = dev(np.zeros((32, hq, D), np.float16), dtype)
            r.attend(cache, dev(q, dtype), out, dev(np.array(bad_start, np.int32)), dev(np.array(bad_lens, np.int32)), dev(t), max_new=m)
            got = out.numpy().astype(np.float64)
            assert np.all(np.abs(got - want)[good] <= tol[good])


def test_another_stream_and_a_graph():
    """Plan, store and attend on a stream of the caller's, then captured and replayed with new lengths and inputs and eager work between."""
    hip = C.CDLL("libamdhip64.so.7")
    stream = C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    rng = np.random.default_rng(14)
    hq, hkv, D, page, dtype, R, T = 4, 2, 64, 16, "float16", 3, 8
    width, pages = 20, 70
    r = Reader(hq, hkv, D, dtype, page, rope_dim=64)
    kz, vz = np.zeros((pages, hkv, page, D), np.float16), np.zeros((pages, hkv, D, page), np.float16)
    cache = PagedCache(dev(kz), dev(vz))
    free = dev(rng.permutation(pages).astype(np.int32))
    table = dev(np.zeros((R, width), np.int32))
    new, cached, count = DeviceArray((R,), "int32"), DeviceArray((R,), "int32"), DeviceArray((1,), "int32")
    q_start, kv, slots, pos, left = (DeviceArray((n,), d) for n, d in ((R + 1, "int32"), (R, "int32"), (T, "int64"), (T, "int32"), (1, "int32")))
    x = [DeviceArray((T, h, D), dtype) for h in (hq, hkv, hkv)]
    qr, out = DeviceArray((T, hq, D), dtype), DeviceArray((T, hq, D), dtype)

    def put(a, values):
        _lib.check(_lib.lib.mars_copy_to_device(C.c_void_p(a.data_ptr()), C.c_void_p(values.ctypes.data), values.nbytes), "copy")

    def step():
        s = stream.value
        r.plan(new, cached, table, free, count, q_start=q_start, kv_lens=kv, slots=slots, positions=pos, free_count_out=left, stream=s)
        r.store(cache, *x, pos, slots, q_out=qr, stream=s)
        r.attend(cache, qr, out, q_start, kv, table, stream=s)

    state = dict(lens=np.zeros(R, np.int32), free=pages, k=[np.zeros((0, hkv, D))] * R, v=[np.zeros((0, hkv, D))] * R)

    def inputs(n):
        n = np.array(n, np.int32)
        vals = [ref.to_bits(rng.standard_normal((T, h, D)), dtype) for h in (hq, hkv, hkv)]
        put(new, n)
        put(cached, state["lens"])
        put(count, np.array([state["free"]], np.int32))
        for a, b in zip(x, vals):
            put(a, b)
        return n, [ref.from_bits(b, dtype) for b in vals]

    def check(n, vals):
        assert hip.hipStreamSynchronize(stream) == 0
        got, at = out.numpy().astype(np.float64), 0
        p = np.concatenate([state["lens"][i] + np.arange(n[i]) for i in range(R)] + [np.zeros(T - n.sum())]).astype(np.int32)[None]
        qq, kk = (ref.rotate(y, p, 1e4, 64, (32,), False)[0] for y in vals[:2])
        for i in range(R):
            rows = slice(at, at + n[i])
            state["k"][i] = np.concatenate([state["k"][i], ref.rounded(kk[rows], dtype)])
            state["v"][i] = np.concatenate([state["v"][i], vals[2][rows]])
            L = len(state["k"][i])
            P = -(-L // page)
            pad = np.zeros((2, P * page, hkv, D))
            pad[0, :L], pad[1, :L] = state["k"][i], state["v"][i]
            if n[i]:
                want, _, tol, _ = ref.attend(ref.rounded(qq[rows], dtype), pad[0].reshape(P, page, hkv, D).transpose(0, 2, 1, 3),
                                             pad[1].reshape(P, page, hkv, D).transpose(0, 2, 3, 1), [0, n[i]], [L], np.arange(P)[None], dtype)
                # q and k may each be rounded to the other neighbour than here: two roundings more in every score
                assert np.all(np.abs(got[rows] - want) <= tol + 2.0 ** -10 * 16)
            at += n[i]
        state["lens"] = state["lens"] + n
        assert np.array_equal(kv.numpy(), state["lens"])
        state["free"] = int(left.numpy()[0])

    for n in ([5, 0, 3], [1, 1, 1]):
        io = inputs(n)
        step()
        check(*io)
    graph, exe = C.c_void_p(), C.c_void_p()
    io = inputs([1, 1, 1])
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    step()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
    for k, n in enumerate(([1, 1, 1], [2, 4, 1], [0, 1, 0], [1, 1, 6], [1, 1, 1])):
        io = inputs(n) if k else io
        assert hip.hipGraphLaunch(exe, stream) == 0
        check(*io)
        if k == 2:                                       # eager work between replays
            io = inputs([1, 0, 1])
            step()
            check(*io)
    assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0 and hip.hipStreamDestroy(stream) == 0


def test_read_memories_example():
    """examples/read_memories.py: every step of its session against the restatement, over the cache as it stands at the end."""
    import importlib.util

    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("read_memories", ROOT / "examples" / "read_memories.py")
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    s, free = ex.main(say=lambda *_: None)
    assert free == ex.POOL and len(s.steps) == 6
    k, v = s.cache.k_pages.numpy().astype(np.float64), s.cache.v_pages.numpy().astype(np.float64)
    kt, ke = s.cache.times.numpy(), s.cache.episodes.numpy()
    for t in s.steps:                                    # slots are written once, so the end's cache holds every step's
        want, _, tol, _ = ref.attend(t["q"].astype(np.float64), k, v, t["start"], t["lens"], t["table"], "float16", cap=30.0,
                                     decay=s.decay.numpy().astype(np.float64), q_times=t["times"], k_times=kt, q_eps=t["episodes"], k_eps=ke)
        assert np.all(np.abs(t["out"].astype(np.float64) - want) <= tol)
    first, last = s.steps[0], s.steps[-1]
    assert (last["lens"] == np.array(first["new_lens"]) + [5 + i for i in range(3)] + 4).all()


# ---- attend: what the weights' range holds --------------------------------------------
def dense(s, v, es, dtype):
    """Scores s (rows, keys; -inf: not seen) over v (keys, D) in 64 bits, and the bounds of out and lse: the roundings of output
    and weights, scores off by es (rows,), and for float16 the spacing of its subnormals, 2^-25 a weight against a largest of 2^7 or more."""
    top = s.max(1, keepdims=True)
    w = np.exp(s - top)
    total = w.sum(1, keepdims=True)
    o, size, u = w @ v / total, w @ np.abs(v) / total, ref.U[dtype]
    tiny = 2.0 ** -32 * np.sum(np.isfinite(s), 1, keepdims=True) * np.abs(v).max() / total if dtype == "float16" else 0.0
    lse = (top + np.log(total))[:, 0]
    return o, lse, u * np.abs(o) + u * size + 2.2 * es[:, None] * size + tiny + 2.0 ** -24, es + 2.0 ** -20 * (1 + np.abs(lse))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("kind", ["few", "many"])
def test_attend_long_tails(kind, dtype):
    """One key far above tens of thousands of others that weigh something together, e^-17.4 each: none of that is lost, neither in
    requests of single tokens nor in tiles of many rows, each over all keys in one piece."""
    rng = np.random.default_rng(20)
    L, D, page = 32_768, 64, 256
    requests, n, hq, hkv = (256, 1, 4, 4) if kind == "few" else (1, 768, 64, 1)
    one, k, v = make_cache(rng, [L], hkv, D, dtype, page)
    k = np.zeros_like(k)
    k[one[0][0], :, 5, 0] = ref.to_bits(17.4, dtype)
    v = np.full(v.shape, 0, v.dtype)
    j = np.arange(L)
    tail = ref.to_bits(rng.uniform(0.5, 1.5, (L, D)), dtype)
    tail[5] = ref.to_bits(np.where(np.arange(D) < D // 2, 0.0, 1.0), dtype)
    for g in range(hkv):
        v[one[0][j // page], g, :, j % page] = tail
    q = np.zeros((requests * n, hq, D))
    q[..., 0] = 8.0                                      # times D^-0.5: the score is k's element 0
    cache = PagedCache(dev(k, dtype), dev(v, dtype))
    out, lse = dev(ref.to_bits(np.zeros(q.shape), dtype), dtype), dev(np.zeros(q.shape[:2], np.float32))
    Reader(hq, hkv, D, dtype, page).attend(cache, dev(ref.to_bits(q, dtype), dtype), out, dev((np.arange(requests + 1) * n).astype(np.int32)),
                                           dev(np.full(requests, L, np.int32)), dev(np.repeat(one, requests, 0)), lse=lse, max_new=n,
                                           prefix_lens=dev(np.full(requests, L, np.int32)))
    s = np.zeros((1, L))
    s[0, 5] = ref.rounded(17.4, dtype)
    want, wlse, tol, ltol = dense(s, ref.from_bits(tail, dtype), np.array([(D + 8) * 2.0 ** -24 * s.max() + 2.0 ** -20]), dtype)
    assert 8e-4 < want[0, 0] < 1e-3
    err = np.abs(ref.from_bits(out.numpy(), dtype) - want[0]) - tol[0]
    assert np.all(err <= 0), float(err.max())
    assert np.all(np.abs(lse.numpy() - wlse[0]) <= ltol[0])


@pytest.mark.parametrize("n,length", [(1, 2_000), (1, 20_001), (13, 5_000), (70, 6_007), (200, 3_333)])
@pytest.mark.parametrize("hq,hkv,D,dtype,page", [(8, 2, 128, "bfloat16", 64), (6, 6, 64, "float16", 16), (2, 1, 256, "float16", 32)])
def test_attend_scores_that_rise_and_fall(n, length, hq, hkv, D, dtype, page):
    """Scores that rise, fall, or rise and fall along the keys by more than the weights' range with every tile: the running reference
    moves in each, rows in the middle of a wave at other keys than their neighbours, and pieces that are joined differ by hundreds."""
    rng = np.random.default_rng(n + D)
    table, k, v = make_cache(rng, [length], hkv, D, dtype, page)
    j = np.arange(length)
    kf = ref.from_bits(k, dtype)
    q = rng.standard_normal((n, hq, D)) * 0.5
    q[..., 0] = D ** 0.5 * np.where(rng.random((n, hq)) < 0.5, 1.0, -0.5)    # times D^-0.5: that part of the score is +-k's element 0
    for shape in (j, length - j, length / 2 - np.abs(j - length // 2)):
        kf[table[0][j // page], :, j % page, 0] = (shape * (400.0 / length) + shape % 7 * 0.1)[:, None] if length > 4000 else (shape * 0.1)[:, None]
        check_attend(Reader(hq, hkv, D, dtype, page), dtype, ref.to_bits(q, dtype), ref.to_bits(kf, dtype), v, [0, n], [length], table, max_new=(0, n))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_attend_scores_of_any_size_in_tiles(dtype):
    """Scores far from zero in requests of many rows, in one piece and in many."""
    rng = np.random.default_rng(16)
    n, D, page = 40, 64, 16
    for L in (200, 3_000):
        table, k, v = make_cache(rng, [L, L], 1, D, dtype, page)
        q = ref.to_bits(rng.standard_normal((2 * n, 2, D)), dtype)
        for scale in (-40.0, 1e-6, 30.0):
            check_attend(Reader(2, 1, D, dtype, page), dtype, q, k, v, [0, n, 2 * n], [L, L], table, max_new=(0, n), scale=scale)


@pytest.mark.parametrize("n,dtype", [(1, "float16"), (1, "bfloat16"), (40, "float16"), (40, "bfloat16")])
def test_attend_caps_of_any_size(n, dtype):
    """s = cap tanh(s / cap) for caps from below the scores to far above them, where it is s itself. Scores off by 2^-20 cap for
    caps up to 64, and by 2^-19 |s| (tanh to 2^-20 of its value, and its argument's roundings) above."""
    rng = np.random.default_rng(n)
    D, page, L = 64, 16, 300 + n
    table, k, v = make_cache(rng, [L], 1, D, dtype, page)
    q = ref.to_bits(6.0 * rng.standard_normal((n, 2, D)), dtype)
    cache, j = PagedCache(dev(k, dtype), dev(v, dtype)), np.arange(L)
    kf, vf = (ref.from_bits(x, dtype) for x in (k, v))
    kf, vf = kf[table[0][j // page], 0, j % page], vf[table[0][j // page], 0, :, j % page]
    r, start, lens, d_table, dq = Reader(2, 1, D, dtype, page), dev(np.array([0, n], np.int32)), dev(np.array([L], np.int32)), dev(table), dev(q, dtype)

    def call(cap):
        out, lse = dev(ref.to_bits(np.zeros(q.shape), dtype), dtype), dev(np.zeros((n, 2), np.float32))
        r.attend(cache, dq, out, start, lens, d_table, lse=lse, cap=cap, max_new=n)
        return ref.from_bits(out.numpy(), dtype), lse.numpy()

    seen = j[None] <= (L - n + np.arange(n))[:, None]
    none = call(0.0)
    for cap in (1e-3, 20.0, 64.0, 65.0, 130.0, 300.0, 1e4, 1e6, 1e8, 1e30, 3.4e38):
        got, glse = call(cap)
        for h in range(2):
            s = ref.from_bits(q, dtype)[:, h] @ kf.T * D ** -0.5
            most = np.max(np.where(seen, np.abs(s), 0), 1)
            es = (D + 8) * 2.0 ** -24 * np.max(np.where(seen, np.abs(ref.from_bits(q, dtype)[:, h]) @ np.abs(kf.T) * D ** -0.5, 0), 1)
            es = es + (2.0 ** -20 * cap if cap <= 64 else 2.0 ** -19 * most) + 2.0 ** -20
            want, wlse, tol, ltol = dense(np.where(seen, cap * np.tanh(s / cap), -np.inf), vf, es, dtype)
            assert np.all(np.abs(got[:, h] - want) <= tol), (cap, h, float((np.abs(got[:, h] - want) - tol).max()))
            assert np.all(np.abs(glse[:, h] - wlse) <= ltol), (cap, h, float((np.abs(glse[:, h] - wlse) - ltol).max()))
            if cap >= 1e8:                               # no cap at all, to the last bits of the scores
                assert np.all(np.abs(got - none[0])[:, h] <= 2 * tol) and np.all(np.abs(glse - none[1])[:, h] <= 2 * ltol)


@pytest.mark.parametrize("n", [1, 40])
def test_attend_scores_of_zero_at_the_largest_scales(n):
    """Scores of exactly 0 stay 0 where the scale, or the scale over the cap, is as large as its type holds: every key weighs the same."""
    rng = np.random.default_rng(n)
    D, page, L, dtype = 64, 16, 200 + n, "float16"
    table, k, v = make_cache(rng, [L], 1, D, dtype, page)
    q = np.zeros((n, 2, D), np.float16)
    j = np.arange(L)
    vf = v.astype(np.float64)[table[0][j // page], 0, :, j % page]
    s = np.where(j[None] <= (L - n + np.arange(n))[:, None], 0.0, -np.inf)
    want, _, tol, _ = dense(s, vf, np.full(n, 2.0 ** -20), dtype)
    for opt in (dict(scale=3.4e38), dict(scale=-3.4e38), dict(cap=1e-40), dict(scale=3e38, cap=30.0), dict(scale=3e38, cap=1e5)):
        out = dev(np.ones(q.shape, np.float16))
        Reader(2, 1, D, dtype, page).attend(PagedCache(dev(k), dev(v)), dev(q), out, dev(np.array([0, n], np.int32)), dev(np.array([L], np.int32)),
                                            dev(table), max_new=n, **opt)
        assert np.all(np.abs(out.numpy().astype(np.float64) - want[:, None]) <= tol[:, None]), opt


def test_plan_of_the_most_tokens():
    """num_tokens of 2^31 - 1, all but a few of them padding: the last rows are written as the first ones are."""
    T, page, width = 2 ** 31 - 1, 16, 4
    slots, pos = DeviceArray((T,), "int64"), DeviceArray((T,), "int32")
    ends = (0, T - 3_000)                                # the first rows and the last
    for a, dt in ((slots, np.int64), (pos, np.int32)):
        mark = np.full(3_000, -7, dt)
        for at in ends:
            _lib.check(_lib.lib.mars_copy_to_device(C.c_void_p(a.data_ptr() + at * mark.itemsize), C.c_void_p(mark.ctypes.data), mark.nbytes), "copy")
    free = np.arange(9, dtype=np.int32)
    q_start, kv, out, table = DeviceArray((3,), "int32"), DeviceArray((2,), "int32"), DeviceArray((1,), "int32"), dev(np.zeros((2, width), np.int32))
    Reader(page_size=page).plan(dev(np.array([20, 3], np.int32)), dev(np.array([0, 5], np.int32)), table, dev(free), dev(np.array([9], np.int32)),
                                q_start=q_start, kv_lens=kv, slots=slots, positions=pos, free_count_out=out)
    want = ref.plan(np.array([20, 3]), np.array([0, 5]), np.zeros((2, width), np.int32), free, 9, 3_000, page)
    for a, w, pad in ((slots, want[3], -1), (pos, want[4], 0)):
        for at in ends:
            got = np.empty(3_000, w.dtype)
            _lib.check(_lib.lib.mars_copy_to_host(C.c_void_p(got.ctypes.data), C.c_void_p(a.data_ptr() + at * got.itemsize), got.nbytes), "copy")
            np.testing.assert_array_equal(got, w if at == 0 else np.full(3_000, pad, w.dtype))


# ---- store: more tokens than k_kv_store takes -------------------------------------------
@pytest.mark.parametrize("D,rope,sections,adjacent", [(64, 64, (32,), False), (64, 64, (32,), True), (64, 48, (4, 20, 0), True), (64, 16, (0, 3, 5), False),
                                                      (64, 0, (), False), (128, 64, (32,), False), (128, 128, (16, 24, 24), True),
                                                      (128, 32, (16,), True), (256, 256, (128,), False), (256, 256, (40, 40, 48), True),
                                                      (256, 112, (56,), False), (256, 0, (), False)])
@pytest.mark.parametrize("tokens", [1025, 1089])
def test_store_many_rotations(D, rope, sections, adjacent, tokens):
    run_store(tokens, 6, 3, D, "float16", 32, rope, sections, adjacent, packed=tokens == 1025, seed=rope + D)
    run_store(tokens, 2, 1, D, "bfloat16", 64, rope, sections, adjacent, inverse=True, seed=rope + D + 1)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("tokens", [1025, 1100])
def test_store_many_layouts(tokens, D):
    run_store(tokens, 4, 2, D, "bfloat16", 64, D, (D // 2,), interleaved=True, seed=1)
    run_store(tokens, 4, 2, D, "float16", 16, D, (D // 4, D // 8, D // 8), in_place=True, seed=2)
    run_store(tokens, 4, 2, D, "float16", 128, D // 2, (D // 4,), True, in_place=True, seed=2)
    run_store(tokens, 4, 2, D, "float16", 16, D, (D // 2,), inverse=True, packed=False, in_place=True, seed=3)
    # slots in no order, one page for each token, chunks that go on at slots that are not multiples of 8, forwards and backwards
    rng = np.random.default_rng(5)
    run_store(tokens, 2, 1, D, "float16", 16, D, (D // 2,), slots=rng.permutation(tokens * 3)[:tokens].astype(np.int64), pages=-(-tokens * 3 // 16))
    run_store(tokens, 2, 1, D, "bfloat16", 16, D, (D // 2,), slots=np.arange(tokens, dtype=np.int64)[::-1].copy() + 3, pages=-(-tokens // 16) + 1)
    run_store(tokens, 2, 2, D, "bfloat16", 32, D, (D // 2,), slots=np.arange(tokens, dtype=np.int64) + 5, pages=-(-tokens // 32) + 1)
    run_store(tokens, 2, 2, D, "float16", 256, D, (D // 2,), slots=np.arange(tokens, dtype=np.int64) + 8, pages=-(-tokens // 256) + 1)


@pytest.mark.parametrize("tokens", [40, 1100])
def test_store_in_parts(tokens):
    """q alone and k, v alone: the bits of the call that takes all; times and episodes left as they are where none are given."""
    rng = np.random.default_rng(tokens)
    hq, hkv, D, page, dtype = 6, 2, 64, 32, "float16"
    r = Reader(hq, hkv, D, dtype, page, rope_dim=D, rope_sections=(16, 8, 8))
    q, k, v = (dev(ref.to_bits(rng.standard_normal((tokens, h, D)), dtype)) for h in (hq, hkv, hkv))
    pages = -(-tokens // page) + 2
    pos, slots = dev(rng.integers(0, 5_000, (3, tokens)).astype(np.int32)), dev((rng.permutation(tokens) + 11).astype(np.int64))

    def cache():
        return PagedCache(dev(np.zeros((pages, hkv, page, D), np.float16)), dev(np.zeros((pages, hkv, D, page), np.float16)),
                          dev(np.full(pages * page, -3, np.float32)), dev(np.full(pages * page, -3, np.int32)))

    both, alone = cache(), cache()
    q_both, q_alone = (dev(np.zeros((tokens, hq, D), np.float16)) for _ in range(2))
    r.store(both, q, k, v, pos, slots, q_out=q_both, times=dev(np.ones(tokens, np.float32)), episodes=dev(np.ones(tokens, np.int32)))
    r.store(None, q, None, None, pos, None, q_out=q_alone)
    r.store(alone, None, k, v, pos, slots)
    np.testing.assert_array_equal(q_alone.numpy().view(np.uint16), q_both.numpy().view(np.uint16))
    np.testing.assert_array_equal(alone.k_pages.numpy().view(np.uint16), both.k_pages.numpy().view(np.uint16))
    np.testing.assert_array_equal(alone.v_pages.numpy().view(np.uint16), both.v_pages.numpy().view(np.uint16))
    assert np.all(alone.times.numpy() == -3) and np.all(alone.episodes.numpy() == -3)
    hit = np.isin(np.arange(pages * page), slots.numpy())
    np.testing.assert_array_equal(both.times.numpy(), np.where(hit, 1, -3))
    np.testing.assert_array_equal(both.episodes.numpy(), np.where(hit, 1, -3))
    assert alone.k_pages.numpy().any() and q_alone.numpy().any()


def test_store_many_past_32_bits():
    """More tokens than k_kv_store takes, to pages whose elements lie past 2^31: the slots read back by their own addresses."""
    hkv, D, page, dtype, tokens = 2, 128, 256, "float16", 1_100
    n = hkv * page * D
    pages = 2 ** 31 // n + 40
    kb, vb = (DeviceArray((pages, hkv, page, D), dtype) for _ in range(2))
    rng = np.random.default_rng(13)
    ids = np.array([pages - 1, 3, pages - 9, pages - 30, 2 ** 31 // n + 1])
    j = np.arange(tokens)
    slots = ids[j // page].astype(np.int64) * page + j % page
    assert slots.max() * hkv * D > 2 ** 31
    x = [ref.to_bits(rng.standard_normal((tokens, hkv, D)), dtype) for _ in range(2)]
    Reader(hkv, hkv, D, dtype, page).store(PagedCache(kb, _As(vb, (pages, hkv, D, page))), None, dev(x[0]), dev(x[1]), None, dev(slots))
    for base, want, order in ((kb, x[0], (0, 2, 1, 3)), (vb, x[1], (0, 3, 1, 2))):
        for p, i in enumerate(ids):
            got = np.empty(n, np.float16)
            _lib.check(_lib.lib.mars_copy_to_host(C.c_void_p(got.ctypes.data), C.c_void_p(base.data_ptr() + 2 * n * int(i)), got.nbytes), "copy")
            got = got.reshape((1, hkv, page, D) if base is kb else (1, hkv, D, page)).transpose(order)[0]
            rows = want[p * page:(p + 1) * page]
            np.testing.assert_array_equal(got[:len(rows)].view(np.uint16), rows.view(np.uint16))


@pytest.mark.parametrize("kind", ["few", "many"])
def test_attend_capped_scores_one_by_one(kind):
    """Every row sees one key, so its lse is that key's capped score: within 2^-19 of its value and 2^-21 (the reference lies up to 7
    away), however small it is beside the cap, for scores from far below the cap to far above it."""
    D, page, n = 64, 16, 200
    s = np.concatenate([np.geomspace(1e-4, 100.0, n // 2), -np.geomspace(1e-4, 100.0, n // 2)])
    k = np.zeros((-(-n // page) if kind == "many" else n, 1, page, D))
    k[(np.arange(n) // page, 0, np.arange(n) % page, 0) if kind == "many" else (np.arange(n), 0, 0, 0)] = s
    q = np.zeros((n, 1, D))
    q[..., 0] = 8.0                                      # times D^-0.5: the score is k's element 0
    s = ref.rounded(s, "float16")
    cache = PagedCache(dev(k.astype(np.float16)), dev(np.ones((len(k), 1, D, page), np.float16)), None, dev(np.arange(len(k) * page, dtype=np.int32)))
    few = kind == "few"
    start, lens = (np.arange(n + 1), np.ones(n)) if few else (np.array([0, n]), np.array([n]))
    table = np.arange(len(k), dtype=np.int32).reshape((n, 1) if few else (1, -1))
    for cap in (1.0, 20.0, 30.0, 50.0, 64.0, 65.0, 1e3, 1e5):
        out, lse = dev(np.zeros((n, 1, D), np.float16)), dev(np.zeros((n, 1), np.float32))
        Reader(1, 1, D, "float16", page).attend(cache, dev(q.astype(np.float16)), out, dev(start.astype(np.int32)), dev(lens.astype(np.int32)), dev(table),
                                                lse=lse, cap=cap, max_new=1 if few else n, q_episodes=dev(np.full(n, -1, np.int32)) if few else dev(np.arange(n, dtype=np.int32)))
        want = cap * np.tanh(s / cap)
        err = np.abs(lse.numpy()[:, 0] - want)
        assert np.all(err <= 2.0 ** -19 * np.abs(want) + 2.0 ** -21), (cap, float((err - 2.0 ** -19 * np.abs(want)).max()))
        assert np.all(out.numpy() == 1)


def test_plan_of_more_tokens_than_lengths_hold():
    """A request that would pass 2^31 - 1 tokens is not served; one that reaches them is."""
    page, width = 256, 2 ** 23 + 1
    table, free = dev(np.full((2, width), 5, np.int32)), dev(np.array([70, 71, 72], np.int32))
    q_start, kv, slots, pos, out, after = (DeviceArray((n,), d) for n, d in ((3, "int32"), (2, "int32"), (31, "int64"), (31, "int32"), (1, "int32"),
                                                                            (2, "int32")))
    have = np.array([2 ** 31 - 10, 2 ** 31 - 12], np.int32)
    Reader(page_size=page).plan(dev(np.array([20, 11], np.int32)), dev(have), table, free, dev(np.array([3], np.int32)), q_start=q_start, kv_lens=kv,
                                slots=slots, positions=pos, free_count_out=out, next_lens=after)
    np.testing.assert_array_equal(kv.numpy(), [0, 2 ** 31 - 1])
    np.testing.assert_array_equal(after.numpy(), [2 ** 31 - 10, 2 ** 31 - 1])
    np.testing.assert_array_equal(slots.numpy(), [-1] * 20 + [5 * page + 244 + i for i in range(11)])
    np.testing.assert_array_equal(pos.numpy()[20:], have[1] + np.arange(11))
    assert out.numpy()[0] == 3 and np.all(table.numpy() == 5)
