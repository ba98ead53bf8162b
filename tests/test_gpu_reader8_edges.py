"""Shared prefixes whose first request does not hold them, and 8-bit values and weights at the ends of their ranges."""
from __future__ import annotations

import numpy as np
import pytest

import mars_amd
import reader8_ref as ref8
import reader_ref as ref
from mars_amd.reader import PagedCache, Reader
from test_gpu_reader import dev, make_cache
from test_gpu_reader8 import check, make_shared, quantise

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    mars_amd.init(0)


# ---- the first request of a group -------------------------------------------------------
@pytest.mark.parametrize("held8", [False, True])
@pytest.mark.parametrize("S", [160, 3_024])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("kind", ["not served", "ended", "short", "several", "none"])
def test_shared_first_request_without_the_prefix(kind, n, S, held8):
    """A group's first request that has not the prefix cached, its row of the table naming other pages or none: the others read the prefix by the
    row of one that has, or each for itself."""
    rng = np.random.default_rng(S + n)
    hq, hkv, D, page, dtype = 4, 2, 64, 16, "float16"
    groups = [(S, [(3, n), (9, n), (40, n), (0, 1), (17, n), (2, n), (33, 2)]), (96, [(5, 1), (6, n)])]
    if kind == "ended":
        groups[0][1][0] = (3, 0)                         # no new tokens either
    table, k, v, q_start, lens, starts, shared = make_shared(rng, groups, hkv, D, dtype, page)
    pages = k.shape[0]
    wrong = {"several": (0, 1, 2, 3, 4), "none": range(7)}.get(kind, (0,))
    for r in wrong:
        new = int(q_start[r + 1] - q_start[r])
        lens[r] = 0 if kind in ("not served", "ended") or r % 2 else S - 16 + new            # a page less than the prefix
        table[r] = rng.integers(0, pages, table.shape[1]) if r % 2 or kind == "short" else rng.choice([-1, pages, 10 ** 9, 2 ** 31 - 1], table.shape[1])
        used = -(-lens[r] // page)
        table[r, :used] = rng.permutation(pages)[:used]  # its own tokens lie there
    q = ref.to_bits(rng.standard_normal((int(q_start[-1]), hq, D)), dtype)
    c, held = quantise(k, v, dtype) if held8 else ((k, v), (ref.from_bits(k, dtype), ref.from_bits(v, dtype)))
    check(Reader(hq, hkv, D, dtype, page), dtype, q, c, held, q_start, lens, table, max_new=(0, n, 1), groups=(starts, shared))


# ---- weights far below a shared prefix's ------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
def test_own_keys_far_below_a_shared_prefix(D):
    """A request of many rows behind a prefix that the kernel of few rows read, its own keys' weights some 2^-28 of the prefix's: float16 weights are off by
    up to 2^-32 of the largest. Prefix keys score 20, own ones 0.5; the prefix's values are 0."""
    hq, hkv, page, dtype, S, own, n, G = 4, 1, 16, "float16", 16, 700, 20, 60
    rng = np.random.default_rng(D)
    table, k, v, q_start, lens, starts, shared = make_shared(rng, [(S, [(own, n)])] + [(16, [(3, 1)]) for _ in range(G)], hkv, D, dtype, page)
    T = int(q_start[-1])
    # k: elements of 1/8 times the score, q of 1 under scale 8 / D
    k[...] = 0.5 / 8
    v[...] = 40960.0
    k[table[0, 0]], v[table[0, 0]] = 20.0 / 8, 0.0
    c, held = quantise(k, v, dtype)
    q = np.ones((T, hq, D), np.float16)
    got = np.asarray(check(Reader(hq, hkv, D, dtype, page), dtype, q, c, held, q_start, lens, table, max_new=(0,), groups=(starts, shared), scale=8.0 / D))[:n]
    keys = (own + 1 + np.arange(n))[:, None, None]       # own ones that each row sees
    w = np.exp(-19.5)
    total = S + keys * w
    want = keys * w * 40960.0 / total
    # the output's rounding and its weights' to 2^-32 of the largest; scores of fp32 as in reader_ref
    tol = 2.0 ** -11 * want + keys * 2.0 ** -32 * 40960.0 / total + 2.2 * ((D + 8) * 2.0 ** -24 * 20 + 2.0 ** -20) * want + 2.0 ** -24
    assert np.all(np.abs(got - want) <= tol), (float(got[0, 0, 0]), float(want[0, 0, 0]))


# ---- values at the ends of bfloat16 ------------------------------------------------------
@pytest.mark.parametrize("decay", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("held8", [True, False])
def test_attend_largest_values(held8, D, decay):
    """A key whose values are near the type's largest and whose weight is nearly 2^8 times the reference's, some of its values 0: those elements get
    what the other keys give. The large ones are beyond the sums' range (2^7 times 3.19e38 is 2^134.9, fp32 ends at 2^128): infinities, or their average."""
    hq, hkv, page, dtype, L = 2, 1, 64, "bfloat16", 900
    rng = np.random.default_rng(D)
    table, k, v = make_cache(rng, [L], hkv, D, dtype, page)
    at = 256                                             # the fifth step of 64 keys: the wave of the first one
    pg, off = table[0][at // page], at % page
    x = ref.from_bits(v, dtype)
    large = np.arange(D) % 3 == 0
    x[pg, 0, :, off] = np.where(large, 240 * 2.0 ** 120, 0.0)
    k = np.zeros(k.shape)
    k[pg, 0, off] = 1.0
    k, v = ref.to_bits(k, dtype), ref.to_bits(x, dtype)
    c, held = quantise(k, v, dtype) if held8 else ((k, v), (ref.from_bits(k, dtype), ref.from_bits(v, dtype)))
    assert not held8 or c[3][pg, 0, off] == 247          # the largest that is stored
    q = ref.to_bits(np.ones((1, hq, D)), dtype)
    opt = dict(decay=np.zeros(hq, np.float32), q_times=np.zeros(1, np.float32), k_times=np.zeros(k.shape[0] * page, np.float32)) if decay else {}
    want, _, tol, _ = ref.attend(ref.from_bits(q, dtype), *held, [0, 1], [L], table, dtype, scale=5.5445 / D, **opt)
    t = {n: dev(opt[n]) for n in ("decay", "q_times") if n in opt}
    cache = PagedCache(dev(c[0], None if held8 else dtype), dev(c[1], None if held8 else dtype), dev(opt["k_times"]) if opt else None, None,
                       *(dev(y) for y in c[2:]))
    for m in (0, 1):
        out = dev(np.zeros(q.shape, np.uint16), dtype)
        Reader(hq, hkv, D, dtype, page).attend(cache, dev(q, dtype), out, dev(np.array([0, 1], np.int32)), dev(np.array([L], np.int32)), dev(table), scale=5.5445 / D,
                                               max_new=m, **t)
        got = ref.from_bits(out.numpy(), dtype)
        with np.errstate(invalid="ignore"):
            fine = np.abs(got - want) <= tol
        assert np.all(fine[:, :, ~large]) and np.all((fine | (got == np.inf))[:, :, large]), (m, got[0, 0, :6], want[0, 0, :6])


@pytest.mark.parametrize("decay", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attend_smallest_values(D, decay):
    """Heads whose values all take the least exponent, weights times 2^-117 still count."""
    hq, hkv, page, dtype, L = 2, 1, 64, "bfloat16", 700
    rng = np.random.default_rng(D)
    table, k, v = make_cache(rng, [L], hkv, D, dtype, page)
    c, _ = quantise(k, v, dtype)
    c[3][...] = 10
    c[1][...] = np.where(c[1] & 0x40, c[1], c[1] | 0x40)                 # sizes of 2 to 448 times 2^-117
    c[1][(c[1] & 0x7F) == 0x7F] ^= 1
    held = ref8.pages_held(*c)
    q = ref.to_bits(rng.standard_normal((1, hq, D)), dtype)
    opt = dict(decay=np.zeros(hq, np.float32), q_times=np.zeros(1, np.float32), k_times=np.zeros(k.shape[0] * page, np.float32)) if decay else {}
    out = np.asarray(check(Reader(hq, hkv, D, dtype, page), dtype, q, c, held, [0, 1], [L], table, max_new=(1,), **opt))
    want, _, tol, _ = ref.attend(ref.from_bits(q, dtype), held[0], held[1] * 2.0 ** 117, [0, 1], [L], table, dtype)
    # scaled to sizes of 1. reader_ref's bound, and for a weight's two parts in bfloat16, whose least step is 2^-133: half of that a key, at 2^-117
    # and values of up to 448; weights are at least half of exp(s - top)
    j = np.arange(L)
    s = np.einsum("hd,jd->hj", ref.from_bits(q, dtype)[0], held[0][table[0][j // page], 0, j % page]) * D ** -0.5
    least = 2.0 ** -17 * 448 * L / (0.5 * np.exp(s - s.max(1, keepdims=True)).sum(1))
    assert np.all(np.abs(out * 2.0 ** 117 - want) <= tol + least[None, :, None]), float(np.max(np.abs(out * 2.0 ** 117 - want) - tol))


# ---- values that the reader's type does not have -----------------------------------------
@pytest.mark.parametrize("n,length", [(1, 200), (1, 5_000), (3, 200)])
def test_attend_values_of_the_other_type(n, length):
    """A cache with values beyond float16's largest, read by a float16 reader's few rows: taken as they are held, also where a NaN elsewhere has rows
    looked over again."""
    hq, hkv, D, page, dtype = 4, 2, 64, 16, "float16"
    rng = np.random.default_rng(length)
    table, k, v = make_cache(rng, [length], hkv, D, dtype, page)
    k = ref.to_bits(ref.from_bits(k, dtype) / 4, dtype)
    c, _ = quantise(k, v, dtype)
    for j in (5, 70, 150):
        pg, off = table[0][j // page], j % page
        c[1][pg, :, :, off] = 0x70                       # 128 times 2^13: over the keys some 2^20 / length
        c[3][pg, :, off] = 140
    for nan in (False, True):
        if nan:
            c[1][table[0][40 // page], 1, 7, 40 % page] = 0x7F
        held = ref8.pages_held(*c)
        q = ref.to_bits(rng.standard_normal((n, hq, D)), dtype)
        out = check(Reader(hq, hkv, D, dtype, page), dtype, q, c, held, [0, n], [length], table, max_new=(n,))
        assert np.isfinite(out).sum() == out.size - (2 * n if nan else 0)
