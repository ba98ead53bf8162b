"""Shared prefixes whose first request does not hold them, or beside whose weights a request's own are small."""
from __future__ import annotations

import numpy as np
import pytest

import mars_amd
import reader_ref as ref
from mars_amd.reader import Reader
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
