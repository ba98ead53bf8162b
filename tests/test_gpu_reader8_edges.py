"""Shared prefixes whose first request does not hold them."""
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
