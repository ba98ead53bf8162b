"""The reading path's operators restated in 64 bits (numpy), and the error bounds their tests hold the kernels to.

Bounds, per value, from the operations' roundings (u: unit roundoff of the 16-bit type, 2^-11 or 2^-8 / 2):
  attend  the output's rounding u |o|; each weight's rounding to 16 bits u sum(p |v|) (float16: and the spacing of its
          subnormals, 2^-25 per weight against a largest weight of at least 1); scores off by at most `es`, which moves
          every normalised weight by a factor within exp(+-2 es); es = (D + 8) 2^-24 max sum|q k| scale for the fp32
          product, 2^-20 cap for the bounded tanh, 2^-22 |bias| for the age term, 2^-20 for exp2 and the sums.
  store   the output's rounding u |y|; angles within 2^-19 of a radian (the phase rounded to 2^-25 turns and the error of
          sincospi), times |a| + |b| of the pair.
"""
from __future__ import annotations

import numpy as np

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def to_bits(x, dtype):
    """float array -> the device array's numpy form (float16, or bfloat16 bits as uint16, both rounded to nearest even)."""
    x = np.asarray(x, np.float32)
    if dtype == "float16":
        return x.astype(np.float16)
    b = x.view(np.uint32)
    out = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), out)


def from_bits(b, dtype):
    if dtype == "float16":
        return b.astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rounded(x, dtype):
    return from_bits(to_bits(x, dtype), dtype)


def plan(new, cached, table, free_pages, free_count, num_tokens, page):
    """Request by request. Returns table, q_start, kv_lens, slots, positions, free_count_out."""
    table = table.copy()
    width = table.shape[1]
    start, kv = [0], []
    slots, pos = np.full(num_tokens, -1, np.int64), np.zeros(num_tokens, np.int32)
    wanted = taken = 0                       # pages asked for so far (served or not); pages handed out
    for r, (n, c) in enumerate(zip(np.maximum(new, 0).tolist(), np.maximum(cached, 0).tolist())):
        first = start[-1]
        start.append(first + n)
        have, pages = -(-c // page), -(-(c + n) // page)
        fits = pages <= width and first + n <= num_tokens
        need = pages - have if fits else 0
        served = fits and (need == 0 or wanted + need <= free_count)
        if served:
            for j in range(have, pages):
                table[r, j] = free_pages[free_count - 1 - (wanted + j - have)]
            if need:
                taken = wanted + need
        wanted += need
        kv.append(c + n if served else 0)
        for i in range(n):
            if first + i < num_tokens:
                pos[first + i] = c + i
                if served:
                    slots[first + i] = int(table[r, (c + i) // page]) * page + (c + i) % page
    return table, np.array(start, np.int32), np.array(kv, np.int32), slots, pos, free_count - taken


def rotate(x, positions, theta, rope_dim, sections, adjacent, inverse=False):
    """x (tokens, heads, dim) float64; positions (axes, tokens). Returns the turned x and |a| + |b| of each element's pair."""
    y, size = x.copy(), np.zeros_like(x)
    half = rope_dim // 2
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    for i in range(half):
        ang = positions[axis[i]].astype(np.float64) * theta ** (-2.0 * i / rope_dim)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        s = -s if inverse else s
        p, r = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        a, b = x[..., p], x[..., r]
        y[..., p], y[..., r] = a * c - b * s, a * s + b * c
        size[..., p] = size[..., r] = np.abs(a) + np.abs(b)
    return y, size


def attend(q, k_pages, v_pages, q_start, kv_lens, table, dtype, scale=None, cap=0.0, decay=None, q_times=None, k_times=None,
           q_eps=None, k_eps=None, prefix=None):
    """All arrays numpy; q (T, Hq, D), k_pages (N, Hkv, P, D), v_pages (N, Hkv, D, P) float64; k_times, k_eps per slot.
    Returns out, lse, and the bounds of both. Rows that no request owns are NaN."""
    T, hq, D = q.shape
    _, hkv, P, _ = k_pages.shape
    scale = D ** -0.5 if scale is None else scale
    out, lse = np.full((T, hq, D), np.nan), np.full((T, hq), np.nan)
    tol, ltol = np.full((T, hq, D), np.nan), np.full((T, hq), np.nan)
    u = U[dtype]
    for r in range(len(kv_lens)):
        b, e, L = int(q_start[r]), int(q_start[r + 1]), int(kv_lens[r])
        n = e - b
        if n == 0:
            continue
        j = np.arange(L)
        page, off = table[r][j // P].astype(np.int64), j % P
        slot = page * P + off
        p = L - n + np.arange(n)
        seen = j[None] <= p[:, None]
        if prefix is not None:
            seen = seen | (j < prefix[r])[None]
        if q_eps is not None:
            a, c = q_eps[b:e][:, None], k_eps[slot][None]
            seen = seen & ((a < 0) | (c < 0) | (a == c))
        for h in range(hq):
            g = h // (hq // hkv)
            k, v = k_pages[page, g, off], v_pages[page, g, :, off]
            with np.errstate(all="ignore"):
                s = q[b:e, h] @ k.T * scale
                es = (D + 8) * 2.0 ** -24 * np.max(np.where(seen, np.abs(q[b:e, h]) @ np.abs(k.T) * abs(scale), 0), axis=1, initial=0)
                if cap:
                    s = cap * np.tanh(s / cap)
                    es = es + cap * 2.0 ** -20
                if decay is not None:
                    bias = decay[h] * np.maximum(0.0, q_times[b:e, None].astype(np.float64) - k_times[slot][None].astype(np.float64))
                    s = s - bias
                    es = es + 2.0 ** -22 * np.max(np.where(seen & (bias < 1e4), bias, 0), axis=1, initial=0)
                es = es + 2.0 ** -20
                s = np.where(seen, s, -np.inf)
                top = np.max(s, axis=1, initial=-np.inf)
                w = np.where(seen, np.exp(s - np.where(top == -np.inf, 0, top)[:, None]), 0)
                l = w.sum(1)
                empty = l == 0
                d = np.where(empty, 1, l)[:, None]
                vz = np.zeros((n, D))
                az = np.zeros((n, D))
                for i in range(n):                       # keys not seen take no part, whatever they hold
                    m = seen[i]
                    vz[i] = w[i, m] @ v[m]
                    az[i] = w[i, m] @ np.abs(v[m])
                o, A = vz / d, az / d
                few = 2.0 ** -25 * L * np.max(np.abs(np.where(np.isfinite(v), v, 0)), initial=0) / d if dtype == "float16" else 0
                out[b:e, h] = np.where(empty[:, None], 0, o)
                lse[b:e, h] = np.where(empty, -np.inf, top + np.log(np.where(empty, 1, l)))
                tol[b:e, h] = u * np.abs(o) + u * A + 2.2 * es[:, None] * A + few + 2.0 ** -24
                ltol[b:e, h] = es + 2.0 ** -20 * (1 + np.abs(np.where(empty, 0, lse[b:e, h])))
    return out, lse, tol, ltol
