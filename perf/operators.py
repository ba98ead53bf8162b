"""The reading work that is measured: laying out, filling and attending to the paged cache of the memories' tokens.

Paths, one call of mars_amd.reader each:
  "plan"    block table, slot map and positions of a step, from the requests' lengths
  "store"   q and k rotated by their (time, height, width) positions; k, v, time and episode written to their slots
  "attend"  new tokens (one, or a chunk) of every request over the request's cached tokens

k_pages is (pages, kv_heads, page, head_dim) and v_pages (pages, kv_heads, head_dim, page); page ids are in no order. A case's
lengths come from its own numbers ("lens" seeds them), everything else from prepare()'s seed.
"""
import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    wide = dict(type="bf16", hq=32, hkv=8, d=128, page=64)              # grouped heads of 128
    narrow = dict(type="fp16", hq=12, hkv=12, d=64, page=16)            # the width of an embedding row: 12 heads of 64
    bare = dict(cap=0.0, decay=0.0, episode=0, prefix=0, lens=1)
    return [
        # eight agents, one token each: the step's tables where only latency counts
        dict(name="plan_8", path="plan", requests=8, chunk=1, long=0, cached=2000, page=16, lens=1),
        # a busy server's step: 768 requests, one in sixteen of them with a chunk of new tokens
        dict(name="plan_768", path="plan", requests=768, chunk=512, long=16, cached=8000, page=64, lens=2),
        # single tokens of 32 requests, one position axis
        dict(name="store_32", path="store", tokens=32, slots=32_768, axes=1, rope=64, theta=1e4, pairs="half", **narrow),
        # chunks of image and text tokens, 4,099 of them, three axes
        dict(name="store_4099", path="store", tokens=4_099, slots=65_536, axes=3, rope=128, theta=1e6, pairs="half", **wide),
        # the smallest question: one token over one retrieved episode
        dict(name="attend_one_137", path="attend", requests=1, chunk=1, long=1, cached=136, spread=0.0, **narrow, **bare),
        # one token over a long memory: few rows, many keys
        dict(name="attend_one_131k", path="attend", requests=1, chunk=1, long=1, cached=131_070, spread=0.0, **wide, **bare),
        # a decode step of 64 requests of ragged length
        dict(name="attend_64", path="attend", requests=64, chunk=1, long=1, cached=7_800, spread=0.9, **wide, **bare),
        # the same with scores capped and decayed by age, every request asking within one of its episodes of 900 tokens
        dict(name="attend_scoped_48", path="attend", requests=48, chunk=1, long=1, cached=6_001, spread=0.5, type="fp16", hq=16, hkv=2, d=128, page=32,
             cap=30.0, decay=0.02, episode=900, prefix=0, lens=3),
        # drafted tokens checked: five at a time, three query heads to a key head
        dict(name="attend_drafts_24", path="attend", requests=24, chunk=5, long=1, cached=3_001, spread=0.7, type="bf16", hq=12, hkv=4, d=64, page=16, **bare),
        # a step of chunked prompts: two chunks of 511 among 22 single tokens, decayed by age
        dict(name="attend_mixed_24", path="attend", requests=24, chunk=511, long=12, cached=2_600, spread=0.8, **wide, **{**bare, "decay": 0.02}),
        # packed memories encoded from nothing: each token sees its own episode and a shared prefix; capped and decayed
        dict(name="attend_packed_4001", path="attend", requests=2, chunk=4_001, long=1, cached=0, spread=0.0, **{**narrow, "page": 32},
             cap=50.0, decay=0.05, episode=700, prefix=96, lens=5),
        # the largest: long chunks over as many cached tokens again
        dict(name="attend_chunk_4096", path="attend", requests=2, chunk=4_096, long=1, cached=4_100, spread=0.0, **wide, **bare),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["plan", "store", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if path == "plan":
        return dict(path=path, requests=_log(rng, 1, 1_024), chunk=_log(rng, 1, 600), long=rng.choice([0, 1, 4, 16]),
                    cached=_log(rng, 10, 16_000), page=page, lens=rng.randint(1, 10**6))
    d = rng.choice([64, 64, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    heads = dict(type=rng.choice(["fp16", "bf16"]), hq=hkv * rng.choice([1, 2, 3, 4]), hkv=hkv, d=d, page=page)
    if path == "store":
        return dict(path=path, tokens=_log(rng, 1, 6_000), slots=65_536, axes=rng.choice([1, 3, 3]), rope=rng.choice([d, d, d // 2]),
                    theta=rng.choice([1e4, 1e6]), pairs=rng.choice(["half", "half", "adjacent"]), **heads)
    opts = dict(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), decay=rng.choice([0.0, 0.0, 0.02, 0.1]), episode=rng.choice([0, 0, 150, 1_100]),
                prefix=rng.choice([0, 0, 40]), lens=rng.randint(1, 10**6), spread=rng.choice([0.0, 0.5, 0.95]))
    room = 250_000_000 // (hkv * d)                                      # tokens of a gigabyte
    kind = rng.choice(["single", "single", "few", "chunk", "chunk", "mixed"])
    if kind == "single":
        r = _log(rng, 1, 96)
        return dict(path=path, requests=r, chunk=1, long=1, cached=_log(rng, 20, max(30, min(60_000, room // r))), **heads, **opts)
    if kind == "few":
        r = _log(rng, 1, 40)
        return dict(path=path, requests=r, chunk=rng.randint(2, 12), long=1, cached=_log(rng, 20, max(30, min(120_000, room) // r)), **heads, **opts)
    if kind == "mixed":
        return dict(path=path, requests=rng.randint(4, 24), chunk=_log(rng, 30, 500), long=rng.choice([4, 8]), cached=_log(rng, 50, 2_500), **heads, **opts)
    r = rng.randint(1, 2)
    most = 4_096 if r * heads["hq"] * d <= 8_192 else 2_400
    return dict(path=path, requests=r, chunk=_log(rng, 13, most), long=1, cached=rng.choice([0, _log(rng, 20, most)]), **heads, **opts)


def _lens(case):
    """New and cached tokens of each request. long: 1 gives every request a chunk, k one in k, 0 none; the others one token."""
    rng = random.Random(case["lens"])
    r, long = case["requests"], case["long"]
    new = [case["chunk"] if long and i % long == long - 1 else 1 for i in range(r)]
    if case["path"] == "plan":
        return new, [rng.randint(0, case["cached"]) for _ in range(r)]
    return new, [int(round(case["cached"] * (1 - case["spread"] * rng.random()))) for _ in range(r)]


def _scope(case, new, cached):
    """Each request's episode asked for (-1: all)."""
    rng = random.Random(case["lens"] + 1)
    return [rng.randint(0, (c - 1) // case["episode"]) if case["episode"] and c else -1 for c in cached]


def _episodes(case, n, c, scope):
    """Episodes of a request's tokens (all of them), and those that its new tokens ask within: token j lies in episode j // length, a prefix
    and new tokens after cached ones in none; new tokens without cached ones ask within their own episodes."""
    e, key = case["episode"], torch.arange(c + n, device=DEV)
    own_episode = torch.where((key < case["prefix"]) | ((key >= c) if c else (key < 0)), -1, key // max(e, 1))
    return own_episode, torch.full((n,), scope, device=DEV) if c else own_episode


def _ceil(a, b):
    return -(-a // b)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    if case["path"] == "plan":
        _prepare_plan(case, g, s)
    elif case["path"] == "store":
        _prepare_store(case, g, s)
    else:
        _prepare_attend(case, g, s)
    if own:
        from mars_amd import reader
        s["lib"] = reader
        geometry = dict(page_size=case["page"])
        if "hq" in case:
            geometry.update(q_heads=case["hq"], kv_heads=case["hkv"], head_dim=case["d"], dtype={"fp16": "float16", "bf16": "bfloat16"}[case["type"]])
        if case["path"] == "store":
            geometry.update(rope_dim=case["rope"], rope_theta=case["theta"], rope_sections=_sections(case), rope_adjacent=case["pairs"] == "adjacent")
        s["reader"] = reader.Reader(**geometry)
        if "k_pages" in s:
            s["cache"] = reader.PagedCache(s["k_pages"], s["v_pages"], times=s["k_times"], episodes=s["k_episodes"])
    return s


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _prepare_plan(case, g, s):
    new, cached = _lens(case)
    p, r, t = case["page"], len(new), sum(new)
    width = max(_ceil(c + n, p) for c, n in zip(cached, new))
    have = [_ceil(c, p) for c in cached]
    need = sum(_ceil(c + n, p) - h for c, n, h in zip(cached, new, have))
    ids = torch.randperm(sum(have) + need + 64, device=DEV, generator=g).to(torch.int32)
    table = torch.zeros(r, width, dtype=torch.int32, device=DEV)
    owned = torch.arange(width, device=DEV)[None, :] < _i32(have)[:, None]
    table[owned] = ids[:sum(have)]
    s.update(new=_i32(new), cached=_i32(cached), table=table, free=ids[sum(have):].clone(), free_count=_i32([need + 64]),
             q_start=_i32([0] * (r + 1)), kv_lens=_i32([0] * r), positions=_i32([0] * t), free_out=_i32([0]),
             slots=torch.zeros(t, dtype=torch.int64, device=DEV))


def _sections(case):
    half = case["rope"] // 2
    return (half,) if case["axes"] == 1 else (half // 4, half // 4 + half // 8, half - half // 4 - half // 4 - half // 8)


def _pages(case, pages, g):
    shape = (pages, case["hkv"], case["page"], case["d"])
    k = torch.randn(shape, device=DEV, generator=g, dtype=torch.float32).to(TYPES[case["type"]])
    v = torch.randn((shape[0], shape[1], shape[3], shape[2]), device=DEV, generator=g, dtype=torch.float32).to(TYPES[case["type"]])
    return k, v


def _prepare_store(case, g, s):
    t, p, d, dt = case["tokens"], case["page"], case["d"], TYPES[case["type"]]
    # one projection gives q, k and v of a token side by side
    qkv = torch.randn(t, case["hq"] + 2 * case["hkv"], d, device=DEV, generator=g).to(dt)
    s["q"], s["k"], s["v"] = qkv.split([case["hq"], case["hkv"], case["hkv"]], dim=1)
    s["k_pages"], s["v_pages"] = _pages(case, case["slots"] // p, g)
    s["k_times"] = torch.zeros(case["slots"], device=DEV)
    s["k_episodes"] = torch.full((case["slots"],), -1, dtype=torch.int32, device=DEV)
    order = torch.randperm(case["slots"] // p, device=DEV, generator=g)
    at = torch.arange(t, device=DEV)
    if t <= 64:                                                          # single tokens: a page of its own for each
        s["slots"] = order[at] * p + at % p
    else:                                                                # chunks: pages filled in order, from the middle of one
        at = at + p // 2 + 1
        s["slots"] = order[at // p] * p + at % p
    time = 20_000 + torch.arange(t, device=DEV) // 64
    grid = [time, torch.randint(0, 48, (t,), device=DEV, generator=g), torch.randint(0, 64, (t,), device=DEV, generator=g)]
    s["positions"] = torch.stack(grid[:case["axes"]]).to(torch.int32)
    s["times"] = 600 * torch.rand(t, device=DEV, generator=g)
    s["episodes"] = torch.randint(0, 1000, (t,), device=DEV, generator=g).to(torch.int32)
    s["q_out"] = torch.empty(t, case["hq"], d, dtype=dt, device=DEV)


def _prepare_attend(case, g, s):
    new, cached = _lens(case)
    scope = _scope(case, new, cached)
    p, r, t = case["page"], len(new), sum(new)
    lens = [c + n for c, n in zip(cached, new)]
    width, total = max(_ceil(x, p) for x in lens), sum(_ceil(x, p) for x in lens)
    ids = torch.randperm(total + 3, device=DEV, generator=g).to(torch.int32)
    table = torch.zeros(r, width, dtype=torch.int32, device=DEV)
    table[torch.arange(width, device=DEV)[None, :] < _i32([_ceil(x, p) for x in lens])[:, None]] = ids[:total]
    s["k_pages"], s["v_pages"] = _pages(case, total + 3, g)
    s.update(table=table, kv_lens=_i32(lens), q_start=_i32([sum(new[:i]) for i in range(r + 1)]), n_max=max(new), l_max=max(lens))
    s["q"] = torch.randn(t, case["hq"], case["d"], device=DEV, generator=g).to(TYPES[case["type"]])
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(t, case["hq"], device=DEV)
    s["decay"] = s["q_times"] = s["q_episodes"] = s["prefix"] = s["k_times"] = s["k_episodes"] = None
    if case["prefix"]:
        s["prefix"] = _i32([case["prefix"]] * r)
    if case["decay"]:
        # ages of a few minutes; a quarter of the heads forget four times as fast as the next
        s["decay"] = case["decay"] * 0.25 ** (torch.arange(case["hq"], device=DEV) % 4).to(torch.float32)
        s["k_times"] = torch.zeros((total + 3) * p, device=DEV)
    req = torch.repeat_interleave(torch.arange(r, device=DEV), s["kv_lens"].long(), output_size=sum(lens))
    begin = torch.cumsum(s["kv_lens"].long(), 0) - s["kv_lens"]
    at = torch.arange(sum(lens), device=DEV) - begin[req]                # every request's tokens in a row
    slot, is_new = table[req, at // p].long() * p + at % p, at >= _i32(cached)[req]
    if case["decay"]:
        age = 600 * torch.rand(sum(lens), device=DEV, generator=g)
        time = age[torch.argsort(req * 1000.0 + age.double())]           # rising within each request
        s["k_times"][slot], s["q_times"] = time, time[is_new]
    if case["episode"]:
        of = [_episodes(case, n, c, ask) for n, c, ask in zip(new, cached, scope)]
        s["k_episodes"] = torch.full(((total + 3) * p,), -1, dtype=torch.int32, device=DEV)
        s["k_episodes"][slot] = torch.cat([key for key, _ in of]).to(torch.int32)
        s["q_episodes"] = torch.cat([ask for _, ask in of]).to(torch.int32)


def run(s):
    if not own:
        return {"plan": _plain_plan, "store": _plain_store, "attend": _plain_attend}[s["case"]["path"]](s)
    stream = torch.cuda.current_stream().cuda_stream
    path = s["case"]["path"]
    if path == "plan":
        s["reader"].plan(s["new"], s["cached"], s["table"], s["free"], s["free_count"], q_start=s["q_start"], kv_lens=s["kv_lens"],
                         slots=s["slots"], positions=s["positions"], free_count_out=s["free_out"], stream=stream)
        return [s["table"], s["q_start"], s["kv_lens"], s["slots"], s["positions"], s["free_out"]]
    if path == "store":
        s["reader"].store(s["cache"], s["q"], s["k"], s["v"], s["positions"], s["slots"], q_out=s["q_out"], times=s["times"],
                          episodes=s["episodes"], stream=stream)
        return [s["q_out"], s["k_pages"], s["v_pages"], s["k_times"], s["k_episodes"]]
    s["reader"].attend(s["cache"], s["q"], s["out"], s["q_start"], s["kv_lens"], s["table"], lse=s["lse"], cap=s["case"]["cap"], decay=s["decay"],
                       q_times=s["q_times"], q_episodes=s["q_episodes"], prefix_lens=s["prefix"], max_new=s["n_max"], stream=stream)
    return [s["out"], s["lse"]]


def _plain_plan(s):
    p, r, t = s["case"]["page"], s["new"].numel(), s["slots"].numel()
    new, cached, free = s["new"].long(), s["cached"].long(), s["free_count"].long()
    width = s["table"].shape[1]
    have, pages = (cached + p - 1) // p, (cached + new + p - 1) // p
    end = torch.cumsum(new, 0)
    start = torch.cat([end.new_zeros(1), end])
    fits = (pages <= width) & (end <= t)
    need = torch.where(fits, pages - have, 0)
    taken = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (taken <= free))
    used = torch.where(served & (need > 0), taken, 0).max()
    j = torch.arange(width, device=DEV)
    fresh = served[:, None] & (j >= have[:, None]) & (j < pages[:, None])
    at = free - 1 - ((taken - need)[:, None] + j - have[:, None])
    table = torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], s["table"])
    tok = torch.arange(t, device=DEV)
    req = (torch.searchsorted(start, tok, right=True) - 1).clamp(max=r - 1)
    pos = cached[req] + tok - start[req]
    slots = torch.where(served[req], table[req, (pos // p).clamp(max=width - 1)].long() * p + pos % p, -1)
    kv = torch.where(served, cached + new, 0)
    return [table, start.to(torch.int32), kv.to(torch.int32), slots, pos.to(torch.int32), (free - used).to(torch.int32)]


def _rotate(x, cos, sin, case):
    rd, x = case["rope"], x.float()
    turn, rest = x[..., :rd], x[..., rd:]
    if case["pairs"] == "half":
        a, b = turn[..., :rd // 2], turn[..., rd // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)
    a, b = turn[..., 0::2], turn[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), rest], -1)


def _axes(case):
    """The position axis that each frequency turns with."""
    sections = _sections(case)
    return torch.repeat_interleave(torch.arange(len(sections), device=DEV), torch.tensor(sections, device=DEV), output_size=case["rope"] // 2)


def _plain_store(s):
    case, p = s["case"], s["case"]["page"]
    freq = case["theta"] ** (-torch.arange(0, case["rope"], 2, device=DEV, dtype=torch.float32) / case["rope"])
    angle = s["positions"].float()[_axes(case)].T * freq                 # (tokens, rope / 2)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    q_out = _rotate(s["q"], cos, sin, case).to(s["q"].dtype)
    page, at = s["slots"] // p, s["slots"] % p
    s["k_pages"][page, :, at] = _rotate(s["k"], cos, sin, case).to(s["k"].dtype)
    s["v_pages"][page, :, :, at] = s["v"]
    s["k_times"][s["slots"]] = s["times"]
    s["k_episodes"][s["slots"]] = s["episodes"]
    return [q_out, s["k_pages"], s["v_pages"], s["k_times"], s["k_episodes"]]


def _plain_attend(s):
    case = s["case"]
    r, width = s["table"].shape
    hq, hkv, d, n, keys = case["hq"], case["hkv"], case["d"], s["n_max"], s["l_max"]
    table, lens, start = s["table"].long(), s["kv_lens"].long(), s["q_start"].long()
    k = s["k_pages"][table].permute(0, 2, 4, 1, 3).reshape(r, hkv, d, -1)[..., :keys].float()       # (requests, heads, d, keys)
    v = s["v_pages"][table].permute(0, 2, 1, 4, 3).reshape(r, hkv, -1, d)[:, :, :keys].float()      # (requests, heads, keys, d)
    i, j = torch.arange(n, device=DEV), torch.arange(keys, device=DEV)
    count = start[1:] - start[:-1]
    row = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)                                      # (requests, n)
    q = s["q"][row].float().reshape(r, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(r, hkv, -1, d)
    x = (torch.matmul(q, k.contiguous()) * d ** -0.5).reshape(r, hq, n, keys)
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    limit = (lens - count)[:, None] + i + 1
    if s["prefix"] is not None:
        limit = torch.maximum(limit, s["prefix"].long()[:, None])
    seen = j < torch.minimum(limit, lens[:, None])[..., None]                                        # (requests, n, keys)
    slot = (table[:, :, None] * case["page"] + torch.arange(case["page"], device=DEV)).reshape(r, -1)[:, :keys]
    if s["decay"] is not None:
        age = (s["q_times"][row][..., None] - s["k_times"][slot][:, None]).clamp(min=0)
        x = x - s["decay"][:, None, None] * age[:, None]
    if s["q_episodes"] is not None:
        ask, key = s["q_episodes"][row][..., None], s["k_episodes"][slot][:, None]
        seen = seen & ((ask < 0) | (key < 0) | (ask == key))
    x = torch.where(seen[:, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.reshape(r, hkv, -1, keys), v.contiguous()).reshape(r, hq, n, d) / torch.where(total > 0, total, 1)
    lse = (top + torch.log(total))[..., 0]
    mine = torch.arange(s["q"].shape[0], device=DEV)
    req = torch.searchsorted(start, mine, right=True) - 1
    return [o[req, :, mine - start[req]].to(s["q"].dtype), lse[req, :, mine - start[req]]]


def work(case):
    if case["path"] == "plan":
        new, cached = _lens(case)
        p, r, t = case["page"], len(new), sum(new)
        fresh = sum(_ceil(c + n, p) - _ceil(c, p) for c, n in zip(cached, new))
        # lengths in and out, the pages that new tokens go to, a slot and a position for each token
        return dict(bytes=r * 16 + fresh * 8 + sum(_ceil(c + n, p) - c // p for c, n in zip(cached, new)) * 4 + t * 12, flops=0)
    d = case["d"]
    if case["path"] == "store":
        t = case["tokens"]
        return dict(bytes=t * ((2 * case["hq"] + 4 * case["hkv"]) * d * 2 + 4 * case["axes"] + 8 + 16),
                    flops=t * (case["hq"] + case["hkv"]) * case["rope"] * 3)
    new, cached = _lens(case)
    scope = _scope(case, new, cached)
    e, pairs, keys = case["episode"], 0, 0
    for n, c, ask in zip(new, cached, scope):
        m = min(case["prefix"], c + n)
        if e and c:                                                      # of the cached tokens: one episode and the prefix; and the new ones
            seen = max(0, min(ask * e + e, c) - max(ask * e, m)) + min(m, c)
            pairs, keys = pairs + n * seen + n * (n + 1) // 2, keys + seen + n
        elif e:                                                          # the prefix, and what came before in the token's own episode
            parts = [min(a + e, n) - max(a, m) for a in range(0, n, e) if min(a + e, n) > m]
            pairs, keys = pairs + m * m + sum(x * m + x * (x + 1) // 2 for x in parts), keys + n
        else:
            ahead = max(0, m - c)
            pairs, keys = pairs + n * c + n * (n + 1) // 2 + ahead * (ahead - 1) // 2, keys + c + n
    tokens = sum(new)
    more = (4 if case["decay"] else 0) + (4 if case["episode"] else 0)
    total = sum(new) + sum(cached) if case["episode"] else keys          # every key's episode is looked at
    return dict(bytes=keys * (case["hkv"] * d * 4 + (4 if case["decay"] else 0)) + total * (4 if case["episode"] else 0)
                + tokens * (case["hq"] * (d * 4 + 4) + more) + sum(_ceil(a + b, case["page"]) for a, b in zip(new, cached)) * 4,
                flops=4 * d * case["hq"] * pairs)


def exact(case, seed):
    if case["path"] == "plan":
        return None                                                      # whole numbers alone
    s, p, d = prepare(case, seed), case["page"], case["d"]
    if case["path"] == "store":
        half = case["rope"] // 2
        axis = [a for a, count in enumerate(_sections(case)) for _ in range(count)]
        turned = [s["q"].double(), s["k"].double()]
        for x in turned:
            for i in range(half):
                a, b = (i, i + half) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
                angle = s["positions"][axis[i]].double()[:, None] * math.exp(-2 * i / case["rope"] * math.log(case["theta"]))
                u, v = x[..., a].clone(), x[..., b].clone()
                x[..., a] = u * torch.cos(angle) - v * torch.sin(angle)
                x[..., b] = u * torch.sin(angle) + v * torch.cos(angle)
        k, v, times = s["k_pages"].double(), s["v_pages"].double(), s["k_times"].double()
        k[s["slots"] // p, :, s["slots"] % p] = turned[1]
        v[s["slots"] // p, :, :, s["slots"] % p] = s["v"].double()
        times[s["slots"]] = s["times"].double()
        return [turned[0], k, v, times, None]
    new, cached = _lens(case)
    group = case["hq"] // case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device=DEV)
    for r, (n, c) in enumerate(zip(new, cached)):
        first, at = sum(new[:r]), torch.arange(c + n, device=DEV)
        page, off = s["table"][r].long()[at // p], at % p
        for b in range(0, n, 1024):                                      # queries at a time
            rows = torch.arange(b, min(n, b + 1024), device=DEV)
            seen = at[None] <= c + rows[:, None]
            if s["prefix"] is not None:
                seen = seen | (at < s["prefix"][r])[None]
            if s["q_episodes"] is not None:
                ask, key = s["q_episodes"][first + rows][:, None], s["k_episodes"][page * p + off][None]
                seen = seen & ((ask == -1) | (key == -1) | (ask == key))
            for h in range(case["hq"]):
                k, v = s["k_pages"][page, h // group, off].double(), s["v_pages"][page, h // group, :, off].double()
                x = s["q"][first + rows, h].double() @ k.T.contiguous() / math.sqrt(d)
                if case["cap"]:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                if s["decay"] is not None:
                    old = (s["q_times"][first + rows].double()[:, None] - s["k_times"][page * p + off].double()[None]).clamp(min=0)
                    x = x - float(s["decay"][h]) * old
                x = x.masked_fill(~seen, -math.inf)
                lse[first + rows, h] = torch.logsumexp(x, 1)
                out[first + rows, h] = torch.nan_to_num(torch.softmax(x, 1)) @ v
    return [out, lse]
