"""The reading work over caches that are held in 8 bits, or whose first pages several requests share.

Paths:
  "store"   q and k rotated, k and v quantised as they are written to their slots; what these slots then stand for, read back
  "load"    k, v, time and episode of any slots read back from a quantised cache as rows of 16 bits
  "attend"  new tokens (one, or a chunk) of every request over the request's tokens in a quantised cache
  "shared"  the same, where the requests of a group have a long prefix of their tokens in common, in a cache of 16 or 8 bits

A quantised page holds e4m3 values and, for each token and kv head, the exponents of a power of two for k and for v: an element is
its e4m3 value times 2^(exponent - 127), with the least exponent that keeps the head's largest element within 448. k_pages is (pages,
kv_heads, page, head_dim), v_pages (pages, kv_heads, head_dim, page), k_scales and v_scales (pages, kv_heads, page); page ids are in
no order. A case's lengths come from its own numbers ("lens" seeds them), everything else from prepare()'s seed.
"""
import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
LEAST = {"fp16": -15, "bf16": -117}          # exponents that keep every value a value of the type


def listed():
    wide = dict(type="bf16", hq=32, hkv=8, d=128, page=64)              # grouped heads of 128
    narrow = dict(type="fp16", hq=12, hkv=12, d=64, page=16)            # the width of an embedding row: 12 heads of 64
    alone = dict(bits=8, groups=0, shared=0)
    bare = dict(cap=0.0, decay=0.0, episode=0, prefix=0, lens=1)
    return [
        # single tokens of 32 requests, one position axis
        dict(name="store_32", path="store", tokens=32, slots=32_768, axes=1, rope=64, theta=1e4, pairs="half", **narrow),
        # chunks of image and text tokens, 4,099 of them, three axes
        dict(name="store_4099", path="store", tokens=4_099, slots=65_536, axes=3, rope=128, theta=1e6, pairs="half", **wide),
        # one retrieved episode's tokens, to be placed anew
        dict(name="load_137", path="load", tokens=137, run=137, slots=32_768, **narrow),
        # the memories of many answers, moved to another cache: runs of 700 tokens that begin anywhere in a page
        dict(name="load_20011", path="load", tokens=20_011, run=700, slots=65_536, **wide),
        # the smallest question: one token over one retrieved episode
        dict(name="attend_one_137", path="attend", requests=1, chunk=1, long=1, cached=136, spread=0.0, **narrow, **alone, **bare),
        # one token over a long memory: few rows, many keys
        dict(name="attend_one_131k", path="attend", requests=1, chunk=1, long=1, cached=131_070, spread=0.0, **wide, **alone, **bare),
        # a decode step of 64 requests of ragged length
        dict(name="attend_64", path="attend", requests=64, chunk=1, long=1, cached=7_800, spread=0.9, **wide, **alone, **bare),
        # a step of chunked prompts: two chunks of 511 among 22 single tokens, scores capped and decayed by age, within an episode of 900 tokens
        dict(name="attend_mixed_24", path="attend", requests=24, chunk=511, long=12, cached=2_600, spread=0.8, **wide, **alone,
             **{**bare, "cap": 30.0, "decay": 0.02, "episode": 900}),
        # long chunks over twice as many cached tokens
        dict(name="attend_chunk_2048", path="attend", requests=2, chunk=2_048, long=1, cached=4_100, spread=0.0, **wide, **alone, **bare),
        # eight agents ask about one conversation of 4,160 tokens, each some tokens into its answer
        dict(name="shared_8", path="shared", requests=8, chunk=1, long=1, cached=130, spread=0.9, bits=16, groups=1, shared=4_160, **narrow, **bare),
        # five conversations, 40 questions of 1 or 6 tokens about them; scores capped and decayed by age
        dict(name="shared_40", path="shared", requests=40, chunk=6, long=3, cached=900, spread=0.9, bits=16, groups=5, shared=6_016,
             type="fp16", hq=16, hkv=2, d=128, page=32, **{**bare, "cap": 30.0, "decay": 0.02}),
        # a busy server: 64 answers at once from one memory of 32,768 tokens
        dict(name="shared_64", path="shared", requests=64, chunk=1, long=1, cached=1_000, spread=0.9, bits=8, groups=1, shared=32_768, **wide, **bare),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["store", "load", "attend", "attend", "shared", "shared"])
    page = rng.choice([16, 32, 64, 128])
    d = rng.choice([64, 64, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    heads = dict(type=rng.choice(["fp16", "bf16"]), hq=hkv * rng.choice([1, 2, 3, 4]), hkv=hkv, d=d, page=page)
    if path == "store":
        return dict(path=path, tokens=_log(rng, 1, 6_000), slots=65_536, axes=rng.choice([1, 3, 3]), rope=rng.choice([d, d, d // 2]),
                    theta=rng.choice([1e4, 1e6]), pairs=rng.choice(["half", "half", "adjacent"]), **heads)
    if path == "load":
        return dict(path=path, tokens=_log(rng, 1, 30_000), run=_log(rng, 1, 1_500), slots=65_536, **heads)
    opts = dict(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), decay=rng.choice([0.0, 0.0, 0.02, 0.1]), lens=rng.randint(1, 10**6))
    room = 250_000_000 // (hkv * d)                                      # tokens of a gigabyte in 16 bits
    if path == "shared":
        r = _log(rng, 2, 72)
        groups = rng.choice([1, 1, 2, max(1, r // 6)])
        return dict(path=path, requests=r, chunk=rng.choice([1, 1, rng.randint(2, 9)]), long=rng.choice([1, 2, 5]), cached=_log(rng, 1, 1_500),
                    spread=rng.choice([0.0, 0.5, 0.95]), bits=rng.choice([8, 16]), groups=groups,
                    shared=_log(rng, 200, min(33_000, room // (2 * groups), 2_200_000_000 // (r * hkv * d))), episode=0, prefix=0, **heads, **opts)
    opts.update(bits=8, groups=0, shared=0, episode=rng.choice([0, 0, 150, 1_100]), prefix=rng.choice([0, 0, 40]), spread=rng.choice([0.0, 0.5, 0.95]))
    kind = rng.choice(["single", "single", "few", "chunk", "mixed"])
    if kind == "single":
        r = _log(rng, 1, 96)
        return dict(path=path, requests=r, chunk=1, long=1, cached=_log(rng, 20, max(30, min(60_000, room // r))), **heads, **opts)
    if kind == "few":
        r = _log(rng, 1, 40)
        return dict(path=path, requests=r, chunk=rng.randint(2, 12), long=1, cached=_log(rng, 20, max(30, min(120_000, room) // r)), **heads, **opts)
    if kind == "mixed":
        return dict(path=path, requests=rng.randint(4, 24), chunk=_log(rng, 30, 500), long=rng.choice([4, 8]), cached=_log(rng, 50, 2_500), **heads, **opts)
    most = 2_000 if heads["hq"] * d <= 4_096 else 1_400
    return dict(path=path, requests=rng.randint(1, 2), chunk=_log(rng, 13, most), long=1, cached=rng.choice([0, _log(rng, 20, 2_400)]), **heads, **opts)


def _ceil(a, b):
    return -(-a // b)


def _groups(case):
    """The first request of each group, and the number of requests behind the last; none: no prefix is shared."""
    n, r = case["groups"], case["requests"]
    cuts = sorted(random.Random(case["lens"] + 2).sample(range(1, r), n - 1)) if n > 1 else []
    return [0, *cuts, r] if n else []


def _prefixes(case):
    """The tokens that the requests of each group share: whole pages."""
    rng, p = random.Random(case["lens"] + 3), case["page"]
    return [max(1, int(case["shared"] * (1 if case["groups"] == 1 else rng.uniform(0.6, 1))) // p) * p for _ in range(case["groups"])]


def _lens(case):
    """New and cached tokens of each request, the prefix among them. long: 1 gives every request a chunk, k one in k; the others one token."""
    rng = random.Random(case["lens"])
    r, long = case["requests"], case["long"]
    new = [case["chunk"] if i % long == long - 1 else 1 for i in range(r)]
    cached = [int(round(case["cached"] * (1 - case["spread"] * rng.random()))) for _ in range(r)]
    starts = _groups(case)
    for first, end, shared in zip(starts, starts[1:], _prefixes(case)):
        cached[first:end] = [c + shared for c in cached[first:end]]
    return new, cached


def _scope(case, cached):
    """Each request's episode asked for (-1: all)."""
    rng = random.Random(case["lens"] + 1)
    return [rng.randint(0, (c - 1) // case["episode"]) if case["episode"] and c else -1 for c in cached]


def _episodes(case, n, c, scope):
    """Episodes of a request's tokens (all of them), and those that its new tokens ask within: token j lies in episode j // length, a prefix
    and new tokens after cached ones in none; new tokens without cached ones ask within their own episodes."""
    e, key = case["episode"], torch.arange(c + n, device=DEV)
    of = torch.where((key < case["prefix"]) | ((key >= c) if c else (key < 0)), -1, key // max(e, 1))
    return of, torch.full((n,), scope, device=DEV) if c else of


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _quantised(x, least):
    """e4m3 values (as bytes) of x (..., head_dim) and the exponent of each head, as a byte: the least that keeps it within 448."""
    top = torch.where(torch.isfinite(x), x.abs(), 0).amax(-1)
    m, e = torch.frexp(top)                                              # m in [1/2, 1): 448 is 7/8 of 2^9
    e = torch.where(top > 0, e - 9 + (m > 0.875).to(e.dtype), least).clamp(min=least)
    y = torch.where(torch.isfinite(x), torch.ldexp(x, -e[..., None]), math.nan)
    return y.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _values(bytes_, scales):
    return bytes_.view(torch.float8_e4m3fn).float() * torch.exp2(scales.float() - 127)


def _pages(case, pages, g, s):
    """Pages of random tokens, whose sizes differ by a few octaves."""
    shape, dt = (pages, case["hkv"], case["page"], case["d"]), TYPES[case["type"]]
    for name in "k", "v":
        x = torch.randn(shape, device=DEV, generator=g, dtype=torch.float32)
        x *= torch.exp2(0.7 * torch.randn(shape[:3], device=DEV, generator=g, dtype=torch.float32))[..., None]
        if case.get("bits", 8) == 8:
            x, s[name + "_scales"] = _quantised(x, LEAST[case["type"]])
        else:
            x = x.to(dt)
        s[name + "_pages"] = x if name == "k" else x.transpose(2, 3).contiguous()


def _sections(case):
    half = case["rope"] // 2
    return (half,) if case["axes"] == 1 else (half // 4, half // 4 + half // 8, half - half // 4 - half // 4 - half // 8)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    {"store": _prepare_store, "load": _prepare_load, "attend": _prepare_attend, "shared": _prepare_attend}[case["path"]](case, g, s)
    if own:
        from mars_amd import reader
        more = dict(rope_dim=case["rope"], rope_theta=case["theta"], rope_sections=_sections(case), rope_adjacent=case["pairs"] == "adjacent") if "rope" in case else {}
        s["reader"] = reader.Reader(q_heads=case["hq"], kv_heads=case["hkv"], head_dim=case["d"], dtype={"fp16": "float16", "bf16": "bfloat16"}[case["type"]],
                                    page_size=case["page"], **more)
        s["cache"] = reader.PagedCache(s["k_pages"], s["v_pages"], times=s["k_times"], episodes=s["k_episodes"], k_scales=s.get("k_scales"), v_scales=s.get("v_scales"))
    return s


def _rows_out(case, s):
    for name in "k_out", "v_out":
        s[name] = torch.empty(case["tokens"], case["hkv"], case["d"], dtype=TYPES[case["type"]], device=DEV)


def _prepare_store(case, g, s):
    t, p, d, dt = case["tokens"], case["page"], case["d"], TYPES[case["type"]]
    # one projection gives q, k and v of a token side by side
    qkv = torch.randn(t, case["hq"] + 2 * case["hkv"], d, device=DEV, generator=g).to(dt)
    s["q"], s["k"], s["v"] = qkv.split([case["hq"], case["hkv"], case["hkv"]], dim=1)
    _pages(case, case["slots"] // p, g, s)
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
    _rows_out(case, s)


def _prepare_load(case, g, s):
    t, p, run = case["tokens"], case["page"], case["run"]
    _pages(case, case["slots"] // p, g, s)
    s["k_times"] = 600 * torch.rand(case["slots"], device=DEV, generator=g)
    s["k_episodes"] = torch.randint(0, 1000, (case["slots"],), device=DEV, generator=g).to(torch.int32)
    order = torch.randperm(case["slots"] // p, device=DEV, generator=g)
    first = torch.randint(0, max(1, case["slots"] - run), (_ceil(t, run),), device=DEV, generator=g)
    at = torch.arange(t, device=DEV)
    at = first[at // run] + at % run                                     # a place in the order of the pages
    s["slots"] = order[at // p] * p + at % p
    s["times"], s["episodes"] = torch.empty(t, device=DEV), torch.empty(t, dtype=torch.int32, device=DEV)
    _rows_out(case, s)


def _prepare_attend(case, g, s):
    new, cached = _lens(case)
    scope, starts, prefixes = _scope(case, cached), _groups(case), _prefixes(case)
    p, r, t = case["page"], len(new), sum(new)
    lens = [c + n for c, n in zip(cached, new)]
    width = max(_ceil(x, p) for x in lens)
    owner = [i for i, (a, b) in enumerate(zip(starts, starts[1:])) for _ in range(b - a)] or [None] * r
    common = [0 if o is None else prefixes[o] // p for o in owner]       # pages of each request that its group shares
    total = sum(x // p for x in prefixes) + sum(_ceil(x, p) - c for x, c in zip(lens, common))
    ids = torch.randperm(total + 3, device=DEV, generator=g).to(torch.int32)
    table, at = torch.zeros(r, width, dtype=torch.int32, device=DEV), 0
    for a, b, x in zip(starts, starts[1:], prefixes):
        table[a:b, :x // p] = ids[at:at + x // p]
        at += x // p
    col = torch.arange(width, device=DEV)[None, :]
    table[(col >= _i32(common)[:, None]) & (col < _i32([_ceil(x, p) for x in lens])[:, None])] = ids[at:total]
    _pages(case, total + 3, g, s)
    s.update(table=table, kv_lens=_i32(lens), q_start=_i32([sum(new[:i]) for i in range(r + 1)]), n_max=max(new), l_max=max(lens))
    s["group_start"], s["shared_lens"] = (_i32(starts), _i32(prefixes)) if starts else (None, None)
    s["q"] = torch.randn(t, case["hq"], case["d"], device=DEV, generator=g).to(TYPES[case["type"]])
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(t, case["hq"], device=DEV)
    s["decay"] = s["q_times"] = s["q_episodes"] = s["prefix"] = s["k_times"] = s["k_episodes"] = None
    if case["prefix"]:
        s["prefix"] = _i32([case["prefix"]] * r)
    if case["decay"]:
        # ages of a few minutes, the memories in order of their rank; a quarter of the heads forget four times as fast as the next
        s["decay"] = case["decay"] * 0.25 ** (torch.arange(case["hq"], device=DEV) % 4).to(torch.float32)
        s["k_times"] = 600 * torch.rand((total + 3) * p, device=DEV, generator=g)
        s["q_times"] = 600 + torch.rand(t, device=DEV, generator=g)
    if case["episode"]:
        req = torch.repeat_interleave(torch.arange(r, device=DEV), s["kv_lens"].long(), output_size=sum(lens))
        begin = torch.cumsum(s["kv_lens"].long(), 0) - s["kv_lens"]
        at = torch.arange(sum(lens), device=DEV) - begin[req]            # every request's tokens in a row
        slot = table[req, at // p].long() * p + at % p
        of = [_episodes(case, n, c, ask) for n, c, ask in zip(new, cached, scope)]
        s["k_episodes"] = torch.full(((total + 3) * p,), -1, dtype=torch.int32, device=DEV)
        s["k_episodes"][slot] = torch.cat([key for key, _ in of]).to(torch.int32)
        s["q_episodes"] = torch.cat([ask for _, ask in of]).to(torch.int32)


def run(s):
    if not own:
        return {"store": _plain_store, "load": _plain_load, "attend": _plain_attend, "shared": _plain_attend}[s["case"]["path"]](s)
    stream = torch.cuda.current_stream().cuda_stream
    path = s["case"]["path"]
    if path == "store":
        s["reader"].store(s["cache"], s["q"], s["k"], s["v"], s["positions"], s["slots"], q_out=s["q_out"], times=s["times"],
                          episodes=s["episodes"], stream=stream)
        s["reader"].load(s["cache"], s["slots"], s["k_out"], s["v_out"], stream=stream)
        return [s["q_out"], s["k_out"], s["v_out"], s["k_times"], s["k_episodes"]]
    if path == "load":
        s["reader"].load(s["cache"], s["slots"], s["k_out"], s["v_out"], times=s["times"], episodes=s["episodes"], stream=stream)
        return [s["k_out"], s["v_out"], s["times"], s["episodes"]]
    s["reader"].attend(s["cache"], s["q"], s["out"], s["q_start"], s["kv_lens"], s["table"], lse=s["lse"], cap=s["case"]["cap"], decay=s["decay"],
                       q_times=s["q_times"], q_episodes=s["q_episodes"], prefix_lens=s["prefix"], group_start=s["group_start"],
                       shared_lens=s["shared_lens"], max_new=s["n_max"], stream=stream)
    return [s["out"], s["lse"]]


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
    freq = case["theta"] ** (-torch.arange(0, case["rope"], 2, device=DEV, dtype=torch.float64) / case["rope"])
    angle = s["positions"].double()[_axes(case)].T * freq                # (tokens, rope / 2), in 64 bits: positions are far
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q_out = _rotate(s["q"], cos, sin, case).to(s["q"].dtype)
    page, at, least = s["slots"] // p, s["slots"] % p, LEAST[case["type"]]
    s["k_pages"][page, :, at], s["k_scales"][page, :, at] = _quantised(_rotate(s["k"], cos, sin, case), least)
    s["v_pages"][page, :, :, at], s["v_scales"][page, :, at] = _quantised(s["v"].float(), least)
    s["k_times"][s["slots"]] = s["times"]
    s["k_episodes"][s["slots"]] = s["episodes"]
    return [q_out, *_read_back(s), s["k_times"], s["k_episodes"]]


def _read_back(s):
    page, at = s["slots"] // s["case"]["page"], s["slots"] % s["case"]["page"]
    return [_values(s["k_pages"][page, :, at], s["k_scales"][page, :, at][..., None]).to(s["k_out"].dtype),
            _values(s["v_pages"][page, :, :, at], s["v_scales"][page, :, at][..., None]).to(s["v_out"].dtype)]


def _plain_load(s):
    return [*_read_back(s), s["k_times"][s["slots"]], s["k_episodes"][s["slots"]]]


def _plain_attend(s):
    case = s["case"]
    r, width = s["table"].shape
    hq, hkv, d, n, keys = case["hq"], case["hkv"], case["d"], s["n_max"], s["l_max"]
    table, lens, start = s["table"].long(), s["kv_lens"].long(), s["q_start"].long()
    k, v = s["k_pages"], s["v_pages"]
    if case["bits"] == 8:
        k, v = _values(k, s["k_scales"][..., None]), _values(v, s["v_scales"][:, :, None])
    k = k[table].permute(0, 2, 4, 1, 3).reshape(r, hkv, d, -1)[..., :keys].float()                  # (requests, heads, d, keys)
    v = v[table].permute(0, 2, 1, 4, 3).reshape(r, hkv, -1, d)[:, :, :keys].float()                 # (requests, heads, keys, d)
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
    d, t = case["d"], case.get("tokens", 0)
    slot = case["hkv"] * (2 * d + 2)                                     # a token's bytes in a quantised cache
    if case["path"] == "store":                                          # q, k, v in, q out; the slots written, and read back
        return dict(bytes=t * ((2 * case["hq"] + 4 * case["hkv"]) * d * 2 + slot + 4 * case["axes"] + 8 + 16),
                    flops=t * (case["hq"] + case["hkv"]) * case["rope"] * 3)
    if case["path"] == "load":
        return dict(bytes=t * (slot + case["hkv"] * d * 4 + 8 + 16), flops=t * case["hkv"] * d * 2)
    new, cached = _lens(case)
    scope, starts = _scope(case, cached), _groups(case)
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
    keys -= sum(x * (b - a - 1) for a, b, x in zip(starts, starts[1:], _prefixes(case)))        # a group's prefix is read once
    tokens = sum(new)
    more = (4 if case["decay"] else 0) + (4 if e else 0)
    total = sum(new) + sum(cached) if e else keys                        # every key's episode is looked at
    key = (slot if case["bits"] == 8 else case["hkv"] * d * 4) + (4 if case["decay"] else 0)
    return dict(bytes=keys * key + total * (4 if e else 0) + tokens * (case["hq"] * (d * 4 + 4) + more)
                + sum(_ceil(a + b, case["page"]) for a, b in zip(new, cached)) * 4, flops=4 * d * case["hq"] * pairs)


def _nearest(x, least):
    """What a slot stands for after x (tokens, heads, d) in 64 bits was written to it."""
    top = x.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=least))
    unit = torch.where((unit / 2 * 448 >= top) & (unit > 2.0 ** least), unit / 2, torch.where(unit * 448 < top, unit * 2, unit))
    y = x / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)     # 3 bits behind the leading one, 2^-9 at least
    return torch.round(y / step) * step * unit                           # round: halves to even


def exact(case, seed):
    s, p, d = prepare(case, seed), case["page"], case["d"]
    if case["path"] == "load":
        page, off = s["slots"] // p, s["slots"] % p
        found = []
        for name in "k", "v":
            pages, scales = s[name + "_pages"].view(torch.float8_e4m3fn), s[name + "_scales"][page, :, off].double()
            rows = torch.empty(s["k_out"].shape, dtype=torch.float64, device=DEV)
            for h in range(case["hkv"]):
                held = pages[:, h].double()
                rows[:, h] = (held[page, off] if name == "k" else held[page, :, off]) * torch.pow(2.0, scales[:, h] - 127)[:, None]
            found.append(rows)
        return [*found, s["k_times"].double()[s["slots"]], None]
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
        times, least = s["k_times"].double(), LEAST[case["type"]]
        times[s["slots"]] = s["times"].double()
        return [turned[0], _nearest(turned[1], least), _nearest(s["v"].double(), least), times, None]
    new, cached = _lens(case)
    group = case["hq"] // case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device=DEV)
    for r, (n, c) in enumerate(zip(new, cached)):
        first, at = sum(new[:r]), torch.arange(c + n, device=DEV)
        page, off = s["table"][r].long()[at // p], at % p
        for h in range(case["hq"]):
            k, v = s["k_pages"][page, h // group, off], s["v_pages"][page, h // group, :, off]
            if case["bits"] == 8:
                k, v = (x.view(torch.float8_e4m3fn).double() * torch.pow(2.0, s[name][page, h // group, off].double() - 127)[:, None]
                        for x, name in ((k.contiguous(), "k_scales"), (v.contiguous(), "v_scales")))
            k, v = k.double(), v.double()
            for b in range(0, n, 1024):                                  # queries at a time
                rows = torch.arange(b, min(n, b + 1024), device=DEV)
                seen = at[None] <= c + rows[:, None]
                if s["prefix"] is not None:
                    seen = seen | (at < s["prefix"][r])[None]
                if s["q_episodes"] is not None:
                    ask, key = s["q_episodes"][first + rows][:, None], s["k_episodes"][page * p + off][None]
                    seen = seen & ((ask == -1) | (key == -1) | (ask == key))
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
