"""The cases that time the paged key/value cache of an autoregressive code generator (qwen3_tts_amd.kvcache.PagedKV): the per-head
norm + rotation that fills it, the attention that reads it (sliding window, first tokens that stay visible), the same over a cache
held in 4 bits, and the operations on its pages.  `run` computes them in plain torch, or with `own` through the package."""
import math
import random

import torch

own = False
DEV = "cuda"
GROUP = 32            # values of a 4-bit row that share a step
EPS = 1e-6


# ---- cases ----------------------------------------------------------------------------------------------------------------------
def _case(name, op, dtype, rows, new, past, heads, kv_heads, dim, page, window=0, sinks=0, rot=None, norm=True, layers=1, kind=""):
    c = dict(op=op, dtype=dtype, rows=rows, new=new, past=past, heads=heads, kv_heads=kv_heads, dim=dim, page=page, window=window,
             sinks=sinks, rot=dim if rot is None else rot, norm=norm, layers=layers, kind=kind)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one generated token for each of 64 requests: latency of the step's first operator
        _case("append step bf16", "append", "bf16", 64, 1, 2000, 16, 8, 128, 32),
        # prompts of 24 requests enter the cache at once
        _case("append prompts bf16", "append", "bf16", 24, 2000, 0, 16, 8, 128, 32),
        # the codec transformer's own head layout, without head norms, single precision, odd lengths
        _case("append f32 ragged", "append", "f32", 7, 331, 45, 16, 16, 64, 16, norm=False),
        # prompts into a 4-bit cache, and their values read back
        _case("append prompts int4", "append", "int4", 16, 1000, 37, 16, 8, 128, 32),
        # a generation step over full contexts, as many requests as memory traffic needs
        _case("attend step bf16", "attend", "bf16", 32, 1, 16000, 16, 8, 128, 32),
        # ONE request far into a long-form text, windowed with four first tokens: latency
        _case("attend step window", "attend", "bf16", 1, 1, 100000, 16, 8, 128, 32, window=4096, sinks=4),
        # prompts of mixed length, causal; and a longer one under a window: the matrix-bound side
        _case("attend prompts bf16", "attend", "bf16", 6, 4000, 500, 16, 8, 128, 32, window=2048, sinks=4),
        # the codec transformer's heads and window (72), single precision
        _case("attend f32 window 72", "attend", "f32", 5, 701, 90, 16, 16, 64, 16, window=72),
        # a generation step over 4-bit contexts: small (latency) and large (traffic)
        _case("attend step int4 small", "attend", "int4", 8, 1, 700, 16, 8, 128, 32),
        _case("attend step int4", "attend", "int4", 64, 1, 16000, 16, 8, 128, 32),
        # 120 requests start from 8 cached voice prompts: shared pages, copies of the partly filled ones
        _case("fork prompts", "pages", "bf16", 128, 1, 400, 16, 8, 128, 32, layers=16, kind="fork"),
        # half of the requests of a pool have ended: the live pages move to its front
        _case("compact pool", "pages", "bf16", 64, 1, 900, 16, 8, 128, 32, layers=16, kind="compact"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "pages"])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "pages":
        kind = rng.choice(["fork", "compact", "step"])
        return _case(None, op, rng.choice(["bf16", "int4", "f32"]), rng.randint(3, 128), 1, _log(rng, 20, 900), 8, rng.randint(1, 8),
                     rng.choice([64, 128]), max(page, 16), layers=rng.randint(1, 12), kind=kind, window=rng.randint(1, 300), sinks=rng.randint(0, 40))
    dtype = rng.choice(["bf16", "bf16", "int4", "f32"])
    dim = rng.choice([64, 128, 256] if dtype == "int4" else [16, 64, 80, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7])
    window, sinks = (0, 0) if rng.random() < 0.3 else (_log(rng, 1, 5000), rng.choice([0, 1, 4, 37, 128]))
    if rng.random() < 0.5:           # a step: one new token a request
        rows, new, past = _log(rng, 1, 96), 1, _log(rng, 1, 9000)
        past = min(past, int(1e9 / (rows * kv_heads * dim * 8)))
    else:                            # prompts, or pieces of them
        rows, new, past = rng.randint(1, 9), _log(rng, 2, 1500), rng.choice([0, _log(rng, 1, 1500)])
        rows = max(1, min(rows, int(1e11 / (4.0 * dim * heads * new * (new + past)))))
    rot = dim if dtype == "int4" or dim < 32 else rng.choice([dim, dim, dim // 2])
    return _case(None, op, dtype, rows, new, past, heads, kv_heads, dim, page, window, sinks, rot, rng.random() < 0.7)


def _lengths(c):
    """(tokens in the cache, the new ones among them) of each request: by the case alone, from near the longest down to a fifth."""
    r = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    new = [1 if c["new"] == 1 else c["new"] if i == 0 else r.randint(max(1, c["new"] // 5), c["new"]) for i in range(c["rows"])]
    past = [c["past"] if i == 0 else r.randint(c["past"] // 5, c["past"]) for i in range(c["rows"])]
    return [p + n for p, n in zip(past, new)], new


def _visible(length, new, window, sinks):
    """(pairs of a query and a key it sees, keys seen by any query) of one request."""
    pairs, first = 0, length - new
    for p in range(first, length):
        w = p + 1 if not window else min(window, p + 1)
        pairs += w + (min(sinks, p + 1 - w) if window else 0)
    lo = max(0, first - window + 1) if window else 0
    return pairs, length - lo + min(sinks, lo)


def work(c):
    lens, new = _lengths(c)
    T, D, H, G = sum(new), c["dim"], c["heads"], c["kv_heads"]
    act = 4 if c["dtype"] == "f32" else 2
    held = {"f32": 4.0, "bf16": 2.0, "int4": 0.5 + 2.0 / GROUP}[c["dtype"]]
    if c["op"] == "append":
        out = T * G * D * 2 * act if c["dtype"] == "int4" else 0          # the 4-bit values, read back
        return {"bytes": T * D * (2 * H * act + 2 * G * (act + held)) + out + T * c["rot"] * 4, "flops": T * D * (H + G) * 8}
    if c["op"] == "attend":
        seen = [_visible(a, b, c["window"], c["sinks"]) for a, b in zip(lens, new)]
        return {"bytes": 2 * T * H * D * act + sum(k for _, k in seen) * 2 * G * D * held, "flops": 4.0 * D * H * sum(p for p, _ in seen)}
    page = 2.0 * c["layers"] * G * c["page"] * D * held
    meta = 8.0 * c["rows"]
    if c["kind"] == "fork":
        parents = max(1, c["rows"] // 16)
        part = sum(1 for i in range(c["rows"] - parents) if lens[i % parents] % c["page"])
        shared = sum(lens[i % parents] // c["page"] for i in range(c["rows"] - parents))
        return {"bytes": 2 * page * part + meta + 12.0 * shared, "flops": 0}
    if c["kind"] == "compact":
        return {"bytes": 2 * page * _moved(c) + 8.0 * _pool(c)["pages"], "flops": 0}
    return {"bytes": meta * 4 + 8.0 * _pool(c)["pages"], "flops": 0}


# ---- what a program has in hand ---------------------------------------------------------------------------------------------------
def _pool(c):
    """Where the requests' pages lie: table rows (lists) and counts, by the case alone.  Pages are handed out in a shuffled order, as
    after hours of requests that come and go."""
    lens, new = _lengths(c)
    r = random.Random(len(lens) * 7919 + sum(lens))
    ps = c["page"]
    fork = c["op"] == "pages" and c["kind"] == "fork"
    parents = max(1, c["rows"] // 16)
    used = [0 if fork and i >= parents else -(-n // ps) for i, n in enumerate(lens)]
    if fork:
        lens = [n if i < parents else 0 for i, n in enumerate(lens)]
    pages = sum(used) + c["rows"] + 3 + sum(used) // 8
    ids = list(range(pages))
    r.shuffle(ids)
    table, at = [], 0
    for n in used:
        table.append(ids[at:at + n])
        at += n
    if c["op"] == "pages" and c["kind"] == "compact":        # every second request has ended
        table = [t if i % 2 == 0 else [] for i, t in enumerate(table)]
        lens = [n if i % 2 == 0 else 0 for i, n in enumerate(lens)]
    return dict(lens=lens, new=new, table=table, pages=pages, width=max(-(-(max(lens) + 1) // ps), max(used)) + 1)


def _moved(c):
    live = sorted(p for t in _pool(c)["table"] for p in t)
    return sum(1 for p in live if p >= len(live))


def _values(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    p = _pool(c)
    act = torch.float32 if c["dtype"] == "f32" else torch.bfloat16
    L, P, G, ps, D, H = c["layers"], p["pages"], c["kv_heads"], c["page"], c["dim"], c["heads"]
    s = dict(c=c, act=act, p=p)
    if c["dtype"] == "int4":
        for n in "kv":
            low, high = (torch.randint(1, 16, (L, P, G, ps, D // 2), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2))
            s[n] = high.mul_(16).add_(low)                    # values -7 .. 7, held as 1 .. 15
            s[n + "_scale"] = (torch.rand((L, P, G, ps, D // GROUP), generator=g, device=DEV) * 0.3 + 0.15).to(torch.bfloat16)
    else:
        for n in "kv":
            s[n] = _values(g, (L, P, G, ps, D), act)
        s["k_scale"] = s["v_scale"] = None
    table = torch.full((c["rows"], p["width"]), -1, dtype=torch.int32)
    refs = torch.zeros(P, dtype=torch.int32)
    for i, t in enumerate(p["table"]):
        table[i, : len(t)] = torch.tensor(t, dtype=torch.int32)
        refs[torch.tensor(t, dtype=torch.long)] += 1
    s["table0"], s["refs0"], s["lens0"] = table.to(DEV), refs.to(DEV), torch.tensor(p["lens"], dtype=torch.int32, device=DEV)
    s["table"], s["refs"], s["lens"] = s["table0"].clone(), s["refs0"].clone(), s["lens0"].clone()
    s["status"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    s["kv"] = None                                            # the program's handle: run() makes it on its first pass
    if c["op"] == "pages":
        parents = max(1, c["rows"] // 16)
        order = torch.randperm(c["rows"], generator=g, device=DEV).to(torch.int32)
        s["rows"] = order if c["kind"] == "step" else torch.arange(c["rows"], dtype=torch.int32, device=DEV)
        s["children"] = torch.arange(parents, c["rows"], dtype=torch.int32, device=DEV)
        s["parents"] = (s["children"] - parents) % parents
        return s
    T = sum(p["new"])
    s["rows"] = torch.arange(c["rows"], dtype=torch.int32, device=DEV)
    s["offsets"] = None if c["new"] == 1 else torch.tensor([0] + p["new"], dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)
    if c["op"] == "attend":
        s["q"] = _values(g, (T, H, D), torch.float32).mul_(2).to(act)
        return s
    qkv = _values(g, (T, (H + 2 * G) * D), torch.float32).mul_(3).to(act)      # one projection's output; q, k and v are views of it
    s["q"], s["kn"], s["vn"] = (x.view(T, -1, D) for x in qkv.split([H * D, G * D, G * D], dim=1))
    s["qw"], s["kw"] = (torch.rand(D, generator=g, device=DEV) + 0.5 for _ in range(2)) if c["norm"] else (None, None)
    R = c["rot"]
    ang = torch.arange(p["width"] * ps, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    s["cos"], s["sin"] = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    return s


# ---- the operators ------------------------------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from qwen3_tts_amd.kvcache import PagedKV
    c, kv = s["c"], s["kv"]
    if kv is None:
        kv = s["kv"] = PagedKV.from_tensors(s["k"], s["v"], s["table"], s["lens"], s["refs"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                            status=s["status"])
    if c["op"] == "append":
        q = kv.append(0, s["q"], s["kn"], s["vn"], s["rows"], s["offsets"], q_weight=s["qw"], k_weight=s["kw"], rope=(s["cos"], s["sin"]), eps=EPS)
        k, v = kv.gather(0, s["rows"], s["offsets"], tokens=q.shape[0], dtype="bf16") if c["dtype"] == "int4" else (kv.k, kv.v)
        return {"q": q, "k": k, "v": v}
    if c["op"] == "attend":
        return kv.attend(0, s["q"], s["rows"], s["offsets"], window=c["window"], sinks=c["sinks"])
    kv.table.copy_(s["table0"])
    kv.refs.copy_(s["refs0"])
    kv.lens.copy_(s["lens0"])
    out = {"table": kv.table, "refs": kv.refs, "lens": kv.lens}
    if c["kind"] == "fork":
        kv.fork(s["parents"], s["children"])
    elif c["kind"] == "compact":
        kv.compact()
    else:
        kv.trim(s["rows"], c["window"], c["sinks"])
        kv.reserve(s["rows"])
        return out
    return dict(out, **_page_values(s)) if c["dtype"] == "int4" else dict(out, k=kv.k, v=kv.v)


def _page_values(s):
    """4-bit pools: the bytes that were moved, as the whole numbers they stand for (moving them computes nothing)."""
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _unpack(x, scale):
    """4-bit rows [.., D/2] and steps [.., D/32] -> float32 [.., D]: byte [m][g] of a row holds values 32 g + m (low half) and 32 g + 16 + m."""
    D = x.shape[-1] * 2
    b = x.reshape(x.shape[:-1] + (16, D // GROUP)).transpose(-1, -2)
    n = torch.stack([b % 16, b // 16], dim=-2).float() - 8.0                    # [.., D/32, 2, 16]
    return (n * scale.float()[..., None, None]).reshape(x.shape[:-1] + (D,))


def _pack(x):
    """float32 [.., D] -> (bytes [.., D/2], steps [.., D/32]): step = absmax / 7 in bfloat16, values to the nearest multiple."""
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // GROUP, 2, 16))
    step = (g.abs().amax((-1, -2)) / 7.0).to(torch.bfloat16)
    n = torch.where(step[..., None, None] > 0, torch.round(g / step.float()[..., None, None]), torch.zeros_like(g)).clamp(-7, 7) + 8
    b = (n[..., 0, :] + 16 * n[..., 1, :]).to(torch.uint8)                       # [.., D/32, 16]
    return b.transpose(-1, -2).reshape(x.shape[:-1] + (x.shape[-1] // 2,)), step


def _where(s):
    """Request, position, page and slot of every new token."""
    c, ps = s["c"], s["c"]["page"]
    if s["offsets"] is None:
        b = torch.arange(s["rows"].shape[0], device=DEV)
        back = torch.ones_like(b)
    else:
        off = s["offsets"].long()
        t = torch.arange(s["q"].shape[0], device=DEV)
        b = torch.searchsorted(off, t, right=True) - 1
        back = off[b + 1] - t
    row = s["rows"].long()[b]
    pos = s["lens"].long()[row] - back
    return b, row, pos, s["table"].long()[row, pos // ps], pos % ps


def _run_plain(s):
    c = s["c"]
    if c["op"] == "append":
        return _append_plain(s)
    if c["op"] == "attend":
        return _attend_plain(s)
    s["table"].copy_(s["table0"])
    s["refs"].copy_(s["refs0"])
    s["lens"].copy_(s["lens0"])
    out = {"table": s["table"], "refs": s["refs"], "lens": s["lens"]}
    if c["kind"] == "step":
        _trim_plain(s)
        _reserve_plain(s)
        return out
    pairs = _fork_plain(s) if c["kind"] == "fork" else _compact_plain(s)
    src, dst = pairs
    for n in ("k", "v", "k_scale", "v_scale"):
        if s[n] is not None:
            s[n][:, dst] = s[n][:, src]
    return dict(out, **_page_values(s)) if c["dtype"] == "int4" else dict(out, k=s["k"], v=s["v"])


def _append_plain(s):
    c = s["c"]
    b, row, pos, page, slot = _where(s)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    R = c["rot"]

    def turn(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        lo, hi = x[..., : R // 2], x[..., R // 2: R]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., R:]], -1)

    q, k, v = turn(s["q"], s["qw"]), turn(s["kn"], s["kw"]), s["vn"].float()
    if c["dtype"] != "int4":
        s["k"][0, page, :, slot] = k.to(s["act"])
        s["v"][0, page, :, slot] = v.to(s["act"])
        return {"q": q.to(s["act"]), "k": s["k"], "v": s["v"]}
    back = []
    for n, x in (("k", k), ("v", v)):
        s[n][0, page, :, slot], s[n + "_scale"][0, page, :, slot] = _pack(x)
        back.append(_unpack(s[n][0, page, :, slot], s[n + "_scale"][0, page, :, slot]).to(torch.bfloat16))
    return {"q": q.to(s["act"]), "k": back[0], "v": back[1]}


def _attend_plain(s):
    """Every request's keys and values gathered to one padded tensor, one product, a masked softmax, one product."""
    c, p = s["c"], s["p"]
    S, H, G, D, ps = c["rows"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    n, width = max(p["new"]), -(-max(p["lens"]) // ps)
    pages = s["table"].long()[s["rows"].long()][:, :width].clamp(min=0)

    def held(x, scale):
        x = x[0, pages]                                                          # [S, width, G, ps, D]
        x = x.float() if scale is None else _unpack(x, scale[0, pages])
        return x.transpose(2, 3).reshape(S, width * ps, G, D).permute(0, 2, 1, 3)   # [S, G, L, D]

    q = s["q"].float()
    b, row, pos, _, _ = _where(s)
    if s["offsets"] is None:
        i = torch.zeros_like(b)
    else:
        i = torch.arange(q.shape[0], device=DEV) - s["offsets"].long()[b]
    qp = torch.zeros((S, n, H, D), device=DEV)
    qp[b, i] = q
    at = torch.full((S, n), -1, dtype=torch.long, device=DEV)
    at[b, i] = pos
    qp = qp.view(S, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(S, G, (H // G) * n, D)
    x = torch.matmul(qp, held(s["k"], s["k_scale"]).transpose(-1, -2)) / math.sqrt(D)
    t = torch.arange(width * ps, device=DEV)
    see = t <= at[..., None]
    if c["window"]:
        see = see & ((t > at[..., None] - c["window"]) | (t < c["sinks"]))
    x = x.view(S, G, H // G, n, -1).masked_fill_(~see[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    w = torch.exp_(x.sub_(torch.where(m > -math.inf, m, torch.zeros_like(m))))
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(w.view(S, G, (H // G) * n, -1), held(s["v"], s["v_scale"]))
    o = o.view(S, G, H // G, n, D).permute(0, 3, 1, 2, 4).reshape(S, n, H, D)
    return o[b, i].to(s["act"])


def _free_first(refs):
    """Free pages in ascending order, then the others; and how many are free."""
    return torch.sort((refs > 0).to(torch.int32), stable=True).indices, (refs == 0).sum()


def _trim_plain(s):
    c, rows, ps = s["c"], s["rows"].long(), s["c"]["page"]
    t = s["table"][rows]
    j = torch.arange(t.shape[1], device=DEV)
    gone = (t >= 0) & (j * ps >= c["sinks"]) & ((j + 1) * ps <= (s["lens"][rows] - c["window"])[:, None])
    drop = torch.zeros(s["refs"].shape[0] + 1, dtype=torch.int32, device=DEV)
    drop.index_add_(0, torch.where(gone, t.long(), torch.full_like(t, s["refs"].shape[0]).long()).view(-1), torch.ones(t.numel(), dtype=torch.int32, device=DEV))
    s["refs"].sub_(drop[:-1])
    s["table"][rows] = torch.where(gone, torch.full_like(t, -1), t)


def _reserve_plain(s):
    rows, ps = s["rows"].long(), s["c"]["page"]
    t, old = s["table"][rows], s["lens"][rows]
    j = torch.arange(t.shape[1], device=DEV)
    need = (j >= (-(-old // ps))[:, None]) & (j < (-(-(old + 1) // ps))[:, None])
    rank = need.view(-1).cumsum(0).view(need.shape) - 1
    order, free = _free_first(s["refs"])
    got = need & (rank < free)
    ids = order[rank.clamp(0, order.shape[0] - 1)].to(torch.int32)
    s["table"][rows] = torch.where(got, ids, t)
    mark = torch.zeros(s["refs"].shape[0] + 1, dtype=torch.int32, device=DEV)
    mark[torch.where(got, ids.long(), torch.full_like(rank, s["refs"].shape[0])).view(-1)] = 1
    s["refs"].add_(mark[:-1])
    s["lens"][rows] = old + 1


def _fork_plain(s):
    """Full pages shared, a partly filled last page copied to the lowest free page: the (source, destination) pairs."""
    up, ch, ps = s["parents"].long(), s["children"].long(), s["c"]["page"]
    t, n = s["table"][up], s["lens"][up]
    j = torch.arange(t.shape[1], device=DEV)
    full = j < (n // ps)[:, None]
    part = (j == (n // ps)[:, None]) & (n % ps > 0)[:, None]
    src = torch.masked_select(t, part).long()
    order, _ = _free_first(s["refs"])
    dst = order[: src.shape[0]]
    new = torch.where(full, t, torch.full_like(t, -1))
    new[part] = dst.to(torch.int32)
    s["refs"].index_add_(0, torch.masked_select(new, new >= 0).long(), torch.ones(int((new >= 0).sum()), dtype=torch.int32, device=DEV))
    s["table"][ch], s["lens"][ch] = new, n
    return src, dst


def _compact_plain(s):
    """Live pages behind the first `live` ones move, in order, to the holes before them."""
    live = s["refs"] > 0
    count = int(live.sum())
    src = live[count:].nonzero().view(-1) + count
    dst = (~live[:count]).nonzero().view(-1)
    to = torch.arange(live.shape[0], device=DEV)
    to[src] = dst
    t = s["table"]
    t.copy_(torch.where(t >= 0, to[t.long().clamp(min=0)].to(torch.int32), t))
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    return src, dst


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------------------------
def _rows64(s, which, i, tokens):
    """Stored keys or values of request i's positions `tokens`, float64 [tokens, kv heads, dim]."""
    ps, t = s["c"]["page"], torch.as_tensor(tokens, device=DEV)
    ids = torch.tensor(s["p"]["table"][i], device=DEV)[t // ps]
    x = s[which][0][ids, :, t % ps]
    if s["c"]["dtype"] != "int4":
        return x.double()
    st, out = s[which + "_scale"][0][ids, :, t % ps].double(), torch.empty(x.shape[:-1] + (s["c"]["dim"],), dtype=torch.float64, device=DEV)
    for d in range(s["c"]["dim"]):
        byte = x[..., (d % 16) * (s["c"]["dim"] // GROUP) + d // GROUP].long()
        out[..., d] = ((byte >> 4 if d % GROUP >= 16 else byte & 15) - 8).double() * st[..., d // GROUP]
    return out


def exact(case, seed):
    c = dict(case)
    if c["op"] == "pages":
        return None
    s = prepare(case, seed)
    p, D, H, G = s["p"], c["dim"], c["heads"], c["kv_heads"]
    starts = [sum(p["new"][:i]) for i in range(c["rows"])]
    if c["op"] == "attend":
        out = torch.zeros((sum(p["new"]), H, D), dtype=torch.float64, device=DEV)
        for i in range(c["rows"]):
            L, n = p["lens"][i], p["new"][i]
            lo = max(0, L - n - c["window"] + 1) if c["window"] else 0
            seen = list(range(min(c["sinks"], lo))) + list(range(lo, L))
            k, v, t = _rows64(s, "k", i, seen), _rows64(s, "v", i, seen), torch.tensor(seen, device=DEV)
            for a in range(0, n, 512):
                b = min(n, a + 512)
                at = torch.arange(L - n + a, L - n + b, device=DEV)[:, None]
                see = t[None] <= at
                if c["window"]:
                    see &= (at - t[None] < c["window"]) | (t[None] < c["sinks"])
                for h in range(H):
                    x = s["q"][starts[i] + a: starts[i] + b, h].double() @ k[:, h // (H // G)].t() * D ** -0.5
                    w = torch.softmax(torch.where(see, x, torch.full_like(x, -math.inf)), -1)
                    out[starts[i] + a: starts[i] + b, h] = w @ v[:, h // (H // G)]
        return out
    pos = torch.cat([torch.arange(L - n, L, device=DEV) for L, n in zip(p["lens"], p["new"])])
    R = c["rot"]
    angle = s["cos"][pos].double(), s["sin"][pos].double()

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS) * w.double()
        y = x.clone()
        for d in range(R // 2):
            a, b = x[..., d], x[..., d + R // 2]
            co, si = angle[0][:, d, None], angle[1][:, d, None]
            y[..., d], y[..., d + R // 2] = a * co - b * si, b * co + a * si
        return y

    q, new = turned(s["q"], s["qw"]), {"k": turned(s["kn"], s["kw"]), "v": s["vn"].double()}
    if c["dtype"] == "int4":
        for n, x in new.items():
            y = x.view(x.shape[0], G, D // GROUP, GROUP)
            st = (y.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16).double()
            new[n] = ((y / st).round().clamp(-7, 7) * st).reshape(x.shape)
        return {"q": q, "k": new["k"], "v": new["v"]}
    ids = torch.cat([torch.tensor(p["table"][i], device=DEV)[torch.arange(L - n, L, device=DEV) // c["page"]]
                     for i, (L, n) in enumerate(zip(p["lens"], p["new"]))])
    pools = {}
    for n, x in new.items():
        pools[n] = s[n].double()
        for h in range(G):
            pools[n][0, ids, h, pos % c["page"]] = x[:, h]
    return {"q": q, "k": pools["k"], "v": pools["v"]}
