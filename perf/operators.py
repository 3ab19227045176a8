"""The operators that serve a paged key/value pool, as they are timed and checked on a GPU.

Three operators make one decode step of many requests: `plan` (block tables and slot maps from
the requests' lengths), `append` (QK-norm, RoPE and the scatter of new keys and values into
pages) and `attend` (attention of one new token over the pages). `run` computes them in plain
torch operations, or, where `own` is true, through syrinx_b200.paged. `exact` restates them
request by request in float64.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"


# ---- cases --------------------------------------------------------------------------------

def _attend(name, n, lo, hi, heads, kv_heads, hd, page, q, cache, layout, pick, empty=0):
    c = {"op": "attend", "n": n, "lo": lo, "hi": hi, "heads": heads, "kv_heads": kv_heads, "hd": hd,
         "page": page, "q": q, "cache": cache, "layout": layout, "pick": pick, "empty": empty}
    return {"name": name, **c} if name else c


def _append(name, tokens, run, pad, heads, kv_heads, hd, page, x, cache, layout, norm, interleaved, far):
    c = {"op": "append", "tokens": tokens, "run": run, "pad": pad, "heads": heads, "kv_heads": kv_heads, "hd": hd,
         "page": page, "x": x, "cache": cache, "layout": layout, "norm": norm, "interleaved": interleaved,
         "far": far}
    return {"name": name, **c} if name else c


def _plan(name, n, grow, prompts, drop, longest, page, pick):
    c = {"op": "plan", "n": n, "grow": grow, "prompts": prompts, "drop": drop, "longest": longest,
         "page": page, "pick": pick}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one utterance of a small speech model just after its prompt: latency alone counts
        _attend("attend 1x128 16/8x64 f32", 1, 128, 128, 16, 8, 64, 64, "f32", "f32", "hnd", 1),
        # 14 query heads over 2 kv heads (a group of 7): eight short dialogue turns of odd lengths
        _attend("attend 8x~200 14/2x64 bf16", 8, 65, 391, 14, 2, 64, 16, "bf16", "bf16", "nhd", 2),
        # eight utterances per GPU at the 4B shape, 256..1536 positions, f32 activations over 16-bit pages
        _attend("attend 8x~900 32/8x128 f32/bf16", 8, 256, 1536, 32, 8, 128, 64, "f32", "bf16", "hnd", 3),
        # one long utterance in latency mode, exact f32 pages
        _attend("attend 1x8192 32/8x128 f32", 1, 8192, 8192, 32, 8, 128, 64, "f32", "f32", "hnd", 4),
        # a serving batch of very uneven requests, one slot of it empty
        _attend("attend 64x1..4099 32/8x128 bf16", 64, 1, 4099, 32, 8, 128, 16, "bf16", "bf16", "nhd", 5, 1),
        # the largest: long documents side by side
        _attend("attend 32x~20000 32/8x128 bf16", 32, 8001, 32768, 32, 8, 128, 64, "bf16", "bf16", "hnd", 6),
        # a decode step's new rows: one token of each of eight utterances
        _append("append 8 32/8x128 f32/bf16", 8, 1, 0, 32, 8, 128, 64, "f32", "bf16", "hnd", True, True, 1536),
        # a prompt of 509 tokens in a buffer of 512, rotate-half, no norm
        _append("append 509 14/2x64 f32", 509, 509, 3, 14, 2, 64, 64, "f32", "f32", "hnd", False, False, 1024),
        # prompts of many requests at once, half precision throughout
        _append("append 16384 32/8x128 bf16", 16384, 700, 0, 32, 8, 128, 16, "bf16", "bf16", "nhd", True, False, 32768),
        # a decode step's bookkeeping: every one of eight utterances grows by a token
        _plan("plan 8 decode", 8, 8, 0, 0, 1536, 64, 7),
        # continuous batching: most grow by one, some arrive with prompts, some leave
        _plan("plan 256 mixed", 256, 220, 12, 20, 4096, 16, 8),
        # a large fleet of short pages
        _plan("plan 2048 mixed", 2048, 1800, 97, 131, 8192, 16, 9),
    ]


def _between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "plan"])
    types = rng.choice([("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
    heads, kv_heads = rng.choice([(16, 8), (14, 2), (32, 8), (4, 2), (8, 8), (16, 2), (8, 1), (16, 1), (30, 10), (5, 1)])
    hd = rng.choice([32, 64, 64, 128, 128, 128, 256])
    if heads // kv_heads > 8 and hd == 256:
        hd = 128
    page = rng.choice([8, 16, 16, 32, 64, 64, 128])
    layout = rng.choice(["hnd", "nhd"])
    if kind == "attend":
        n = _between(rng, 1, 96)
        row = 2 * kv_heads * hd * SIZE[types[1]]
        most = min(32768, 1_500_000_000 // (row * n), 2_000_000_000 // (4 * heads * n))
        hi = _between(rng, 1, max(2, most))
        lo = _between(rng, 1, hi)
        return _attend("", n, lo, hi, heads, kv_heads, hd, page, types[0], types[1], layout, rng.randrange(1 << 30),
                       rng.choice([0, 0, 1, 2]) if n > 2 else 0)
    if kind == "append":
        tokens = _between(rng, 1, 9000)
        run = rng.choice([1, _between(rng, 1, tokens)])
        return _append("", tokens, run, rng.choice([0, 0, 1, 7]), heads, kv_heads, hd, page, types[0], types[1],
                       layout, rng.random() < 0.5, rng.random() < 0.5, run + _between(rng, 64, 32768))
    n = _between(rng, 1, 2000)
    drop, prompts = rng.randrange(n // 8 + 1), rng.randrange(n // 16 + 1)
    return _plan("", n, rng.randrange(n - drop - prompts + 1), prompts, drop, _between(rng, 16, 8192), page,
                 rng.randrange(1 << 30))


def _lens(c):
    """The requests' lengths of an attend case: spread over [lo, hi], their logarithm where that spans much."""
    r = random.Random(c["pick"])
    lens = [c["hi"]] + [_between(r, c["lo"], c["hi"]) if c["hi"] > 16 * c["lo"] else r.randint(c["lo"], c["hi"])
                        for _ in range(c["n"] - 1)]
    r.shuffle(lens)
    for i in r.sample(range(c["n"]), c["empty"]):
        lens[i] = 0
    return lens


def _changes(c):
    """(cached lengths, changes) of a plan case: grown by one, arrived with a prompt, left, or idle."""
    r = random.Random(c["pick"])
    n, longest = c["n"], c["longest"]
    kinds = ["grow"] * c["grow"] + ["prompt"] * c["prompts"] + ["drop"] * c["drop"]
    kinds += ["idle"] * (n - len(kinds))
    r.shuffle(kinds)
    lens, delta = [], []
    for kind in kinds:
        if kind == "prompt":
            lens.append(0)
            delta.append(r.randint(1, max(1, longest // 8)))
        else:
            lens.append(r.randint(1, max(1, longest - 1)) if kind != "idle" else r.randint(0, longest))
            delta.append({"grow": 1, "drop": -lens[-1], "idle": 0}[kind])
    return lens, delta


def _pages(length, page):
    return (length + page - 1) // page


# ---- inputs -------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 11)
    return g


def _cache(c, n_pages, g):
    """K or V pages: [pages, kv heads, page, hd] ("hnd") or [pages, page, kv heads, hd] ("nhd")."""
    shape = ((n_pages, c["kv_heads"], c["page"], c["hd"]) if c["layout"] == "hnd"
             else (n_pages, c["page"], c["kv_heads"], c["hd"]))
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32 if c["cache"] == "f32" else
                       torch.bfloat16 if c["cache"] == "bf16" else torch.float16)


def prepare(case, seed):
    g = _gen(seed)
    return {"attend": _prepare_attend, "append": _prepare_append, "plan": _prepare_plan}[case["op"]](case, g)


def _prepare_attend(c, g):
    lens = _lens(c)
    need = [_pages(x, c["page"]) for x in lens]
    n_pages, width = sum(need) + 3, max(need + [1]) + 1
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    held = torch.tensor(need, device=DEV)
    col = torch.arange(width, device=DEV)
    mine = col[None, :] < held[:, None]
    table = torch.zeros((c["n"], width), dtype=torch.int32, device=DEV)
    table[mine] = ids[: sum(need)]
    qt = DTYPES[c["q"]]
    q = (1.5 * torch.randn((c["n"], c["heads"], c["hd"]), generator=g, device=DEV)).to(qt)
    return {"case": c, "q": q, "k": _cache(c, n_pages, g), "v": _cache(c, n_pages, g), "table": table,
            "lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "scale": 1.0 / math.sqrt(c["hd"]),
            "longest": max(lens), "out": torch.empty_like(q),
            "lse": torch.empty((c["n"], c["heads"]), dtype=torch.float32, device=DEV)}


def _prepare_append(c, g):
    T, rows = c["tokens"], c["tokens"] + c["pad"]
    H, Hkv, hd = c["heads"], c["kv_heads"], c["hd"]
    # each request's rows are `run` consecutive positions, in pages of its own
    run, ps = c["run"], c["page"]
    requests, each = (T + run - 1) // run, _pages(run + ps - 1, ps)
    n_pages = requests * each + 2
    ids = torch.randperm(n_pages, generator=g, device=DEV)
    j = torch.arange(T, device=DEV)
    first = torch.randint(0, c["far"] - run + 1, (requests,), generator=g, device=DEV)
    at = first[j // run] % ps + j % run
    slots = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    slots[:T] = (ids[j // run * each + at // ps] * ps + at % ps).to(torch.int32)
    pos = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    pos[:T] = (first[j // run] + j % run).to(torch.int32)
    inv = 1.0 / (1e6 ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd))
    ang = torch.arange(c["far"], device=DEV, dtype=torch.float64)[:, None] * inv[None, :]
    x = torch.randn((rows, (H + 2 * Hkv) * hd), generator=g, device=DEV).to(DTYPES[c["x"]])
    s = {"case": c, "x": x, "slots": slots, "pos": pos, "cos": ang.cos().float(), "sin": ang.sin().float(),
         "k": _cache(c, n_pages, g), "v": _cache(c, n_pages, g), "q_norm": None, "k_norm": None,
         "out": torch.zeros((rows, H * hd), dtype=x.dtype, device=DEV)}
    if c["norm"]:
        s["q_norm"] = 0.5 + torch.rand(hd, generator=g, device=DEV)
        s["k_norm"] = 0.5 + torch.rand(hd, generator=g, device=DEV)
    return s


def _prepare_plan(c, g):
    lens, delta = _changes(c)
    ps, n = c["page"], c["n"]
    held = [_pages(x, ps) for x in lens]
    after = [_pages(max(0, x + d), ps) for x, d in zip(lens, delta)]
    tokens = sum(max(0, d) for d in delta)
    n_free = sum(max(0, b - a) for a, b in zip(held, after)) + 5
    n_pages, width = sum(held) + n_free, max(held + after) + 1
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    table[torch.arange(width, device=DEV)[None, :] < torch.tensor(held, device=DEV)[:, None]] = ids[n_free:]
    free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    free[:n_free] = ids[:n_free]
    most = tokens + tokens // 8 + 1  # a buffer that a program keeps is longer than one step's tokens
    i32 = {"dtype": torch.int32, "device": DEV}
    return {"case": c, "lens": torch.tensor(lens, **i32), "delta": torch.tensor(delta, **i32),
            "n_free": torch.tensor([n_free], **i32), "table": table, "free": free,
            "lens_out": torch.empty(n, **i32), "n_free_out": torch.empty(1, **i32), "slots": torch.empty(most, **i32),
            "seqs": torch.empty(most, **i32), "pos": torch.empty(most, **i32), "starts": torch.empty(n + 1, **i32),
            "status": torch.empty(4, **i32)}


# ---- one pass -----------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"attend": _own_attend, "append": _own_append, "plan": _own_plan}[op](state)
    return {"attend": _plain_attend, "append": _plain_append, "plan": _plain_plan}[op](state)


def _own_attend(s):
    from syrinx_b200 import paged

    paged.attend(s["q"], s["k"], s["v"], s["table"], s["lens"], scale=s["scale"], layout=s["case"]["layout"],
                 out=s["out"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _own_append(s):
    from syrinx_b200 import paged

    c = s["case"]
    paged.append(s["x"], s["k"], s["v"], s["slots"], n_heads=c["heads"], positions=s["pos"], cos=s["cos"], sin=s["sin"],
                 interleaved=c["interleaved"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, layout=c["layout"],
                 out=s["out"])
    return {"q": s["out"], "k": s["k"], "v": s["v"]}


def _own_plan(s):
    from syrinx_b200 import paged

    paged.plan(s["lens"], s["delta"], s["table"], s["free"], s["n_free"], page_size=s["case"]["page"],
               slots=s["slots"], tok_seq=s["seqs"], tok_pos=s["pos"], starts=s["starts"], lens_out=s["lens_out"],
               n_free_out=s["n_free_out"], status=s["status"])
    return _planned(s)


def _planned(s):
    return {k: s[k] for k in ("table", "free", "lens_out", "n_free_out", "slots", "seqs", "pos", "starts", "status")}


def _plain_attend(s):
    c = s["case"]
    n, H, Hkv, hd, ps = c["n"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    P = max(1, _pages(s["longest"], ps))
    ids = s["table"][:, :P].long()
    k, v = s["k"][ids], s["v"][ids]  # [n, P, kv heads, page, hd] or [n, P, page, kv heads, hd]
    order = (0, 2, 1, 3, 4) if c["layout"] == "hnd" else (0, 3, 1, 2, 4)
    k = k.permute(order).reshape(n, Hkv, P * ps, hd).float()
    v = v.permute(order).reshape(n, Hkv, P * ps, hd).float()
    q = s["q"].float().view(n, Hkv, H // Hkv, hd)
    ok = (torch.arange(P * ps, device=q.device)[None, :] < s["lens"][:, None]).view(n, 1, 1, P * ps)
    score = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).masked_fill(~ok, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - top.clamp_min(-3e38))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v) / total.clamp_min(1e-30)
    lse = top + total.log()
    return {"out": out.view(n, H, hd).to(s["q"].dtype), "lse": lse.view(n, H)}


def _rotated(x, cos, sin, interleaved):
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_append(s):
    c = s["case"]
    H, Hkv, hd, ps = c["heads"], c["kv_heads"], c["hd"], c["page"]
    rows = s["x"].shape[0]
    q, k, v = s["x"].float().view(rows, H + 2 * Hkv, hd).split((H, Hkv, Hkv), 1)
    if c["norm"]:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["q_norm"]
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["k_norm"]
    at = s["pos"].clamp_min(0).long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q, k = _rotated(q, cos, sin, c["interleaved"]), _rotated(k, cos, sin, c["interleaved"])
    live = s["slots"] >= 0
    s["out"].copy_(torch.where(live[:, None], q.reshape(rows, H * hd).to(s["x"].dtype), s["out"]))
    # rows without a slot write what the last row that has one writes, to the same place
    row = torch.arange(rows, device=live.device)
    row = torch.where(live, row, (live * row).max())
    slot = s["slots"][row].long()
    page, off = slot // ps, slot % ps
    if c["layout"] == "hnd":
        s["k"][page, :, off] = k[row].to(s["k"].dtype)
        s["v"][page, :, off] = v[row].to(s["v"].dtype)
    else:
        s["k"][page, off] = k[row].to(s["k"].dtype)
        s["v"][page, off] = v[row].to(s["v"].dtype)
    return {"q": s["out"], "k": s["k"], "v": s["v"]}


def _plain_plan(s):
    ps = s["case"]["page"]
    lens, delta, table, free = s["lens"].long(), s["delta"].long(), s["table"], s["free"]
    n_pages, F = free.shape[0], s["n_free"].long()
    after = (lens + delta).clamp_min(0)
    held, need = (lens + ps - 1) // ps, (after + ps - 1) // ps
    give, take = (held - need).clamp_min(0), (need - held).clamp_min(0)
    first = lambda x: x.cumsum(0) - x  # noqa: E731
    G, T = give.sum(), take.sum()
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    giving = (col >= need[:, None]) & (col < held[:, None])
    to = torch.where(giving, F + first(give)[:, None] + col - need[:, None], n_pages)
    stack = torch.cat((free, free[:1])).scatter(0, to.flatten(), table.flatten())
    taking = (col >= held[:, None]) & (col < need[:, None])
    at = torch.where(taking, F + G - 1 - first(take)[:, None] - (col - held[:, None]), 0)
    table.copy_(torch.where(taking, stack[at], table))
    place = torch.arange(n_pages, device=free.device)
    free.copy_(torch.where((place >= F) & (place < F + G - T), stack[:n_pages], free))
    fresh = delta.clamp_min(0)
    total = fresh.sum()
    starts = torch.cat((first(fresh), total[None]))
    j = torch.arange(s["slots"].shape[0], device=free.device)
    live = j < total
    seq = (torch.searchsorted(starts, j, right=True) - 1).clamp_max(lens.shape[0] - 1)
    pos = torch.where(live, lens[seq] + j - starts[seq], 0)
    slot = table[seq, pos // ps] * ps + pos % ps
    s["slots"].copy_(torch.where(live, slot, -1))
    s["seqs"].copy_(torch.where(live, seq, -1))
    s["pos"].copy_(torch.where(live, pos, -1))
    s["starts"].copy_(starts)
    s["lens_out"].copy_(after)
    s["n_free_out"].copy_(F + G - T)
    s["status"].copy_(torch.stack((0 * total, total, T, F[0] + G - T)))
    return _planned(s)


# ---- what a pass cannot do without ----------------------------------------------------------

def work(c):
    if c["op"] == "attend":
        lens = _lens(c)
        keys = sum(lens)
        b = 2 * keys * c["kv_heads"] * c["hd"] * SIZE[c["cache"]] + 2 * c["n"] * c["heads"] * c["hd"] * SIZE[c["q"]]
        b += 4 * c["n"] * c["heads"] + 4 * c["n"] + 4 * sum(_pages(x, c["page"]) for x in lens)
        return {"bytes": b, "flops": 4 * keys * c["heads"] * c["hd"]}
    if c["op"] == "append":
        T, H, Hkv, hd = c["tokens"], c["heads"], c["kv_heads"], c["hd"]
        b = T * ((H + 2 * Hkv) + H) * hd * SIZE[c["x"]] + 2 * T * Hkv * hd * SIZE[c["cache"]]
        b += 8 * (T + c["pad"]) + 4 * min(T, c["far"]) * hd
        return {"bytes": b, "flops": T * (H + Hkv) * hd * (3 + (4 if c["norm"] else 0))}
    lens, delta = _changes(c)
    held = [_pages(x, c["page"]) for x in lens]
    after = [_pages(max(0, x + d), c["page"]) for x, d in zip(lens, delta)]
    tokens = sum(max(0, d) for d in delta)
    moved = sum(abs(a - b) for a, b in zip(held, after))
    b = 16 * c["n"] + 12 * (tokens + tokens // 8 + 1) + 8 * moved + 4 * sum(d > 0 for d in delta) + 28
    return {"bytes": b, "flops": 0}


# ---- the definitions in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    """What run() returns, by the definition of each operator in float64; None for whole numbers."""
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    return _exact_attend(s) if case["op"] == "attend" else _exact_append(s)


def _exact_attend(s):
    c = s["case"]
    G = c["heads"] // c["kv_heads"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device=DEV)
    for i, length in enumerate(s["lens"].tolist()):
        if length == 0:
            continue
        ids = s["table"][i, : _pages(length, c["page"])].long()
        for h in range(c["kv_heads"]):
            if c["layout"] == "hnd":
                k, v = s["k"][ids, h], s["v"][ids, h]
            else:
                k, v = s["k"][ids, :, h], s["v"][ids, :, h]
            k = k.reshape(-1, c["hd"])[:length].double()
            v = v.reshape(-1, c["hd"])[:length].double()
            sc = q[i, h * G:(h + 1) * G] @ k.T * s["scale"]
            lse[i, h * G:(h + 1) * G] = torch.logsumexp(sc, -1)
            out[i, h * G:(h + 1) * G] = torch.softmax(sc, -1) @ v
    return {"out": out, "lse": lse}


def _exact_append(s):
    c = s["case"]
    T, H, Hkv, hd, ps = c["tokens"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    x = s["x"][:T].double()
    pos, slots = s["pos"][:T].long(), s["slots"][:T].long()
    out = s["out"].double()
    K, V = s["k"].double(), s["v"].double()
    z = torch.complex(s["cos"].double(), s["sin"].double())[pos]
    for h in range(H + 2 * Hkv):
        y = x[:, h * hd:(h + 1) * hd]
        if h < H + Hkv:
            if c["norm"]:
                gain = s["q_norm"] if h < H else s["k_norm"]
                y = gain.double() * y * torch.rsqrt(y.pow(2).sum(-1, keepdim=True) / hd + 1e-6)
            if c["interleaved"]:
                y = torch.view_as_real(torch.view_as_complex(y.reshape(T, hd // 2, 2).contiguous()) * z).reshape(T, hd)
            else:
                w = torch.complex(y[:, : hd // 2].contiguous(), y[:, hd // 2:].contiguous()) * z
                y = torch.cat((w.real, w.imag), 1)
        if h < H:
            out[:T, h * hd:(h + 1) * hd] = y
            continue
        into, g = (K, h - H) if h < H + Hkv else (V, h - H - Hkv)
        if c["layout"] == "hnd":
            into[slots // ps, g, slots % ps] = y
        else:
            into[slots // ps, slots % ps, g] = y
    return {"q": out, "k": K, "v": V}
