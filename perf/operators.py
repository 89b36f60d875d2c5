"""Measured cases of the paged serving operators: page planning, the paged append and attention over pages.

A serving step of a batch of requests with different lengths is three calls: ``ops.page_plan`` (which page and row
every new token gets), ``ops.paged_append`` (the new K and V rows go there) and ``ops.paged_attend`` (the new tokens
attend to everything their request holds). The cases cover decode steps, speculative checks of a few tokens, chunks
of long prompts and mixed batches. Where ``own`` is false the operators are computed in elementary torch operations.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases -------------------------------------------------------------------------------------------------------

def _plan(name, batch, page, q_lo, q_hi, singles, hist_hi, done, mix):
    return {"name": name, "op": "plan", "batch": batch, "page": page, "q_lo": q_lo, "q_hi": q_hi, "singles": singles,
            "hist_lo": 0, "hist_hi": hist_hi, "done": done, "mix": mix}


def _append(name, tokens, holes, kv_heads, dim, page, dtype, mix):
    return {"name": name, "op": "append", "tokens": tokens, "holes": holes, "kv_heads": kv_heads, "dim": dim,
            "page": page, "dtype": dtype, "mix": mix}


def _attend(name, batch, q_heads, kv_heads, dim, page, q_lo, q_hi, singles, hist_lo, hist_hi, dtype, mix, softcap=0.0,
            alibi=False, window=0, prefix=0):
    return {"name": name, "op": "attend", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "q_lo": q_lo, "q_hi": q_hi, "singles": singles, "hist_lo": hist_lo, "hist_hi": hist_hi,
            "dtype": dtype, "mix": mix, "softcap": softcap, "alibi": alibi, "window": window, "prefix": prefix}


def listed():
    return [
        # the bookkeeping of one decode step of a busy server: every request gets one token, a few slots change hands
        _plan("plan decode 256", 256, 16, 1, 1, 0, 8192, 5, 1),
        # a step that admits prompts next to running requests: tens of thousands of slots
        _plan("plan prompts 32k", 96, 64, 1, 1024, 33, 16384, 9, 2),
        # K and V rows of a decode step of 16 requests: latency alone
        _append("append decode 16", 16, 0, 8, 128, 16, "bf16", 3),
        # a whole prompt chunk with padding rows behind it: bandwidth
        _append("append chunk 16k", 16384, 301, 8, 128, 64, "fp16", 4),
        # one request of a small model, 4096 tokens: the latency of a single decode call
        _attend("decode 1x4096", 1, 16, 8, 128, 16, 1, 1, 1, 4095, 4095, "bf16", 5),
        # eight long requests of uneven length
        _attend("decode 8x32768", 8, 16, 8, 128, 64, 1, 1, 8, 20001, 32767, "bf16", 6),
        # a batch of sixteen with lengths between short and very long: bandwidth and balance
        _attend("decode 16x65536", 16, 32, 8, 128, 256, 1, 1, 16, 1000, 65535, "bf16", 7),
        # checking a few drafted tokens per request, capped scores
        _attend("draft check 8x4", 8, 32, 8, 128, 16, 2, 4, 0, 500, 9000, "fp16", 8, softcap=50.0),
        # one chunk of a long prompt behind what is cached already
        _attend("chunk 2048 on 32k", 1, 32, 8, 128, 64, 2048, 2048, 0, 30720, 30720, "bf16", 9),
        # fresh prompts of a small model without shared heads, distance bias, head size 64
        _attend("prompts alibi", 8, 16, 16, 64, 32, 65, 1500, 0, 0, 0, "fp16", 10, alibi=True),
        # running requests and prompt chunks in one call: five query heads to a KV head, sliding window, capped scores
        _attend("mixed window", 24, 40, 8, 128, 16, 33, 400, 18, 100, 6000, "bf16", 11, softcap=30.0, window=1024),
        # two prompts whose instructions are read in both directions
        _attend("prefix prompts", 2, 8, 2, 128, 16, 150, 333, 0, 0, 40, "bf16", 12, prefix=100),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "decode", "decode", "chunk", "chunk", "mixed"])
    mix = rng.randrange(1, 1 << 20)
    page = 1 << rng.randrange(3, 9)
    if kind == "plan":
        batch = _log(rng, 1, 512)
        c = _plan("", batch, page, 1, _log(rng, 1, max(1, min(2048, 32768 // batch))), rng.randrange(0, batch + 1),
                  _log(rng, 1, 16384), rng.randrange(0, 1 + batch // 4), mix)
    elif kind == "append":
        tokens = _log(rng, 1, 16384)
        c = _append("", tokens, rng.randrange(0, 1 + tokens // 8), rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), page,
                    rng.choice(["bf16", "fp16"]), mix)
    else:
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8])
        dim, dtype = rng.choice([64, 128, 128]), rng.choice(["bf16", "fp16"])
        more = {"softcap": rng.choice([0.0, 0.0, 30.0, 50.0]), "alibi": rng.random() < 0.25,
                "window": rng.choice([0, 0, _log(rng, 16, 4096)]), "prefix": rng.choice([0, 0, _log(rng, 1, 500)])}
        if kind == "decode":
            batch, hist = _log(rng, 1, 64), _log(rng, 1, 32768)
            q = _log(rng, 1, 8)
            hist = max(1, min(hist, 400000 // batch))                 # tokens cached in all
            c = _attend("", batch, kv_heads * group, kv_heads, dim, page, 1, q, rng.randrange(0, batch + 1),
                        rng.randrange(0, hist + 1), hist, dtype, mix, **more)
        elif kind == "chunk":
            batch, q = _log(rng, 1, 4), _log(rng, 16, 1024)
            hist = _log(rng, 1, 8192)
            c = _attend("", batch, kv_heads * group, kv_heads, dim, page, 1 + q // 2, q, 0, 0, hist, dtype, mix, **more)
        else:
            batch, q = _log(rng, 2, 16), _log(rng, 16, 512)
            hist = _log(rng, 1, 4096)
            c = _attend("", batch, kv_heads * group, kv_heads, dim, page, 1, q, rng.randrange(1, batch), 0, hist, dtype,
                        mix, **more)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------

def _lengths(case):
    """Per request: new tokens, and tokens cached before them. They belong to the case, not to the seed."""
    r = random.Random(case["mix"])
    q, hist = [], []
    for b in range(case["batch"]):
        q.append(1 if b < case["singles"] else r.randint(case["q_lo"], case["q_hi"]))
        hist.append(r.randint(case["hist_lo"], case["hist_hi"]))
    order = list(range(case["batch"]))
    r.shuffle(order)
    return [q[i] for i in order], [hist[i] for i in order]


def _ceil(a, b):
    return -(-a // b)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _page_count(case, q, hist):
    return sum(_ceil(a + b, case["page"]) for a, b in zip(q, hist)) + 3


def _prepare_plan(case, g):
    q, hist = _lengths(case)
    P, B = case["page"], case["batch"]
    width = max(_ceil(a + b, P) for a, b in zip(q, hist)) + 1
    num = sum(_ceil(a + b, P) for a, b in zip(q, hist)) + 64
    perm = torch.randperm(num, generator=g, device="cuda").to(torch.int32)
    have = torch.tensor([_ceil(h, P) for h in hist], device="cuda")
    first = torch.cumsum(have, 0) - have
    at = torch.arange(width, device="cuda")[None, :]
    table = torch.where(at < have[:, None], perm[(first[:, None] + at).clamp(max=num - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    used = sum(_ceil(h, P) for h in hist)
    free = torch.zeros(num, dtype=torch.int32, device="cuda")
    free[: num - used] = perm[used:]
    done = torch.zeros(B, dtype=torch.bool, device="cuda")
    done[torch.randperm(B, generator=g, device="cuda")[: case["done"]]] = True
    return {"case": case, "kv_len": _ints(hist), "q_len": _ints(q), "table": table.contiguous(), "free": free,
            "count": _ints([num - used]), "done": done, "capacity": sum(q) + 5}


def _prepare_append(case, g):
    P, H, D, n = case["page"], case["kv_heads"], case["dim"], case["tokens"]
    dt = DTYPES[case["dtype"]]
    pages = _ceil(n, P) + 5
    shape = (pages, H, P, D)
    pools = [torch.randn(shape, generator=g, device="cuda", dtype=dt) for _ in range(2)]
    # runs of neighbouring rows inside pages that are scattered over the pool, as requests leave them
    order = torch.randperm(pages, generator=g, device="cuda")
    t = torch.arange(n, device="cuda") + 3
    slot = order[t // P] * P + t % P
    if case["holes"]:
        slot[n - case["holes"]:] = -1
    # the rows come as the K and V columns of one fused projection: strided views
    kv = torch.randn((n, 2, H, D), generator=g, device="cuda", dtype=dt)
    return {"case": case, "key": kv[:, 0], "value": kv[:, 1], "slot": slot, "pools": pools}


def _prepare_attend(case, g):
    q, hist = _lengths(case)
    P, B, H, D = case["page"], case["batch"], case["kv_heads"], case["dim"]
    dt = DTYPES[case["dtype"]]
    num = _page_count(case, q, hist)
    width = max(_ceil(a + b, P) for a, b in zip(q, hist))
    perm = torch.randperm(num, generator=g, device="cuda").to(torch.int32)
    need = torch.tensor([_ceil(a + b, P) for a, b in zip(q, hist)], device="cuda")
    first = torch.cumsum(need, 0) - need
    at = torch.arange(width, device="cuda")[None, :]
    table = torch.where(at < need[:, None], perm[(first[:, None] + at).clamp(max=num - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    mult = torch.exp(0.5 * torch.randn((H, 1, D), generator=g, device="cuda"))     # outlier channels, as in real caches
    key = torch.empty((num, H, P, D), dtype=dt, device="cuda")
    step = max(1, (1 << 26) // (H * P * D))
    for i in range(0, num, step):
        key[i:i + step] = torch.randn((min(step, num - i), H, P, D), generator=g, device="cuda") * mult
    value = torch.randn((num, H, P, D), generator=g, device="cuda", dtype=dt)
    query = torch.randn((sum(q), case["q_heads"], D), generator=g, device="cuda").to(dt)
    cu = [0]
    for x in q:
        cu.append(cu[-1] + x)
    s = {"case": case, "query": query, "key": key, "value": value, "table": table.contiguous(),
         "kv_len": _ints([a + b for a, b in zip(q, hist)]), "cu": None if max(q) == 1 else _ints(cu), "max_q": max(q),
         "slopes": None, "prefix": None}
    if case["alibi"]:
        n = case["q_heads"]
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, n + 1, device="cuda", dtype=torch.float32) / n)
    if case["prefix"]:
        s["prefix"] = _ints([max(0, case["prefix"] - 7 * b) for b in range(B)])
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + case["mix"])
    return {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend}[case["op"]](case, g)


# ---- plain forms -------------------------------------------------------------------------------------------------

def _plain_plan(s):
    P, cap = s["case"]["page"], s["capacity"]
    old = torch.where(s["done"], 0, s["kv_len"]).long()
    q = s["q_len"].long()
    table, free = s["table"], s["free"]
    W, num = table.shape[1], free.shape[0]
    gone = torch.where(s["done"], (s["kv_len"].long() + P - 1) // P, 0)
    have, need = (old + P - 1) // P, (old + q + P - 1) // P
    take = need - have
    count, back = s["count"].long()[0], gone.sum()
    short = (take.sum() - count - back).clamp(min=0)
    over = (q.sum() - cap).clamp(min=0)
    narrow = (need > W).sum()
    ok = (short + over + narrow) == 0
    # pages of finished requests go on top of the stack, in request order
    j = torch.arange(W, device=q.device)[None, :]
    put = (count + torch.cumsum(gone, 0) - gone)[:, None] + j
    extra = torch.cat((free, free.new_zeros(1)))
    extra.index_put_((torch.where((j < gone[:, None]) & ok, put, num).reshape(-1),), table.reshape(-1))
    free.copy_(extra[:num])
    # new pages come off the top, again in request order
    top = count + back - 1
    at = (torch.cumsum(take, 0) - take)[:, None] + (j - have[:, None])
    new = (j >= have[:, None]) & (j < need[:, None]) & ok
    table.copy_(torch.where(new, free[(top - at).clamp(0, num - 1)], table))
    qe = torch.where(ok, q, 0)
    cu = torch.cat((qe.new_zeros(1), torch.cumsum(qe, 0)))
    n = torch.arange(cap, device=q.device)
    b = torch.searchsorted(cu[1:].contiguous(), n, right=True)
    live = b < q.shape[0]
    bc = b.clamp(max=q.shape[0] - 1)
    pos = torch.where(live, old[bc] + n - cu[bc], -1)
    page = table[bc, (pos.clamp(min=0) // P).clamp(max=W - 1)].long()
    slot = torch.where(live, page * P + pos.clamp(min=0) % P, -1)
    kv = torch.where(ok, old + q, s["kv_len"].long())
    left = torch.where(ok, count + back - take.sum(), count)
    status = torch.stack((short, over, narrow, torch.zeros_like(short)))
    i32 = torch.int32
    return {"cu_q": cu.to(i32), "kv_len": kv.to(i32), "free_count": left.reshape(1).to(i32), "slot": slot,
            "position": pos.to(i32), "request": torch.where(live, b, -1).to(i32), "status": status.to(i32),
            "page_table": table, "free_pages": free}


def _plain_append(s):
    P, slot = s["case"]["page"], s["slot"]
    valid = slot >= 0
    # a row without a place repeats the first row that has one
    src = torch.where(valid, torch.arange(slot.shape[0], device=slot.device), torch.argmax(valid.to(torch.int32)))
    to = slot[src]
    page, row = to // P, to % P
    for pool, rows in zip(s["pools"], (s["key"], s["value"])):
        pool[page, :, row] = rows[src]
    return s["pools"]


def _plain_attend(s):
    case = s["case"]
    P, D, H = case["page"], case["dim"], case["kv_heads"]
    G = case["q_heads"] // H
    B, W = s["table"].shape
    N, T, Q = s["query"].shape[0], W * P, s["max_q"]
    dev = s["query"].device
    kv = s["kv_len"].long()
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(B + 1, device=dev)
    q_len = cu[1:] - cu[:-1]
    ids = s["table"].long()
    k = s["key"][ids].permute(0, 2, 1, 3, 4).reshape(B, H, T, D).float()
    i = torch.arange(Q, device=dev)[None, :]
    rows = (cu[:-1, None] + i).clamp(max=N - 1)                                    # [B,Q]
    q = s["query"][rows].float().reshape(B, Q, H, G, D).permute(0, 2, 3, 1, 4)     # [B,H,G,Q,D]
    x = torch.matmul(q.reshape(B, H, G * Q, D), k.transpose(-1, -2)).reshape(B, H, G, Q, T)
    del k
    x *= 1.0 / math.sqrt(D)
    if case["softcap"]:
        x = torch.tanh(x / case["softcap"]) * case["softcap"]
    p = (kv - q_len)[:, None] + i                                                  # position of each query [B,Q]
    j = torch.arange(T, device=dev)
    if s["slopes"] is not None:
        x -= s["slopes"].reshape(1, H, G, 1, 1) * (p[:, :, None] - j).abs().float()[:, None, None]
    see = j <= p[:, :, None]
    if s["prefix"] is not None:
        see = see | (j < s["prefix"].long()[:, None, None])
    if case["window"]:
        see = see & (j > p[:, :, None] - case["window"])
    see = (see & (j < kv[:, None, None]))[:, None, None]
    x = torch.where(see, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    safe = torch.where(torch.isinf(top), 0.0, top)
    x = torch.exp(x - safe)
    l = x.sum(-1, keepdim=True)
    v = s["value"][ids].permute(0, 2, 1, 3, 4).reshape(B, H, T, D).float()
    v = torch.where((j < kv[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(x.reshape(B, H, G * Q, T), v).reshape(B, H, G, Q, D)
    o = torch.where(l > 0, o / l, 0.0)
    lse = torch.where(l > 0, safe + torch.log(l), -math.inf)[..., 0]
    # back from [B,H,G,Q] to packed rows
    n = torch.arange(N, device=dev)
    b = torch.searchsorted(cu[1:].contiguous(), n, right=True)
    at = n - cu[b]
    out = o.permute(0, 3, 1, 2, 4)[b, at].reshape(N, H * G, D).to(s["query"].dtype)
    return {"out": out, "lse": lse.permute(0, 3, 1, 2)[b, at].reshape(N, H * G)}


# ---- the framework's calls ---------------------------------------------------------------------------------------

def _own_plan(s):
    from kv_cache_b200 import ops
    r = ops.page_plan(s["kv_len"], s["q_len"], s["table"], s["free"], s["count"], s["case"]["page"], s["capacity"],
                      finished=s["done"])
    return {"cu_q": r.cu_q, "kv_len": r.kv_len, "free_count": r.free_count, "slot": r.slot, "position": r.position,
            "request": r.request, "status": r.status, "page_table": s["table"], "free_pages": s["free"]}


def _own_append(s):
    from kv_cache_b200 import ops
    ops.paged_append(s["key"], s["value"], s["slot"], s["pools"][0], s["pools"][1])
    return s["pools"]


def _own_attend(s):
    from kv_cache_b200 import ops
    out, lse = ops.paged_attend(s["query"], s["key"], s["value"], s["table"], s["kv_len"], cu_q=s["cu"], max_q=s["max_q"],
                                softcap=s["case"]["softcap"], slopes=s["slopes"], window=s["case"]["window"],
                                prefix_len=s["prefix"], return_lse=True)
    return {"out": out, "lse": lse}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attend": _own_attend}[op](state)
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[op](state)


# ---- work and exact results --------------------------------------------------------------------------------------

def _seen(case, q, hist, b, i):
    """Half-open range of keys that query i of request b sees; a prefix shorter than the position adds nothing."""
    p = hist + i
    lo = max(0, p - case["window"] + 1) if case["window"] else 0
    pre = max(0, case["prefix"] - 7 * b) if case["prefix"] else 0
    return lo, min(max(p + 1, pre), hist + q)


def work(case):
    if case["op"] == "append":
        rows = case["tokens"] - case["holes"]
        return {"bytes": rows * case["kv_heads"] * case["dim"] * 2 * 2 * 2 + case["tokens"] * 8, "flops": 0}
    q, hist = _lengths(case)
    P, n = case["page"], sum(q)
    if case["op"] == "plan":
        new = sum(_ceil(a + h, P) - _ceil(h, P) for a, h in zip(q, hist))
        return {"bytes": case["batch"] * 17 + (n + 5) * 16 + new * 8, "flops": 0}
    pairs = keys = 0
    for b in range(case["batch"]):
        spans = [_seen(case, q[b], hist[b], b, i) for i in range(q[b])]
        pairs += sum(max(0, hi - lo) for lo, hi in spans)
        keys += max(0, max(hi for _, hi in spans) - min(lo for lo, _ in spans))
    D, H, Hq = case["dim"], case["kv_heads"], case["q_heads"]
    return {"bytes": keys * H * D * 4 + n * Hq * (D * 4 + 4), "flops": 4 * pairs * D * Hq}


def exact(case, seed):
    """From the definition in 64 bits, request by request and head by head."""
    if case["op"] == "plan":
        return None                                      # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        keep = s["slot"] >= 0
        rows = []
        for pool, new in zip(s["pools"], (s["key"], s["value"])):
            pages, H, P, D = pool.shape
            flat = pool.double().permute(0, 2, 1, 3).reshape(pages * P, H, D)
            flat[s["slot"][keep]] = new[keep].double()
            rows.append(flat.reshape(pages, P, H, D).permute(0, 2, 1, 3).contiguous())
        return rows
    q_len, hist = _lengths(case)
    P, D, H = case["page"], case["dim"], case["kv_heads"]
    G = case["q_heads"] // H
    out = torch.zeros((sum(q_len), case["q_heads"], D), dtype=torch.float64, device="cuda")
    lse = torch.zeros((sum(q_len), case["q_heads"]), dtype=torch.float64, device="cuda")
    n = 0
    for b, (Q, h0) in enumerate(zip(q_len, hist)):
        T = Q + h0
        pages = s["table"][b, : _ceil(T, P)].long()
        spans = torch.tensor([_seen(case, Q, h0, b, i) for i in range(Q)], device="cuda")
        j = torch.arange(T, device="cuda")
        hidden = (j < spans[:, :1]) | (j >= spans[:, 1:])
        dist = (torch.arange(Q, device="cuda")[:, None] + h0 - j).abs().double()
        for hk in range(H):
            k = s["key"][pages, hk].reshape(-1, D)[:T].double()
            v = s["value"][pages, hk].reshape(-1, D)[:T].double()
            for hq in range(hk * G, hk * G + G):
                x = s["query"][n:n + Q, hq].double() @ k.T / math.sqrt(D)
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                if s["slopes"] is not None:
                    x = x - s["slopes"][hq].double() * dist
                x = x.masked_fill(hidden, -math.inf)
                lse[n:n + Q, hq] = torch.logsumexp(x, -1)
                out[n:n + Q, hq] = torch.softmax(x, -1) @ v
        n += Q
    return {"out": out, "lse": lse}
