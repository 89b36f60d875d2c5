"""Plain 64-bit restatements of the paged serving operators, for tests."""
import math
import random

import torch


def plan(kv_len, q_len, table, free, count, P, capacity, finished=None):
    """page_plan on Python lists; returns (dict of results, table, free)."""
    B, W, num = len(kv_len), len(table[0]), len(free)
    table, free = [list(r) for r in table], list(free)
    done = finished or [False] * B
    q = [max(x, 0) for x in q_len]
    gone = [(max(n, 0) + P - 1) // P if d else 0 for n, d in zip(kv_len, done)]
    old = [0 if d else max(n, 0) for n, d in zip(kv_len, done)]
    take = [(o + x + P - 1) // P - (o + P - 1) // P for o, x in zip(old, q)]
    status = [max(0, sum(take) - count - sum(gone)), max(0, sum(q) - capacity),
              sum((o + x + P - 1) // P > W for o, x in zip(old, q)),
              int(not 0 <= count <= num or count + sum(gone) > num or any(g > W for g in gone))]
    if any(status):
        return dict(cu_q=[0] * (B + 1), kv_len=list(kv_len), free_count=[count], slot=[-1] * capacity,
                    position=[-1] * capacity, request=[-1] * capacity, status=status), table, free
    for b in range(B):
        for j in range(gone[b]):
            free[count] = table[b][j]
            count += 1
    cu, slot, position, request = [0], [], [], []
    for b in range(B):
        for i in range(q[b]):
            pos = old[b] + i
            if pos % P == 0:
                count -= 1
                table[b][pos // P] = free[count]
            page = table[b][pos // P]
            slot.append(page * P + pos % P if 0 <= page < num else -1)
            position.append(pos)
            request.append(b)
        cu.append(cu[-1] + q[b])
    pad = [-1] * (capacity - cu[-1])
    return dict(cu_q=cu, kv_len=[o + x for o, x in zip(old, q)], free_count=[count], slot=slot + pad,
                position=position + pad, request=request + pad, status=status), table, free


def visible(kv, q, i, window=0, prefix=0):
    """Half-open key range of token i of a request that holds kv tokens, the last q of them new."""
    p = kv - q + i
    lo = max(0, p - window + 1) if window else 0
    return lo, max(lo, min(kv, max(p + 1, min(prefix, kv))))


def attend(query, key, value, q_lens, kv_lens, scaling, softcap=0.0, slopes=None, window=0, prefix=None):
    """query [N,Hq,D]; key/value: per request [Hkv,kv,D]. Returns (out, lse, bound) in 64 bits on the CPU; ``bound`` is
    what a kernel with fp32 arithmetic and weights rounded to the input type may be off by, element by element:
    one rounding of each weight and one of the result (half a step, eps / 2, each), fp32 error of the scores (the
    products of D terms, the exponent's argument) and of the sums over the keys."""
    N, Hq, D = query.shape
    u = torch.finfo(query.dtype).eps / 2
    q64 = query.double().cpu()
    out = torch.zeros((N, Hq, D), dtype=torch.float64)
    lse = torch.full((N, Hq), -math.inf, dtype=torch.float64)
    bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    n = 0
    for b, (Q, kv) in enumerate(zip(q_lens, kv_lens)):
        k, v = key[b].double().cpu(), value[b].double().cpu()
        G = Hq // k.shape[0]
        spans = torch.tensor([visible(kv, Q, i, window, prefix[b] if prefix else 0) for i in range(Q)]).reshape(Q, 2)
        j = torch.arange(kv)
        see = (j >= spans[:, :1]) & (j < spans[:, 1:])
        dist = (torch.arange(Q)[:, None] + kv - Q - j).abs().double()
        for h in range(Hq):
            qq = q64[n:n + Q, h]
            x = qq @ k[h // G].T * scaling
            ex = qq.abs() @ k[h // G].abs().T * scaling * (D + 16) * 2.0 ** -23
            if softcap:
                x = softcap * torch.tanh(x / softcap)
                ex = ex + softcap * 2.0 ** -20
            if slopes is not None:
                x = x - float(slopes[h]) * dist
                ex = ex + abs(float(slopes[h])) * dist * 2.0 ** -22
            ex = ex + x.abs() * 2.0 ** -21 + 2.0 ** -21
            x = x.masked_fill(~see, -math.inf)
            some = see.any(-1)
            if not bool(some.any()):
                continue
            w = torch.softmax(x[some], -1)
            e = ex.masked_fill(~see, 0.0)[some].amax(-1, keepdim=True)
            rows = torch.arange(n, n + Q)[some]
            o, a = w @ v[h // G], w @ v[h // G].abs()
            out[rows, h] = o
            lse[rows, h] = torch.logsumexp(x[some], -1)
            tiny = kv * 2.0 ** -31 * float(v.abs().max()) if kv else 0.0
            bound[rows, h] = u * o.abs() + (u + 2.5 * e + (kv + 64) * 2.0 ** -22) * a * 1.01 + tiny + (2.0 ** -24 if query.dtype == torch.float16 else 0.0)
            lse_bound[rows, h] = (e[:, 0] + (kv + 64) * 2.0 ** -23) * 1.01 + lse[rows, h].abs() * 2.0 ** -22
        n += Q
    return out, lse, bound, lse_bound


def paged_case(device, q_lens, kv_lens, Hq, Hkv, D, P, dtype, seed=0, spare=0, width=None):
    """Pools with scattered pages (NaN wherever no request has a token), table, lengths, packed queries."""
    g = torch.Generator().manual_seed(seed)
    r = random.Random(seed)
    B = len(q_lens)
    need = [-(-n // P) for n in kv_lens]
    num = sum(need) + 2
    ids = list(range(num))
    r.shuffle(ids)
    W = width or max(1, max(need))
    table = torch.full((B, W), -7, dtype=torch.int32)
    key_pool = torch.full((num, Hkv, P, D), math.nan, dtype=dtype)
    value_pool = torch.full((num, Hkv, P, D), math.nan, dtype=dtype)
    key, value = [], []
    for b in range(B):
        k = (torch.randn((Hkv, kv_lens[b], D), generator=g) * 1.3).to(dtype)
        v = torch.randn((Hkv, kv_lens[b], D), generator=g).to(dtype)
        key.append(k)
        value.append(v)
        for i in range(need[b]):
            page = ids.pop()
            table[b, i] = page
            n = min(P, kv_lens[b] - i * P)
            key_pool[page, :, :n] = k[:, i * P:i * P + n]
            value_pool[page, :, :n] = v[:, i * P:i * P + n]
    query = torch.randn((sum(q_lens) + spare, Hq, D), generator=g).to(dtype)
    cu = [0]
    for q in q_lens:
        cu.append(cu[-1] + q)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    return dict(query=query.to(device), key_pool=key_pool.to(device), value_pool=value_pool.to(device),
                page_table=table.to(device), kv_len=ints(kv_lens), cu_q=ints(cu)), key, value
