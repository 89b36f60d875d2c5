"""Paged serving operators on the GPU against plain 64-bit restatements: page_plan, paged_append, paged_attend, and a
run of them as a server makes it."""
import math
import random

import pytest
import torch

from kv_cache_b200 import _native, ops
from kv_cache_b200.cache import RequestPagedKV

from . import paged_util as ref

pytestmark = pytest.mark.gpu


def device_status(dev):
    import ctypes
    v = ctypes.c_int(0)
    assert _native.lib().kvb_device_status(dev.index or 0, ctypes.byref(v)) == 0
    return v.value


# ---- page_plan -----------------------------------------------------------------------------------------------------

def plan_inputs(B, P, q_hi, len_hi, seed, done_share=0.2, spare_pages=0):
    r = random.Random(seed)
    kv = [r.randint(0, len_hi) for _ in range(B)]
    q = [r.choice([0, 1, 1, r.randint(0, q_hi)]) for _ in range(B)]
    done = [r.random() < done_share for _ in range(B)]
    pages = [-(-n // P) for n in kv]
    W = max(-(-(n + x) // P) for n, x in zip(kv, q)) + 1
    num = sum(-(-(n + x) // P) for n, x in zip(kv, q)) + 1 + spare_pages
    ids = list(range(num))
    r.shuffle(ids)
    table = [[ids.pop() for _ in range(n)] + [-1] * (W - n) for n in pages]
    count = len(ids)
    return kv, q, table, ids + [-1] * (num - count), count, done


def run_plan(dev, kv, q, table, free, count, P, capacity, done, **kw):
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    t = dict(kv_len=i(kv), page_table=i(table), free_pages=i(free), free_count=i([count]))
    p = ops.page_plan(t["kv_len"], i(q), t["page_table"], t["free_pages"], t["free_count"], P, capacity,
                      finished=None if done is None else torch.tensor(done, device=dev), **kw)
    return p, t


def same_plan(p, t, want, table, free):
    for name in ("cu_q", "kv_len", "free_count", "slot", "position", "request", "status"):
        assert getattr(p, name).tolist() == want[name], name
    assert t["page_table"].tolist() == table
    assert t["free_pages"].tolist() == free


@pytest.mark.parametrize("B,P,q_hi,len_hi", [(1, 16, 1, 0), (1, 1, 5, 3), (3, 16, 40, 50), (33, 64, 300, 700), (256, 16, 1, 300),
                                             (1025, 8, 3, 20), (2500, 4, 9, 6), (5, 256, 6000, 100), (70, 32, 600, 3000), (8192, 4, 2, 9)])
@pytest.mark.parametrize("done", [True, False])
def test_plan(cuda_device, B, P, q_hi, len_hi, done):
    kv, q, table, free, count, fin = plan_inputs(B, P, q_hi, len_hi, seed=B * 31 + P)
    capacity = max(1, sum(q) + (B % 3))
    fin = fin if done else None
    want, wt, wf = ref.plan(kv, q, table, free, count, P, capacity, fin)
    assert want["status"] == [0, 0, 0, 0]
    p, t = run_plan(cuda_device, kv, q, table, free, count, P, capacity, fin)
    same_plan(p, t, want, wt, wf)
    assert t["kv_len"].tolist() == kv and t["free_count"].tolist() == [count]
    p, t = run_plan(cuda_device, kv, q, table, free, count, P, capacity, fin, in_place=True)
    assert p.kv_len is t["kv_len"] and p.free_count is t["free_count"]
    same_plan(p, t, want, wt, wf)


@pytest.mark.parametrize("what", ["pages", "tokens", "width", "count", "finished length"])
def test_plan_without_room_changes_nothing(cuda_device, what):
    P, capacity = 8, 64
    kv, q, done = [5, 16, 0, 30], [4, 9, 20, 1], [False, True, False, False]
    table = [[0, -1, -1, -1], [1, 2, -1, -1], [-1, -1, -1, -1], [3, 4, 5, 6]]
    free, count = [7, 8, 9, 10, 11, 12, -1, -1, -1, -1, -1, -1, -1], 6
    if what == "pages":
        count, q[2] = 2, 31
    elif what == "tokens":
        capacity = 33
    elif what == "width":
        q[3] = 3
    elif what == "count":
        count = 14
    else:
        kv[1] = 40
    want, wt, wf = ref.plan(kv, q, table, free, count, P, capacity, done)
    assert any(want["status"]) and wt == table and wf == free
    p, t = run_plan(cuda_device, kv, q, table, free, count, P, capacity, done, in_place=True)
    same_plan(p, t, want, wt, wf)


def test_plan_negative_lengths_count_as_zero_and_bad_pages_have_no_slot(cuda_device):
    kv, q = [-3, 4, 9], [2, -5, 3]
    table = [[-1, -1], [0, -1], [1, 99]]
    want, wt, wf = ref.plan(kv, q, table, [5, 6, 7, 8, 9], 5, 8, 8)
    p, t = run_plan(cuda_device, kv, q, table, [5, 6, 7, 8, 9], 5, 8, 8, None)
    same_plan(p, t, want, wt, wf)
    assert p.slot[:5].tolist()[2:] == [-1, -1, -1]


# ---- paged_append --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("N,Hkv,D,P,dtype", [(1, 1, 64, 16, torch.bfloat16), (5, 8, 128, 1, torch.float16), (777, 3, 128, 32, torch.bfloat16),
                                             (4001, 2, 64, 128, torch.float16), (9, 2, 8, 4, torch.bfloat16),
                                             (13, 2, 72, 16, torch.float16), (6, 1, 1024, 2, torch.bfloat16)])
def test_append(cuda_device, N, Hkv, D, P, dtype):
    g = torch.Generator().manual_seed(N)
    num = -(-N // P) + 3
    slot = torch.randperm(num * P, generator=g)[:N]
    slot[torch.rand(N, generator=g) < 0.2] = -1
    kv = torch.randn((N, 2 * Hkv + 1, D), generator=g).to(dtype)
    k, v = kv[:, 1:Hkv + 1], kv[:, Hkv + 1:]
    pools = [torch.randn((num, P, Hkv, D), generator=g).to(dtype).transpose(1, 2) for _ in range(2)]
    got = [p.to(cuda_device) for p in pools]
    dkv = kv.to(cuda_device)
    ops.paged_append(dkv[:, 1:Hkv + 1], dkv[:, Hkv + 1:], slot.to(cuda_device), *got)
    for pool, rows, have in zip(pools, (k, v), got):
        for n in range(N):
            if slot[n] >= 0:
                pool[slot[n] // P, :, slot[n] % P] = rows[n]
        assert torch.equal(have.cpu(), pool)


def test_append_skips_slots_outside_the_pool_and_reports_them(cuda_device):
    pool = torch.zeros((2, 1, 4, 64), dtype=torch.bfloat16, device=cuda_device)
    rows = torch.ones((4, 1, 64), dtype=torch.bfloat16, device=cuda_device)
    device_status(cuda_device)
    ops.paged_append(rows, rows, torch.tensor([0, -1, -1, 7], device=cuda_device), pool, pool.clone())
    assert device_status(cuda_device) == 0
    ops.paged_append(rows, rows, torch.tensor([0, 8, -2, 1 << 40], device=cuda_device), pool, pool.clone())
    assert device_status(cuda_device) == 7
    assert pool[0, 0, 0].eq(1).all() and pool[1, 0, 3].eq(1).all() and pool.sum() == 128


def test_append_of_nothing(cuda_device):
    pool = torch.zeros((2, 1, 4, 64), dtype=torch.bfloat16, device=cuda_device)
    rows = torch.ones((0, 1, 64), dtype=torch.bfloat16, device=cuda_device)
    ops.paged_append(rows, rows, torch.zeros(0, dtype=torch.int64, device=cuda_device), pool, pool)


# ---- paged_attend --------------------------------------------------------------------------------------------------

def check(dev, q_lens, kv_lens, Hq, Hkv, D, P, dtype, seed=0, scaling=None, softcap=0.0, slopes=None, window=0, prefix=None,
          single=False, max_q=0, spare=0, width=None):
    t, key, value = ref.paged_case(dev, q_lens, kv_lens, Hq, Hkv, D, P, dtype, seed, spare, width)
    if single:
        t["cu_q"] = None
    sl = None if slopes is None else torch.tensor(slopes, dtype=torch.float32)
    out = torch.full_like(t["query"], 7.0)
    got, lse = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"], cu_q=t["cu_q"],
                                max_q=max_q, scaling=scaling, softcap=softcap, slopes=None if sl is None else sl.to(dev),
                                window=window, prefix_len=None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=dev),
                                out=out, return_lse=True)
    assert got is out
    n = sum(q_lens)
    want, wlse, bound, lbound = ref.attend(t["query"][:n], key, value, q_lens, kv_lens, scaling or D ** -0.5, softcap,
                                           None if sl is None else sl.tolist(), window, prefix)
    assert device_status(dev) == 0
    have = got[:n].double().cpu()
    assert torch.isfinite(have).all()
    over = (have - want).abs() / bound.clamp(min=1e-30)
    empty = torch.isinf(wlse)
    assert have[empty].eq(0).all()
    assert (over[~empty].max() if (~empty).any() else 0) <= 1, float(over[~empty].max())
    hl = lse[:n].double().cpu()
    assert torch.equal(torch.isinf(hl), empty)
    assert ((hl - wlse).abs()[~empty] <= lbound[~empty]).all(), float((hl - wlse).abs()[~empty].max())
    assert got[n:].eq(7.0).all()
    return t, got, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 4), (8, 2), (10, 2), (7, 1), (24, 1), (40, 1)])
def test_single_tokens(cuda_device, dtype, D, Hq, Hkv):
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 300, 1000]
    check(cuda_device, [1] * len(kv), kv, Hq, Hkv, D, 16, dtype, seed=Hq + D, single=True, max_q=1)


@pytest.mark.parametrize("P", [1, 2, 8, 16, 64, 256, 1024])
def test_page_sizes(cuda_device, P):
    check(cuda_device, [1, 5, 40, 130, 3], [700, 130, 40, 333, 257], 8, 2, 128, P, torch.bfloat16, seed=P, spare=3)


@pytest.mark.parametrize("max_q", [0, 1, 2, 1000])
@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(8, 2, 128, torch.bfloat16), (6, 6, 64, torch.float16), (15, 3, 128, torch.float16),
                                            (36, 1, 64, torch.bfloat16), (129, 1, 64, torch.bfloat16)])
def test_chunks(cuda_device, max_q, Hq, Hkv, D, dtype):
    """Prompts from their first token on, chunks behind cached tokens, single tokens and idle requests in one call."""
    q = [1, 0, 129, 64, 2, 0, 33, 17, 200, 1]
    kv = [77, 40, 129, 500, 2, 0, 1033, 17, 311, 128]
    check(cuda_device, q, kv, Hq, Hkv, D, 32, dtype, seed=Hq, max_q=max_q, spare=5)


MODS = {"cap": dict(softcap=5.0), "slopes": dict(slopes=True), "window": dict(window=37), "one": dict(window=1),
        "prefix": dict(prefix=[0, 50, 1000, 5, 90, 3]), "all": dict(softcap=20.0, slopes=True, window=100, prefix=[9, 0, 300, 41, 700, 2]),
        "scaling": dict(scaling=0.3)}


@pytest.mark.parametrize("mod", list(MODS))
@pytest.mark.parametrize("q_lens,max_q", [([1, 1, 1, 1, 1, 1], 1), ([3, 1, 4, 2, 1, 0], 4), ([1, 70, 200, 5, 333, 16], 333)])
@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(4, 1, 128, torch.bfloat16), (10, 2, 64, torch.float16)])
def test_score_forms(cuda_device, mod, q_lens, max_q, Hq, Hkv, D, dtype):
    kw = dict(MODS[mod])
    if kw.get("slopes"):
        kw["slopes"] = [2.0 ** (-0.7 * h) - 0.01 for h in range(Hq)]
    kv = [max(a, b) for a, b in zip(q_lens, [250, 131, 300, 64, 700, 1])]
    check(cuda_device, q_lens, kv, Hq, Hkv, D, 16, dtype, seed=5, max_q=max_q, **kw)


@pytest.mark.parametrize("max_q", [1, 300])
def test_rows_that_see_nothing(cuda_device, max_q):
    """More new tokens than keys: the first ones stand before position 0. Requests without a key at all."""
    q, kv = [5, 1, 200, 3, 1], [2, 0, 150, 0, 9]
    check(cuda_device, q, kv, 8, 2, 128, 16, torch.bfloat16, max_q=max_q)


@pytest.mark.parametrize("q,kv,max_q", [([1], [70001], 1), ([1, 1, 1], [3, 33333, 8], 1), ([4], [20000], 4), ([40, 1], [9000, 30001], 40)])
def test_long_keys_are_split_over_the_device(cuda_device, q, kv, max_q):
    check(cuda_device, q, kv, 4, 2, 128, 64, torch.bfloat16, seed=9, max_q=max_q, width=1200)


def test_far_window_reads_no_freed_page(cuda_device):
    """Pages below every window may be gone: their table entries are never looked at."""
    kv, q, W = [500, 2000], [1, 30], 64
    t, key, value = ref.paged_case(cuda_device, q, kv, 4, 2, 128, 16, torch.bfloat16, seed=3)
    for max_q in (1, 30):
        want = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"], cu_q=t["cu_q"], window=W, max_q=max_q)
        table = t["page_table"].clone()
        for b in range(2):
            table[b, :(kv[b] - q[b] - W + 1) // 16] = 1 << 30
        got = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], table, t["kv_len"], cu_q=t["cu_q"], window=W, max_q=max_q)
        assert torch.equal(want, got)
    assert device_status(cuda_device) == 0


@pytest.mark.parametrize("max_q", [1, 50])
def test_bad_device_data_is_reported_and_harms_nothing(cuda_device, max_q):
    q, kv = [1, 50], [100, 90]
    t, key, value = ref.paged_case(cuda_device, q, kv, 4, 2, 128, 16, torch.bfloat16, seed=4)
    kw = dict(cu_q=t["cu_q"], max_q=max_q)
    good = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"], **kw)
    assert device_status(cuda_device) == 0
    table = t["page_table"].clone()
    table[1, 2], table[1, 3] = 1 << 30, -1
    got = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], table, t["kv_len"], **kw)
    assert device_status(cuda_device) == 7
    assert torch.equal(got[:1], good[:1]) and torch.isfinite(got).all()
    # offsets that run backwards or beyond the query are cut to it
    cu = torch.tensor([40, 3, 1 << 30], dtype=torch.int32, device=cuda_device)
    out = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"], cu_q=cu, max_q=max_q,
                           out=torch.full_like(t["query"], 3.0))
    assert out[:3].eq(3.0).all() and torch.isfinite(out).all()
    device_status(cuda_device)


@pytest.mark.parametrize("max_q", [1, 40])
def test_requests_that_share_pages(cuda_device, max_q):
    """A common prefix stored once: two table rows name the same pages."""
    q, kv = [40, 3], [200, 163]
    t, key, value = ref.paged_case(cuda_device, q, kv, 4, 2, 64, 32, torch.float16, seed=6)
    t["page_table"][1, :5] = t["page_table"][0, :5]
    for x in (key, value):
        x[1] = torch.cat((x[0][:, :160], x[1][:, 160:]), 1)
    got = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"], cu_q=t["cu_q"], max_q=max_q)
    want, _, bound, _ = ref.attend(t["query"], key, value, q, kv, 64 ** -0.5)
    assert ((got.double().cpu() - want).abs() <= bound).all()


def test_lengths_beyond_the_table_are_cut_and_reported(cuda_device):
    t, key, value = ref.paged_case(cuda_device, [1, 1], [64, 40], 4, 2, 64, 32, torch.float16, seed=7)
    want = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"])
    assert device_status(cuda_device) == 0
    t["kv_len"][0] = 65
    got = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"])
    assert device_status(cuda_device) == 7 and torch.equal(got, want)


def test_strided_operands(cuda_device):
    """Queries that are columns of a fused projection, pools with tokens outside heads, a table cut from a wider one."""
    q, kv = [1, 60, 7], [90, 200, 7]
    t, key, value = ref.paged_case(cuda_device, q, kv, 8, 2, 128, 16, torch.bfloat16, seed=8)
    want = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"], cu_q=t["cu_q"])
    N = t["query"].shape[0]
    fused = torch.zeros((N, 12, 128), dtype=torch.bfloat16, device=cuda_device)
    fused[:, 2:10] = t["query"]
    kp = t["key_pool"].transpose(1, 2).contiguous().transpose(1, 2)
    vp = torch.zeros((*t["value_pool"].shape[:3], 136), dtype=torch.bfloat16, device=cuda_device)
    vp[..., :128] = t["value_pool"]
    wide = torch.full((3, 40), -5, dtype=torch.int32, device=cuda_device)
    wide[:, 4:4 + t["page_table"].shape[1]] = t["page_table"]
    got = ops.paged_attend(fused[:, 2:10], kp, vp[..., :128], wide[:, 4:4 + t["page_table"].shape[1]], t["kv_len"], cu_q=t["cu_q"])
    assert torch.equal(want, got)


@pytest.mark.parametrize("max_q", [1, 64])
def test_repeatable_on_another_stream_and_in_graphs(cuda_device, max_q):
    """The same bits on a side stream and from two captured graphs replayed one after the other; lengths are read at
    replay."""
    q, kv = [1, 3, 64], [3000, 40, 1500]
    t, key, value = ref.paged_case(cuda_device, q, kv, 8, 2, 128, 16, torch.bfloat16, seed=2)
    call = lambda out=None: ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"],  # noqa: E731
                                             cu_q=t["cu_q"], max_q=max_q, out=out)
    want = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call()
        graphs, outs = [], [torch.zeros_like(want) for _ in range(2)]
        for o in outs:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                call(o)
            graphs.append(graph)
        for graph in graphs:
            graph.replay()
    s.synchronize()
    assert torch.equal(want, got) and all(torch.equal(want, o) for o in outs)
    t["kv_len"] -= torch.tensor([1000, 0, 700], dtype=torch.int32, device=cuda_device)
    want = call()
    with torch.cuda.stream(s):
        s.wait_stream(torch.cuda.default_stream())
        graphs[1].replay()
        graphs[0].replay()
    s.synchronize()
    assert all(torch.equal(want, o) for o in outs)


@pytest.mark.parametrize("max_q", [1, 64])
def test_two_streams_at_once(cuda_device, max_q):
    """Calls in flight on two streams do not disturb each other (each has its own workspace)."""
    cases = []
    for seed, (q, kv) in enumerate([([1, 3, 64], [3000, 40, 1500]), ([64, 1, 1], [900, 2100, 33])]):
        t, _, _ = ref.paged_case(cuda_device, q, kv, 8, 2, 128, 16, torch.bfloat16, seed=seed)
        call = lambda t=t: ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"],  # noqa: E731
                                            cu_q=t["cu_q"], max_q=max_q)
        cases.append((call, call(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (call, _, stream) in enumerate(cases):
            with torch.cuda.stream(stream):
                outs[i].append(call())
    torch.cuda.synchronize()
    for (_, want, _), got in zip(cases, outs):
        assert all(torch.equal(want, o) for o in got)


def test_query_rows_that_are_not_aligned(cuda_device):
    t, _, _ = ref.paged_case(cuda_device, [1, 20], [90, 20], 8, 2, 128, 16, torch.float16, seed=1)
    want = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"], cu_q=t["cu_q"])
    wide = torch.zeros((*t["query"].shape[:2], 131), dtype=torch.float16, device=cuda_device)
    wide[..., 1:129] = t["query"]
    got = ops.paged_attend(wide[..., 1:129], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"], cu_q=t["cu_q"])
    assert torch.equal(want, got)


def test_many_requests(cuda_device):
    r = random.Random(1)
    B = 1500
    kv = [r.randint(0, 40) for _ in range(B)]
    q = [min(n, r.choice([0, 1, 1, 3])) for n in kv]
    check(cuda_device, q, kv, 2, 1, 64, 8, torch.float16, max_q=3)


def test_no_query_rows(cuda_device):
    t, _, _ = ref.paged_case(cuda_device, [0, 0], [5, 9], 4, 2, 64, 8, torch.float16)
    out, lse = ops.paged_attend(t["query"], t["key_pool"], t["value_pool"], t["page_table"], t["kv_len"], cu_q=t["cu_q"], return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_offsets_beyond_32_bits(cuda_device):
    """A pool of more than 2^32 bytes and 2^31 elements: pages at its end."""
    num, P, H, D = 2200, 1024, 8, 128                     # 2.3e9 elements, 4.6 GB
    pool = torch.zeros((num, H, P, D), dtype=torch.bfloat16, device=cuda_device)
    table = torch.tensor([[num - 1], [1], [num - 2]], dtype=torch.int32, device=cuda_device)
    kv = torch.tensor([1024, 7, 300], dtype=torch.int32, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    for page in (num - 1, 1, num - 2):
        pool[page] = torch.randn((H, P, D), generator=g, device=cuda_device)
    query = torch.randn((41, 8, D), generator=g, device=cuda_device).to(torch.bfloat16)
    cu = torch.tensor([0, 1, 2, 41], dtype=torch.int32, device=cuda_device)
    small = pool[[num - 1, 1, num - 2]].clone()
    order = torch.tensor([[0], [1], [2]], dtype=torch.int32, device=cuda_device)
    for max_q in (1, 39):
        got = ops.paged_attend(query, pool, pool, table, kv, cu_q=cu, max_q=max_q)
        assert torch.equal(got, ops.paged_attend(query, small, small, order, kv, cu_q=cu, max_q=max_q))
    rows = torch.randn((2, H, D), generator=g, device=cuda_device).to(torch.bfloat16)
    ops.paged_append(rows, rows, torch.tensor([num * P - 1, (num - 1) * P], device=cuda_device), pool, pool)
    assert torch.equal(pool[num - 1, :, P - 1], rows[0]) and torch.equal(pool[num - 1, :, 0], rows[1])


# ---- a run of them together ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("captured,max_q", [(False, 0), (True, 0), (True, 1)])
def test_serving_run(cuda_device, captured, max_q):
    """Requests come, grow by chunks and single tokens, end, and their rows and pages are used again: every step's
    output equals the 64-bit attention over what each request was given. Two layers share the plan."""
    Hq, Hkv, D, P, B, layers, capacity = 6, 2, 64, 8, 5, 2, 80
    dtype = torch.bfloat16
    kv = RequestPagedKV(layers, B, Hkv, D, P, 60, 24, cuda_device, dtype)
    g = torch.Generator().manual_seed(0)
    held = [[(torch.zeros((Hkv, 0, D), dtype=dtype),) * 2 for _ in range(B)] for _ in range(layers)]
    q_len = torch.zeros(B, dtype=torch.int32, device=cuda_device)
    done = torch.zeros(B, dtype=torch.bool, device=cuda_device)
    ins = torch.zeros((layers, capacity, Hq + 2 * Hkv, D), dtype=dtype, device=cuda_device)
    outs = torch.zeros((layers, capacity, Hq, D), dtype=dtype, device=cuda_device)

    def body():
        kv.step(q_len, capacity, finished=done, max_q=max_q)
        for layer in range(layers):
            x = ins[layer]
            kv.append(layer, x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:])
            kv.attend(layer, x[:, :Hq], out=outs[layer])

    graph = None
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            body()
    steps = [([50, 0, 7, 0, 0], []), ([1, 20, 1, 0, 33], []), ([1, 1, 1, 9, 1], [0]), ([30, 1, 0, 1, 1], [1, 4]), ([1, 1, 1, 1, 1], []),
             ([0, 70, 1, 1, 1], [1]), ([1, 1, 60, 1, 1], [2])]
    for q, fin in steps:
        q_len.copy_(torch.tensor(q, dtype=torch.int32))
        done.zero_()
        if fin:
            done[fin] = True
        x = torch.randn((layers, capacity, Hq + 2 * Hkv, D), generator=g).to(dtype)
        ins.copy_(x)
        outs.fill_(9.0)
        graph.replay() if captured else body()
        assert kv.plan.status.tolist() == [0, 0, 0, 0]
        n = sum(q)
        for layer in range(layers):
            at = 0
            for b in range(B):
                k, v = held[layer][b] if b not in fin else (torch.zeros((Hkv, 0, D), dtype=dtype),) * 2
                new = x[layer, at:at + q[b]]
                held[layer][b] = (torch.cat((k, new[:, Hq:Hq + Hkv].transpose(0, 1)), 1), torch.cat((v, new[:, Hq + Hkv:].transpose(0, 1)), 1))
                at += q[b]
            lens = [h[0].shape[1] for h in held[layer]]
            assert kv.kv_len.tolist() == lens
            want, _, bound, _ = ref.attend(x[layer, :n, :Hq], [h[0] for h in held[layer]], [h[1] for h in held[layer]], q, lens, D ** -0.5)
            assert ((outs[layer, :n].double().cpu() - want).abs() <= bound).all()
            assert outs[layer, n:].eq(9.0).all()
        used = sum(-(-m // P) for m in lens)
        assert kv.free_count.item() == 60 - used
    # a step that does not fit leaves everything as it was
    before = kv.kv_len.clone()
    q_len.fill_(79)
    done.zero_()
    outs.fill_(9.0)
    graph.replay() if captured else body()
    assert kv.plan.status[1].item() == 5 * 79 - capacity
    assert torch.equal(kv.kv_len, before) and outs.eq(9.0).all()
    assert device_status(cuda_device) == 0
