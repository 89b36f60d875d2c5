"""What the paged serving operators refuse before anything is launched, and their plain restatement on small cases."""
import ctypes

import pytest
import torch

from kv_cache_b200 import _native, ops

from . import paged_util as ref

i32 = dict(dtype=torch.int32)


def plan_args(**kw):
    a = dict(kv_len=torch.zeros(3, **i32), q_len=torch.ones(3, **i32), page_table=torch.zeros((3, 4), **i32),
             free_pages=torch.arange(10, **i32), free_count=torch.tensor([10], **i32), page_tokens=8, capacity=5)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(kv_len=torch.zeros(3)), dict(kv_len=torch.zeros((3, 1), **i32)), dict(kv_len=torch.zeros(0, **i32), q_len=torch.zeros(0, **i32)),
    dict(q_len=torch.zeros(2, **i32)), dict(q_len=torch.zeros(6, **i32)[::2]), dict(page_table=torch.zeros((2, 4), **i32)),
    dict(page_table=torch.zeros((3, 4), dtype=torch.int64)), dict(page_table=torch.zeros((4, 3), **i32).T), dict(page_table=torch.zeros((1, 4), **i32).expand(3, 4)),
    dict(free_count=torch.zeros(2, **i32)), dict(free_pages=torch.zeros(0, **i32)), dict(page_tokens=12), dict(page_tokens=0), dict(capacity=0),
    dict(finished=torch.zeros(3)), dict(finished=torch.zeros(2, dtype=torch.bool)),
    dict(out=ops.PagePlan(*[torch.zeros(1, **i32)] * 7)), dict()])
def test_plan_refusals(kw):
    with pytest.raises(RuntimeError):                    # the last case: CPU tensors
        ops.page_plan(**plan_args(**kw))


def append_args(**kw):
    bf = torch.bfloat16
    a = dict(key_rows=torch.zeros((5, 2, 64), dtype=bf), value_rows=torch.zeros((5, 2, 64), dtype=bf), slot=torch.zeros(5, dtype=torch.int64),
             key_pool=torch.zeros((4, 2, 8, 64), dtype=bf), value_pool=torch.zeros((4, 2, 8, 64), dtype=bf))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(key_rows=torch.zeros((5, 2, 64))), dict(value_rows=torch.zeros((4, 2, 64), dtype=torch.bfloat16)), dict(slot=torch.zeros(5, **i32)),
    dict(slot=torch.zeros(4, dtype=torch.int64)), dict(key_pool=torch.zeros((4, 2, 8, 32), dtype=torch.bfloat16)),
    dict(key_pool=torch.zeros((4, 2, 6, 64), dtype=torch.bfloat16), value_pool=torch.zeros((4, 2, 6, 64), dtype=torch.bfloat16)),
    dict(key_pool=torch.zeros((4, 2, 64, 8), dtype=torch.bfloat16).transpose(2, 3)), dict()])
def test_append_refusals(kw):
    with pytest.raises(RuntimeError):
        ops.paged_append(**append_args(**kw))


def attend_args(**kw):
    bf = torch.bfloat16
    a = dict(query=torch.zeros((3, 4, 64), dtype=bf), key_pool=torch.zeros((4, 2, 8, 64), dtype=bf), value_pool=torch.zeros((4, 2, 8, 64), dtype=bf),
             page_table=torch.zeros((3, 2), **i32), kv_len=torch.ones(3, **i32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(query=torch.zeros((3, 4, 64))), dict(query=torch.zeros((3, 4, 64), dtype=torch.float16)), dict(query=torch.zeros((3, 3, 64), dtype=torch.bfloat16)),
    dict(query=torch.zeros((2, 4, 64), dtype=torch.bfloat16)), dict(query=torch.zeros((3, 4, 1, 64), dtype=torch.bfloat16)), dict(kv_len=torch.ones(3)),
    dict(cu_q=torch.zeros(3, **i32)), dict(slopes=torch.zeros(2)), dict(slopes=torch.zeros(4, dtype=torch.float64)), dict(prefix_len=torch.zeros(4, **i32)),
    dict(scaling=0.0), dict(scaling=-1.0), dict(scaling=float("nan")), dict(scaling=float("inf")), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=1e-39, scaling=1.0), dict(window=-1), dict(max_q=-1),
    dict(out=torch.zeros((3, 4, 64))), dict(out=torch.zeros((2, 4, 64), dtype=torch.bfloat16)),
    dict(query=torch.zeros((3, 4, 32), dtype=torch.bfloat16), key_pool=torch.zeros((4, 2, 8, 32), dtype=torch.bfloat16), value_pool=torch.zeros((4, 2, 8, 32), dtype=torch.bfloat16)),
    dict()])
def test_attend_refusals(kw):
    with pytest.raises(RuntimeError):
        ops.paged_attend(**attend_args(**kw))


def test_c_refusals_without_a_device():
    lib = _native.lib()
    x = ctypes.create_string_buffer(4096)
    a = (ctypes.addressof(x) + 255) // 256 * 256

    def attend(**kw):
        p = _native.PagedAttendParams()
        base = dict(query=a, key_pool=a, value_pool=a, page_table=a, kv_len=a, out=a, workspace=a, page_table_stride=2, N=3, B=3, Hq=4, Hkv=2,
                    D=64, W=2, num_pages=4, page_tokens=8, scaling=1.0, q_st=256, q_sh=64, k_sp=1024, k_sh=512, k_st=64, v_sp=1024, v_sh=512, v_st=64)
        base.update(kw)
        for k, v in base.items():
            setattr(p, k, v)
        return lib.kvb_paged_attend(ctypes.byref(p), 999, None)

    assert attend() == 3                                  # every other check passed: there is no device 999
    assert lib.kvb_paged_attend(None, 0, None) == 7
    for bad in (dict(query=None), dict(workspace=None), dict(elem_type=2), dict(scaling=0.0), dict(scaling=float("nan")), dict(softcap=-1.0),
                dict(softcap=1e-39), dict(window=-1), dict(max_q=-1)):
        assert attend(**bad) == 7, bad
    for bad in (dict(D=96), dict(Hq=5), dict(B=0), dict(B=8193), dict(N=2), dict(page_tokens=12), dict(W=0), dict(page_table_stride=1),
                dict(N=-1), dict(num_pages=0), dict(W=1 << 28)):
        assert attend(**bad) == 1, bad
    for bad in (dict(query=a + 2), dict(key_pool=a + 8), dict(workspace=a + 16), dict(q_st=12), dict(v_st=-64), dict(k_sp=4)):
        assert attend(**bad) == 2, bad
    assert lib.kvb_paged_attend_workspace_bytes(3, 3, 4, 2, 2, 8, 96, 0) == 0
    assert lib.kvb_paged_attend_workspace_bytes(3, 3, 4, 2, 2, 8, 64, 0) > 0

    def plan(B=3, W=2, num=4, P=8, cap=5, stride=2, table=a):
        return lib.kvb_page_plan(a, a, None, B, table, stride, W, a, num, a, P, cap, a, a, a, a, a, a, a, 999, None)

    assert plan() == 3 and plan(table=None) == 7
    assert [plan(B=0), plan(B=8193), plan(W=3), plan(num=0), plan(P=3), plan(cap=0), plan(W=1 << 20, stride=1 << 20, P=2048)] == [1] * 7

    def append(D=64, N=5, st=128, k=a, P=8):
        return lib.kvb_paged_append(k, st, 64, a, 128, 64, a, N, 2, D, a, 1024, 512, 64, a, 1024, 512, 64, 4, P, 999, None)

    assert append() == 3 and append(k=None) == 7 and append(st=100) == 2 and append(k=a + 4) == 2
    assert [append(D=12), append(D=0), append(N=-1), append(P=5)] == [1] * 4


def test_the_plain_plan():
    """By hand: request 1 ends and gives back pages 3 and 4, request 0 grows into a page, request 1 starts over."""
    got, table, free = ref.plan([7, 12, 0], [2, 9, 0], [[9, 0], [3, 4], [0, 0]], [5, 6, 0, 0, 0, 0, 0, 0, 0, 0], 2, 8, 12, [False, True, False])
    assert got["cu_q"] == [0, 2, 11, 11] and got["kv_len"] == [9, 9, 0] and got["free_count"] == [1]
    assert table[0] == [9, 4] and table[1] == [3, 6] and free[:4] == [5, 6, 3, 4]
    assert got["slot"] == [79, 32] + list(range(24, 32)) + [48, -1]
    assert got["position"] == [7, 8, 0, 1, 2, 3, 4, 5, 6, 7, 8, -1] and got["status"] == [0, 0, 0, 0]


def test_visible_ranges():
    assert ref.visible(10, 3, 0) == (0, 8) and ref.visible(10, 3, 2) == (0, 10)
    assert ref.visible(10, 3, 1, window=2) == (7, 9) and ref.visible(10, 3, 0, prefix=9) == (0, 9)
    assert ref.visible(2, 5, 0) == (0, 0) and ref.visible(2, 5, 0, prefix=1) == (0, 1)
