"""The four operators of the retrieval-sparse decode path on torch CUDA tensors.

Layouts follow the reference (paths inside littlexi001/kv_cache,
EVAL = ymluo/projects/qwen3_top2_head_limit3_ppl/src/evaluate_qwen3_top2_head_limit3_ppl.py,
QCK = .../src/qabs_cuda_kernels.py):

* ``key`` / ``value``  bf16 ``[B, Hkv, T, D]`` as the HF cache holds them (NOT repeated to query
  heads, unlike EVAL:6248-6251); views with arbitrary batch/head/token strides are accepted.
* ``query``            bf16 ``[B, Hq, D]`` (``[B, Hq, 1, D]`` is accepted and squeezed, EVAL:4424).
* scores               ``[B, H, T]`` (QCK:654-665), indices int64 ``[B, H, S]`` + bool valid
  (QCK:694-705), attention output ``[B, 1, Hq, D]`` (EVAL:4502).

Every function launches on the current torch stream of the tensors' device and calls the C-ABI
library; there is no eager/torch fallback.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional

import torch

from . import _native
from ._native import DecodeStepParams, PagedAttendParams, check

HIST_BINS = 4096


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _raw_stream(index: int) -> int:
    """The current stream of device ``index`` as an address, without making a Stream object (4 us of a 20 us call)."""
    return torch._C._cuda_getCurrentRawStream(index)


def _dev(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise RuntimeError("kv_cache_b200 operators need CUDA tensors; there is no CPU path")
    return t.device.index if t.device.index is not None else torch.cuda.current_device()


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _rows_contiguous(t: torch.Tensor) -> torch.Tensor:
    """[.., T, D] with contiguous D and 16-byte aligned strides, copying only when needed (QCK:595-599)."""
    ok = t.stride(-1) == 1 and all(s % 8 == 0 for s in t.stride()[:-1]) and t.data_ptr() % 16 == 0
    return t if ok else t.contiguous()


def _query3(query: torch.Tensor) -> torch.Tensor:
    if query.dim() == 4:
        if query.shape[2] != 1:
            raise RuntimeError("decode operators take one query token per sequence")
        query = query[:, :, 0, :]
    if query.dim() != 3:
        raise RuntimeError("query must have shape [batch, heads, dim]")
    return _rows_contiguous(query)


# ------------------------------------------------------------------------------------------
# channel choice (host-side policy; an input to every kernel, like dim_indices in QCK:659-665)
# ------------------------------------------------------------------------------------------

def choose_channels(key: torch.Tensor, num_channels: int) -> torch.Tensor:
    """Per KV head, the ``num_channels`` head-dim channels with the largest mean |K| over (B, T);
    ties go to the lower channel; returned ascending as int32 ``[Hkv, C]``."""
    T = key.shape[2]
    total = torch.zeros((key.shape[1], key.shape[3]), dtype=torch.float64, device=key.device)
    for t0 in range(0, T, 16384):                                       # bounded fp32 temporaries
        total += key[:, :, t0:t0 + 16384].float().abs().sum(dim=(0, 2), dtype=torch.float64)
    mean_abs = total / max(1, key.shape[0] * T)                         # [Hkv, D]
    order = torch.sort(mean_abs, dim=-1, descending=True, stable=True).indices[:, :num_channels]
    return torch.sort(order, dim=-1).values.to(torch.int32).contiguous()


# ------------------------------------------------------------------------------------------
# stage 1: quantize / pack
# ------------------------------------------------------------------------------------------

def alloc_side_cache(batch: int, kv_heads: int, capacity: int, num_channels: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    """int4 side cache for ``capacity`` tokens: packed uint8 ``[B,Hkv,cap,C/2]`` and fp32 scale
    ``[B,Hkv,cap]``; capacity is rounded up to 256 tokens so every row start is 16-byte aligned."""
    cap = (int(capacity) + 255) // 256 * 256
    packed = torch.empty((batch, kv_heads, cap, num_channels // 2), dtype=torch.uint8, device=device)
    scale = torch.empty((batch, kv_heads, cap), dtype=torch.float32, device=device)
    return packed, scale


def _check_side_cache(packed: torch.Tensor, scale: torch.Tensor, C_: int) -> None:
    if packed.dtype != torch.uint8 or scale.dtype != torch.float32:
        raise RuntimeError("packed must be uint8 and scale float32")
    if packed.dim() != 4 or scale.dim() != 3 or packed.shape[-1] * 2 != C_:
        raise RuntimeError("side cache shapes must be [B,Hkv,cap,C/2] and [B,Hkv,cap]")
    if packed.stride(3) != 1 or packed.stride(2) != C_ // 2 or scale.stride(2) != 1:
        raise RuntimeError("side cache token rows must be dense")


def quantize(key: torch.Tensor, channel_idx: torch.Tensor,
             out: Optional[tuple[torch.Tensor, torch.Tensor]] = None, t_dst: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """int4 codes (two per byte) of ``key[..., channel_idx]`` with one fp32 scale per token.

    Returns ``(packed[B,Hkv,T,C/2], scale[B,Hkv,T])`` views of a freshly allocated side cache, or
    writes rows ``t_dst .. t_dst+T`` of the cache given in ``out`` and returns it."""
    if key.dtype != torch.bfloat16 or key.dim() != 4:
        raise RuntimeError("key must be bf16 [B,Hkv,T,D]")
    B, Hkv, T, D = key.shape
    C_ = int(channel_idx.shape[-1])
    key = _rows_contiguous(key)
    channel_idx = channel_idx.to(device=key.device, dtype=torch.int32).contiguous()
    if out is None:
        packed, scale = alloc_side_cache(B, Hkv, t_dst + T, C_, key.device)
    else:
        packed, scale = out
    _check_side_cache(packed, scale, C_)
    if packed.shape[2] < t_dst + T:
        raise RuntimeError("side cache too small")
    check(_native.lib().kvb_quantize_pack(
        key.data_ptr(), key.stride(0), key.stride(1), key.stride(2), channel_idx.data_ptr(),
        packed.data_ptr(), packed.stride(0), packed.stride(1),
        scale.data_ptr(), scale.stride(0), scale.stride(1),
        B, Hkv, T, D, C_, t_dst, _dev(key), _stream(key.device)), "kvb_quantize_pack")
    if out is None:
        return packed[:, :, : t_dst + T], scale[:, :, : t_dst + T]
    return packed, scale


def quantize_append(key_row: torch.Tensor, channel_idx: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor,
                    t_dst: int) -> None:
    """Quantizes the single new row ``key_row[B,Hkv,1,D]`` into row ``t_dst`` of the side cache."""
    if key_row.dim() == 4:
        key_row = key_row[:, :, 0, :]
    key_row = _rows_contiguous(key_row)
    B, Hkv, D = key_row.shape
    C_ = int(channel_idx.shape[-1])
    _check_side_cache(packed, scale, C_)
    check(_native.lib().kvb_quantize_append(
        key_row.data_ptr(), key_row.stride(0), key_row.stride(1), channel_idx.data_ptr(),
        packed.data_ptr(), packed.stride(0), packed.stride(1),
        scale.data_ptr(), scale.stride(0), scale.stride(1),
        B, Hkv, D, C_, t_dst, _dev(key_row), _stream(key_row.device)), "kvb_quantize_append")


def unpack_codes(packed: torch.Tensor) -> torch.Tensor:
    """int8 codes ``[..., C]`` of a packed tensor ``[..., C/2]`` (helper for inspection and tests)."""
    lo = (packed << 4).view(torch.int8) >> 4
    hi = packed.view(torch.int8) >> 4
    return torch.stack((lo, hi), dim=-1).flatten(-2)


# ------------------------------------------------------------------------------------------
# stage 2: score
# ------------------------------------------------------------------------------------------

@dataclass
class ScoreResult:
    acc: Optional[torch.Tensor]    # int32 [B,Hq,T] exact partial dot products
    deq: Optional[torch.Tensor]    # fp32  [B,Hq,T] dequantised scores
    gmax: Optional[torch.Tensor]   # fp32  [B,Hkv,T] max over each GQA group
    hist: Optional[torch.Tensor]   # uint32-as-int32 [B*Hkv,4096] histogram of gmax keys


def score(query: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor, channel_idx: torch.Tensor,
          history_count: Optional[int] = None, *, want_acc: bool = True, want_deq: bool = True,
          want_gmax: bool = True, want_hist: bool = False) -> ScoreResult:
    """Exact int32 partial QK of one query token against the first ``history_count`` packed keys."""
    query = _query3(query)
    if query.dtype != torch.bfloat16:
        raise RuntimeError("query must be bf16")
    B, Hq, D = query.shape
    Hkv = packed.shape[1]
    C_ = int(channel_idx.shape[-1])
    _check_side_cache(packed, scale, C_)
    T = packed.shape[2] if history_count is None else int(history_count)
    if T > packed.shape[2]:
        raise RuntimeError("history_count exceeds the side cache")
    dev = query.device
    acc = torch.empty((B, Hq, T), dtype=torch.int32, device=dev) if want_acc else None
    deq = torch.empty((B, Hq, T), dtype=torch.float32, device=dev) if want_deq else None
    gmax = torch.empty((B, Hkv, T), dtype=torch.float32, device=dev) if (want_gmax or want_hist) else None
    hist = torch.zeros((B * Hkv, HIST_BINS), dtype=torch.int32, device=dev) if want_hist else None
    channel_idx = channel_idx.to(device=dev, dtype=torch.int32).contiguous()
    check(_native.lib().kvb_score_decode(
        query.data_ptr(), query.stride(0), query.stride(1),
        packed.data_ptr(), packed.stride(0), packed.stride(1),
        scale.data_ptr(), scale.stride(0), scale.stride(1), channel_idx.data_ptr(),
        B, Hq, Hkv, T, D, C_, _ptr(gmax), _ptr(acc), _ptr(deq), _ptr(hist),
        _dev(query), _stream(dev)), "kvb_score_decode")
    return ScoreResult(acc, deq, gmax, hist)


def score_candidates(query: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor, channel_idx: torch.Tensor,
                     history_count: int, top_k: int, tau: Optional[torch.Tensor] = None):
    """Candidate form of the scorer: per KV head the tokens whose group maximum reaches a sampled
    threshold, as 64-bit composites ``key << 32 | ~token``. Returns ``(cand uint64-as-int64 [B*Hkv,cap],
    count int32 [B*Hkv], tau fp32 [B*Hkv])``; ``count`` may exceed ``cap`` (entries beyond it are lost)."""
    query = _query3(query)
    B, Hq, D = query.shape
    Hkv = packed.shape[1]
    C_ = int(channel_idx.shape[-1])
    _check_side_cache(packed, scale, C_)
    T = int(history_count)
    dev = query.device
    lib = _native.lib()
    cap = lib.kvb_candidate_capacity(min(int(top_k), T))
    if cap == 0:
        raise RuntimeError("top_k too large for the candidate form")
    channel_idx = channel_idx.to(device=dev, dtype=torch.int32).contiguous()
    common = (query.data_ptr(), query.stride(0), query.stride(1), packed.data_ptr(), packed.stride(0), packed.stride(1),
              scale.data_ptr(), scale.stride(0), scale.stride(1), channel_idx.data_ptr(), B, Hq, Hkv, T, D, C_)
    if tau is None:
        tau = torch.empty((B * Hkv,), dtype=torch.float32, device=dev)
        check(lib.kvb_sample_thresholds(*common, int(top_k), tau.data_ptr(), _dev(query), _stream(dev)),
              "kvb_sample_thresholds")
    cand = torch.empty((B * Hkv, cap), dtype=torch.int64, device=dev)
    count = torch.zeros((B * Hkv, 32), dtype=torch.int32, device=dev)
    check(lib.kvb_score_candidates(*common, tau.data_ptr(), cand.data_ptr(), count.data_ptr(), cap, _dev(query),
                                   _stream(dev)), "kvb_score_candidates")
    return cand, count[:, 0], tau


# ------------------------------------------------------------------------------------------
# stage 3: select
# ------------------------------------------------------------------------------------------

def select(scores: torch.Tensor, k: int, *, payload: Optional[torch.Tensor] = None, idx_offset: int = 0,
           hist: Optional[torch.Tensor] = None, return_scores: bool = False,
           index_dtype: torch.dtype = torch.int64, order: str = "score"):
    """Exact top-``k`` columns of every row of ``scores[..., T]``; equal scores go to the lower index.

    ``order="score"`` returns them by (score desc, index asc), ``order="index"`` by ascending index.
    Returns indices ``[..., min(k,T)]`` (and the scores when asked). ``payload`` (int32, same
    shape as scores) replaces the column number as the index that is returned and tie-broken."""
    if order not in ("score", "index"):
        raise RuntimeError("order must be 'score' or 'index'")
    if scores.dtype != torch.float32:
        raise RuntimeError("scores must be float32")
    lead = scores.shape[:-1]
    T = scores.shape[-1]
    s2 = scores.reshape(-1, T)
    if s2.stride(-1) != 1:
        s2 = s2.contiguous()
    R = s2.shape[0]
    kk = min(int(k), T)
    dev = scores.device
    p2 = None
    if payload is not None:
        p2 = payload.reshape(-1, T).to(torch.int32)
        if p2.stride() != s2.stride():
            p2 = p2.contiguous()
            s2 = s2.contiguous()
    lib = _native.lib()
    ws_bytes = lib.kvb_select_topk_workspace_bytes(R, T, kk)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    out32 = torch.empty((R, kk), dtype=torch.int32, device=dev) if index_dtype == torch.int32 else None
    out64 = torch.empty((R, kk), dtype=torch.int64, device=dev) if index_dtype == torch.int64 else None
    if out32 is None and out64 is None:
        raise RuntimeError("index_dtype must be torch.int32 or torch.int64")
    outs = torch.empty((R, kk), dtype=torch.float32, device=dev) if return_scores else None
    check(lib.kvb_select_topk(
        s2.data_ptr(), s2.stride(0), _ptr(p2), R, T, int(k), int(idx_offset), int(order == "index"),
        _ptr(out32), _ptr(out64), _ptr(outs), _ptr(hist), ws.data_ptr(), ws_bytes,
        _dev(scores), _stream(dev)), "kvb_select_topk")
    idx = (out32 if out32 is not None else out64).reshape(*lead, kk)
    if return_scores:
        return idx, outs.reshape(*lead, kk)
    return idx


# ------------------------------------------------------------------------------------------
# final index list (EVAL:2938-3022)
# ------------------------------------------------------------------------------------------

def build_final_indices(selected: torch.Tensor, selected_valid: Optional[torch.Tensor], history_count: int,
                        key_count: int, protect_sink: int = 0, protect_recent: int = 0, keep_self: bool = True,
                        append_protected: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``selected ‖ sink ‖ recent ‖ self`` as int32 ``[..., S]`` with a bool validity mask."""
    lead = selected.shape[:-1]
    kk = selected.shape[-1]
    sel = selected.reshape(-1, kk).to(torch.int32).contiguous()
    sv = None if selected_valid is None else selected_valid.reshape(-1, kk).to(torch.uint8).contiguous()
    R = sel.shape[0]
    lib = _native.lib()
    S = lib.kvb_final_index_count(kk, history_count, protect_sink, protect_recent, int(keep_self))
    dev = selected.device
    out_idx = torch.empty((R, S), dtype=torch.int32, device=dev)
    out_valid = torch.empty((R, S), dtype=torch.uint8, device=dev)
    check(lib.kvb_build_final_indices(
        sel.data_ptr(), _ptr(sv), R, kk, history_count, key_count, protect_sink, protect_recent,
        int(keep_self), int(append_protected), out_idx.data_ptr(), out_valid.data_ptr(),
        _dev(selected), _stream(dev)), "kvb_build_final_indices")
    return out_idx.reshape(*lead, S), out_valid.reshape(*lead, S).bool()


# ------------------------------------------------------------------------------------------
# stage 4: sparse attention
# ------------------------------------------------------------------------------------------

def _mask_rows(attention_mask: Optional[torch.Tensor], B: int, Tk: int) -> Optional[torch.Tensor]:
    """HF additive mask ``[B,1,Tq,Tk']`` -> fp32 rows ``[B,Tk]`` of its first query row (EVAL:4637-4641)."""
    if attention_mask is None:
        return None
    m = attention_mask
    if m.dim() == 4:
        if m.shape[1] != 1:
            raise RuntimeError("per-head attention masks are not supported")
        m = m[:, 0, 0, :Tk]
    elif m.dim() == 2:
        m = m[:, :Tk]
    else:
        raise RuntimeError("attention_mask must be [B,1,Tq,Tk] or [B,Tk]")
    if m.shape[0] == 1 and B != 1:
        m = m.expand(B, -1)
    return m.to(torch.float32).contiguous()


def sparse_attend(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, indices: torch.Tensor,
                  valid: Optional[torch.Tensor] = None, scaling: Optional[float] = None,
                  attention_mask: Optional[torch.Tensor] = None, return_partial: bool = False):
    """Exact softmax attention of one query token over ``key/value[..., indices, :]``.

    ``indices`` is ``[B,Hkv,S]`` (one list per KV head, shared by its query heads) or ``[B,Hq,S]``
    (the layout of QCK:694-705), int32 or int64. Returns bf16 ``[B,1,Hq,D]``; with
    ``return_partial`` returns fp32 ``[B,Hq,D+2]`` = (un-normalised output, max, sum) instead."""
    query = _query3(query)
    B, Hq, D = query.shape
    if key.dim() != 4 or value.shape != key.shape:
        raise RuntimeError("key/value must be [B,Hkv,Tk,D] of equal shape")
    if key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16 or query.dtype != torch.bfloat16:
        raise RuntimeError("query/key/value must be bf16")
    Hkv, Tk = key.shape[1], key.shape[2]
    key = _rows_contiguous(key)
    value = _rows_contiguous(value)
    if indices.dim() != 3 or indices.shape[0] != B:
        raise RuntimeError("indices must be [B,H,S]")
    Hi, S = indices.shape[1], indices.shape[2]
    if indices.dtype not in (torch.int32, torch.int64):
        raise RuntimeError("indices must be int32 or int64")
    indices = indices.contiguous()
    v8 = None if valid is None else valid.to(torch.uint8).contiguous()
    if scaling is None:
        scaling = float(D) ** -0.5
    dev = query.device
    mask = _mask_rows(attention_mask, B, Tk)
    lib = _native.lib()
    ws_bytes = lib.kvb_sparse_attend_workspace_bytes(B, Hq, Hi, S)
    if ws_bytes == 0:
        raise RuntimeError("kvb_sparse_attend: unsupported shape")
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    out = None if return_partial else torch.empty((B, 1, Hq, D), dtype=torch.bfloat16, device=dev)
    part = torch.empty((B, Hq, D + 2), dtype=torch.float32, device=dev) if return_partial else None
    check(lib.kvb_sparse_attend(
        query.data_ptr(), query.stride(0), query.stride(1),
        key.data_ptr(), key.stride(0), key.stride(1), key.stride(2),
        value.data_ptr(), value.stride(0), value.stride(1), value.stride(2),
        indices.data_ptr(), int(indices.dtype == torch.int64), _ptr(v8),
        _ptr(mask), 0 if mask is None else mask.stride(0),
        B, Hq, Hkv, Hi, Tk, D, S, float(scaling), _ptr(out), _ptr(part), ws.data_ptr(), ws_bytes,
        _dev(query), _stream(dev)), "kvb_sparse_attend")
    return part if return_partial else out


def attend_selected(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, selected: torch.Tensor,
                    history_count: int, *, id_base: int = 0, protect_sink: int = 0, protect_recent: int = 0,
                    keep_self: bool = True, append_protected: bool = False, scaling: Optional[float] = None,
                    attention_mask: Optional[torch.Tensor] = None, return_partial: bool = False,
                    selected_count: Optional[torch.Tensor] = None):
    """Attention over the implicit list ``selected ‖ sink ‖ recent ‖ self`` (one list per KV head,
    int32 ``[B,Hkv,kk]``). Ids outside ``[id_base, id_base + history_count)`` contribute nothing,
    which is how a sequence shard attends to the part of a global selection that it owns. With
    ``selected_count`` (int32 ``[B*Hkv]``) only the first ``selected_count[r]`` entries of row ``r`` are used."""
    query = _query3(query)
    B, Hq, D = query.shape
    Hkv, Tk = key.shape[1], key.shape[2]
    key = _rows_contiguous(key)
    value = _rows_contiguous(value)
    if selected.dtype != torch.int32 or selected.dim() != 3 or selected.shape[1] != Hkv:
        raise RuntimeError("selected must be int32 [B,Hkv,kk]")
    selected = selected.contiguous()
    kk = selected.shape[2]
    if scaling is None:
        scaling = float(D) ** -0.5
    dev = query.device
    mask = _mask_rows(attention_mask, B, Tk)
    lib = _native.lib()
    S = lib.kvb_final_index_count(kk, history_count, protect_sink, protect_recent, int(keep_self))
    ws_bytes = lib.kvb_sparse_attend_workspace_bytes(B, Hq, Hkv, S)
    ws = torch.empty(max(ws_bytes, 256), dtype=torch.uint8, device=dev)
    out = None if return_partial else torch.empty((B, 1, Hq, D), dtype=torch.bfloat16, device=dev)
    part = torch.empty((B, Hq, D + 2), dtype=torch.float32, device=dev) if return_partial else None
    check(lib.kvb_attend_selected(
        query.data_ptr(), query.stride(0), query.stride(1),
        key.data_ptr(), key.stride(0), key.stride(1), key.stride(2),
        value.data_ptr(), value.stride(0), value.stride(1), value.stride(2),
        selected.data_ptr(), kk, _ptr(selected_count), int(id_base), int(history_count), int(protect_sink), int(protect_recent),
        int(keep_self), int(append_protected), _ptr(mask), 0 if mask is None else mask.stride(0),
        B, Hq, Hkv, Tk, D, float(scaling), _ptr(out), _ptr(part), ws.data_ptr(), ws.numel(),
        _dev(query), _stream(dev)), "kvb_attend_selected")
    return part if return_partial else out


def sparq_alpha(query: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor, channel_idx: torch.Tensor,
                history_count: int, selected: torch.Tensor, *, selected_count: Optional[torch.Tensor] = None,
                attention_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax mass, under the approximate (int4 partial) logits, of the tokens in ``selected`` (int32
    ``[B,Hkv,kk]``) among all ``history_count`` cached tokens: fp32 ``[B,Hq]`` (the alpha of the reference's
    SparQ blend, EVAL:2720-2722)."""
    query = _query3(query)
    B, Hq, D = query.shape
    Hkv = packed.shape[1]
    C_ = int(channel_idx.shape[-1])
    _check_side_cache(packed, scale, C_)
    T = int(history_count)
    dev = query.device
    selected = selected.to(torch.int32).contiguous()
    cnt = None if selected_count is None else selected_count.reshape(-1).to(torch.int32).contiguous()
    mask = _mask_rows(attention_mask, B, T)
    lib = _native.lib()
    ws = torch.empty(max(256, lib.kvb_sparq_alpha_workspace_bytes(B, Hq, T)), dtype=torch.uint8, device=dev)
    alpha = torch.empty((B, Hq), dtype=torch.float32, device=dev)
    check(lib.kvb_sparq_alpha(
        query.data_ptr(), query.stride(0), query.stride(1), packed.data_ptr(), packed.stride(0), packed.stride(1),
        scale.data_ptr(), scale.stride(0), scale.stride(1), channel_idx.data_ptr(), _ptr(mask),
        0 if mask is None else mask.stride(0), selected.data_ptr(), int(selected.shape[-1]), _ptr(cnt),
        B, Hq, Hkv, T, D, C_, alpha.data_ptr(), ws.data_ptr(), ws.numel(), _dev(query), _stream(dev)), "kvb_sparq_alpha")
    return alpha


def attend_selected_blend(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, selected: torch.Tensor,
                          history_count: int, alpha: torch.Tensor, value_mean: torch.Tensor, *, keep_self: bool = False,
                          scaling: Optional[float] = None, attention_mask: Optional[torch.Tensor] = None,
                          selected_count: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``value_mean + alpha * (attention over selected - value_mean)`` (``torch.lerp(mean, exact, alpha)`` of
    EVAL:2722) in one attention call: ``alpha`` fp32 ``[B,Hq]``, ``value_mean`` fp32 ``[B,Hkv,D]``."""
    query = _query3(query)
    B, Hq, D = query.shape
    Hkv, Tk = key.shape[1], key.shape[2]
    key = _rows_contiguous(key)
    value = _rows_contiguous(value)
    selected = selected.to(torch.int32).contiguous()
    kk = selected.shape[2]
    cnt = None if selected_count is None else selected_count.reshape(-1).to(torch.int32).contiguous()
    if scaling is None:
        scaling = float(D) ** -0.5
    dev = query.device
    mask = _mask_rows(attention_mask, B, Tk)
    alpha = alpha.to(torch.float32).contiguous()
    value_mean = value_mean.to(torch.float32).contiguous()
    lib = _native.lib()
    S = lib.kvb_final_index_count(kk, history_count, 0, 0, int(keep_self))
    ws = torch.empty(max(lib.kvb_sparse_attend_workspace_bytes(B, Hq, Hkv, S), 256), dtype=torch.uint8, device=dev)
    out = torch.empty((B, 1, Hq, D), dtype=torch.bfloat16, device=dev)
    check(lib.kvb_attend_selected_blend(
        query.data_ptr(), query.stride(0), query.stride(1),
        key.data_ptr(), key.stride(0), key.stride(1), key.stride(2),
        value.data_ptr(), value.stride(0), value.stride(1), value.stride(2),
        selected.data_ptr(), kk, _ptr(cnt), int(history_count), int(keep_self), _ptr(mask),
        0 if mask is None else mask.stride(0), alpha.data_ptr(), value_mean.data_ptr(),
        B, Hq, Hkv, Tk, D, float(scaling), out.data_ptr(), ws.data_ptr(), ws.numel(), _dev(query), _stream(dev)),
        "kvb_attend_selected_blend")
    return out


def shard_candidates(query: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor, channel_idx: torch.Tensor,
                     history_count: int, top_k: int, id_offset: int = 0,
                     workspace: Optional[torch.Tensor] = None, split_k: int = 0) -> Optional[torch.Tensor]:
    """Exact local top-``k`` of a sequence shard as 64-bit composites with GLOBAL token ids, int64
    ``[B*Hkv, min(k,T)]``, unordered except that the ``split_k`` best come first when ``0 < split_k < k``.
    Returns ``None`` when the configuration has no candidate front end (the caller then uses
    ``score`` + ``select``)."""
    query = _query3(query)
    B, Hq, D = query.shape
    Hkv = packed.shape[1]
    C_ = int(channel_idx.shape[-1])
    _check_side_cache(packed, scale, C_)
    T = int(history_count)
    dev = query.device
    lib = _native.lib()
    need = lib.kvb_shard_candidates_workspace_bytes(B, Hkv, T, int(top_k))
    ws = workspace if workspace is not None and workspace.numel() >= need else torch.empty(need, dtype=torch.uint8, device=dev)
    out = torch.empty((B * Hkv, min(int(top_k), T)), dtype=torch.int64, device=dev)
    rc = lib.kvb_shard_candidates(
        query.data_ptr(), query.stride(0), query.stride(1), packed.data_ptr(), packed.stride(0), packed.stride(1),
        scale.data_ptr(), scale.stride(0), scale.stride(1), channel_idx.data_ptr(), B, Hq, Hkv, T, D, C_, int(top_k),
        int(split_k), int(id_offset), out.data_ptr(), ws.data_ptr(), ws.numel(), _dev(query), _stream(dev))
    if rc == 1:          # KVB_BAD_SHAPE: not a streaming configuration / k too large for the candidate capacity
        return None
    check(rc, "kvb_shard_candidates")
    return out


def score_select(query: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor, channel_idx: torch.Tensor,
                 history_count: int, top_k: int, ascending: bool = True,
                 workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Stages 2 and 3 in one call: the exact top-``k`` token ids per (batch, KV head) from the int4 cache, int32
    ``[B,Hkv,min(k,T)]`` (ascending when asked and the history is short enough for the on-chip bitmap). Falls
    back to ``score`` + ``select`` for configurations without the candidate front end."""
    query = _query3(query)
    B, Hq, D = query.shape
    Hkv = packed.shape[1]
    C_ = int(channel_idx.shape[-1])
    _check_side_cache(packed, scale, C_)
    T = int(history_count)
    dev = query.device
    lib = _native.lib()
    kk = min(int(top_k), T)
    need = lib.kvb_shard_candidates_workspace_bytes(B, Hkv, T, int(top_k))
    ws = workspace if workspace is not None and workspace.numel() >= need else torch.empty(need, dtype=torch.uint8, device=dev)
    out = torch.empty((B, Hkv, kk), dtype=torch.int32, device=dev)
    rc = lib.kvb_score_select(
        query.data_ptr(), query.stride(0), query.stride(1), packed.data_ptr(), packed.stride(0), packed.stride(1),
        scale.data_ptr(), scale.stride(0), scale.stride(1), channel_idx.data_ptr(), B, Hq, Hkv, T, D, C_, int(top_k),
        int(ascending), out.data_ptr(), ws.data_ptr(), ws.numel(), _dev(query), _stream(dev))
    if rc == 1:          # KVB_BAD_SHAPE: no candidate front end for this shape
        r = score(query, packed, scale, channel_idx, T, want_acc=False, want_deq=False, want_hist=True)
        return select(r.gmax, top_k, hist=r.hist, index_dtype=torch.int32, order="index" if ascending else "score")
    check(rc, "kvb_score_select")
    return out


def rerank_union(query: torch.Tensor, key: torch.Tensor, lists, history_count: int, keep: int, *,
                 counts=None, scaling: Optional[float] = None, attention_mask: Optional[torch.Tensor] = None,
                 force_sink: int = 0, force_recent: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Exact rerank of the union of up to three id lists (current candidates, previous candidates, previous
    final set; the reference's rerank / reuse modes, EVAL:4147-4311, with lists in place of its ``[B,H,T]``
    masks). ``lists``: int32 ``[B,Hi,n_i]`` tensors (``None`` entries allowed after the first), ``Hi`` = KV heads
    (one list per GQA group, scored by the maximum over its query heads) or query heads. Returns
    ``(ids int32 [B,Hi,keep] ascending, -1 padded; count int32 [B,Hi])`` — the ``min(keep, |union|)`` best by
    (exact score desc, id asc)."""
    query = _query3(query)
    B, Hq, D = query.shape
    key = _rows_contiguous(key)
    Hkv = key.shape[1]
    lists = list(lists) + [None] * (3 - len(lists))
    counts = list(counts) + [None] * (3 - len(counts)) if counts is not None else [None] * 3
    if lists[0] is None:
        raise RuntimeError("the first list (current candidates) is required")
    Hi = lists[0].shape[1]
    dev = query.device
    ls = [None if l is None else l.to(torch.int32).contiguous() for l in lists]
    cs = [None if c is None else c.to(torch.int32).contiguous() for c in counts]
    for l in ls:
        if l is not None and (l.dim() != 3 or l.shape[0] != B or l.shape[1] != Hi):
            raise RuntimeError("lists must be [B,Hi,n] with the same Hi")
    ns = [0 if l is None else int(l.shape[2]) for l in ls]
    if scaling is None:
        scaling = float(D) ** -0.5
    mask = _mask_rows(attention_mask, B, int(history_count))
    lib = _native.lib()
    total = min(int(history_count), sum(ns) + int(force_sink) + int(force_recent))
    ws_bytes = lib.kvb_rerank_union_workspace_bytes(B * Hi, total)
    if ws_bytes == 0:
        raise RuntimeError("kvb_rerank_union: the candidate union is too large (more than 16384 entries)")
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    out = torch.empty((B, Hi, int(keep)), dtype=torch.int32, device=dev)
    cnt = torch.empty((B, Hi), dtype=torch.int32, device=dev)
    check(lib.kvb_rerank_union(
        query.data_ptr(), query.stride(0), query.stride(1), key.data_ptr(), key.stride(0), key.stride(1), key.stride(2),
        ls[0].data_ptr(), ns[0], _ptr(cs[0]), _ptr(ls[1]), ns[1], _ptr(cs[1]), _ptr(ls[2]), ns[2], _ptr(cs[2]),
        int(force_sink), int(force_recent), _ptr(mask), 0 if mask is None else mask.stride(0),
        B, Hq, Hkv, Hi, int(history_count), D, float(scaling), int(keep), out.data_ptr(), cnt.data_ptr(),
        ws.data_ptr(), ws_bytes, _dev(query), _stream(dev)), "kvb_rerank_union")
    return out, cnt


def expand_final(ids: torch.Tensor, history_count: int, *, count: Optional[torch.Tensor] = None, force_sink: int = 0,
                 force_recent: int = 0, block_size: int = 1, capacity: Optional[int] = None):
    """The keep set of the rerank modes as a list: ``ids`` (int32 ``[..., n]``, -1 / out-of-range entries
    ignored) plus the protected ranges (EVAL:4306-4311), widened to aligned blocks of ``block_size`` tokens
    (EVAL:2914-2922), de-duplicated and ascending. Returns ``(ids int32 [..., capacity] -1 padded, count)``."""
    lead, n = ids.shape[:-1], ids.shape[-1]
    l2 = ids.reshape(-1, n).to(torch.int32).contiguous()
    R = l2.shape[0]
    c2 = None if count is None else count.reshape(-1).to(torch.int32).contiguous()
    if capacity is None:
        capacity = min(int(history_count), (n + int(force_sink) + int(force_recent)) * max(1, int(block_size)))
    out = torch.empty((R, int(capacity)), dtype=torch.int32, device=ids.device)
    cnt = torch.empty((R,), dtype=torch.int32, device=ids.device)
    check(_native.lib().kvb_expand_final(l2.data_ptr(), n, _ptr(c2), R, int(history_count), int(force_sink),
                                         int(force_recent), int(block_size), out.data_ptr(), int(capacity), cnt.data_ptr(),
                                         _dev(ids), _stream(ids.device)), "kvb_expand_final")
    return out.reshape(*lead, int(capacity)), cnt.reshape(*lead)


def merge_candidates(gathered: torch.Tensor, top_k: int, id_range: int, prefix_k: int = 0,
                     own: Optional[tuple[int, int]] = None):
    """Global top-``k`` token ids (int32 ``[R, k']``) from all-gathered composite lists int64 ``[N,R,kk]``.
    ``prefix_k``: every list has its ``prefix_k`` best entries first (``shard_candidates(split_k=...)``),
    which lets the kernel work on the prefixes alone when that is provably enough. ``own = (base, limit)``:
    also return the winners with ``base <= id < limit`` compacted per row and their count:
    ``(ids, owned int32 [R,k'], owned_count int32 [R])``."""
    N, R, kk = gathered.shape
    gathered = gathered.contiguous()
    kout = min(int(top_k), N * kk)
    dev = gathered.device
    out = torch.empty((R, kout), dtype=torch.int32, device=dev)
    owned = cnt = None
    base = limit = 0
    if own is not None:
        base, limit = int(own[0]), int(own[1])
        owned = torch.empty((R, kout), dtype=torch.int32, device=dev)
        cnt = torch.empty((R,), dtype=torch.int32, device=dev)
    check(_native.lib().kvb_merge_candidates(gathered.data_ptr(), N, R, kk, int(top_k), int(id_range), int(prefix_k),
                                             out.data_ptr(), base, limit, _ptr(owned), _ptr(cnt),
                                             _dev(gathered), _stream(dev)), "kvb_merge_candidates")
    return out if own is None else (out, owned, cnt)


def lse_merge(partials: torch.Tensor) -> torch.Tensor:
    """Combines shard partials fp32 ``[N,B,Hq,D+2]`` into bf16 ``[B,1,Hq,D]``."""
    N, B, Hq, PW = partials.shape
    partials = partials.contiguous()
    out = torch.empty((B, 1, Hq, PW - 2), dtype=torch.bfloat16, device=partials.device)
    check(_native.lib().kvb_lse_merge(partials.data_ptr(), N, B, Hq, PW - 2, out.data_ptr(),
                                      _dev(partials), _stream(partials.device)), "kvb_lse_merge")
    return out


# ------------------------------------------------------------------------------------------
# chunked prefill: block scoring and block selection
# ------------------------------------------------------------------------------------------

PREFILL_BLOCK = 64


def quantize_query_tokens(query: torch.Tensor, channel_idx: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-token int8 codes of a query chunk bf16 ``[B,Hq,Tq,D]`` over the channels of each head's KV
    head: returns ``(qcode int8 [B,Hq,Tq,C], qscale fp32 [B,Hq,Tq])``."""
    if query.dtype != torch.bfloat16 or query.dim() != 4:
        raise RuntimeError("query must be bf16 [B,Hq,Tq,D]")
    if query.stride(-1) != 1:
        query = query.contiguous()
    B, Hq, Tq, D = query.shape
    Hkv, C_ = channel_idx.shape
    dev = query.device
    channel_idx = channel_idx.to(device=dev, dtype=torch.int32).contiguous()
    qcode = torch.empty((B, Hq, Tq, C_), dtype=torch.int8, device=dev)
    qscale = torch.empty((B, Hq, Tq), dtype=torch.float32, device=dev)
    check(_native.lib().kvb_quantize_query_tokens(
        query.data_ptr(), query.stride(0), query.stride(1), query.stride(2), channel_idx.data_ptr(),
        qcode.data_ptr(), qscale.data_ptr(), B, Hq, Hkv, Tq, D, C_, _dev(query), _stream(dev)),
        "kvb_quantize_query_tokens")
    return qcode, qscale


PREFILL_ENGINES = {"auto": 0, "mma": 1, "i8": 2, "f16": 3}


class WidenedKeys:
    """The int4 key codes of a side cache widened once to tensor-core operands (fp16 values or int8 bytes of the
    same integers) in the core-matrix tile layout the prefill scorer reads: ``[B*Hkv, capacity/128, tile]``
    bytes. A chunked prefill scores every chunk of queries against the same keys, so the widening is paid once
    per cache (or once per appended range: ``update`` re-widens from ``first_token`` on), not once per CTA."""

    def __init__(self, packed: torch.Tensor, key_count: Optional[int] = None, engine: str = "f16",
                 capacity: Optional[int] = None):
        if engine not in ("f16", "i8"):
            raise ValueError("engine must be 'f16' or 'i8'")
        B, Hkv, cap_rows, half_c = packed.shape
        self.engine, self.B, self.Hkv, self.C = engine, B, Hkv, 2 * half_c
        self.capacity = int(capacity if capacity is not None else cap_rows)
        nbytes = _native.lib().kvb_prefill_operand_bytes(B, Hkv, self.capacity, self.C, PREFILL_ENGINES[engine])
        if nbytes == 0:
            raise ValueError("unsupported shape for widened prefill operands")
        self.buffer = torch.empty(nbytes, dtype=torch.uint8, device=packed.device)
        self.key_count = 0
        self.update(packed, packed.shape[2] if key_count is None else int(key_count), 0)

    def update(self, packed: torch.Tensor, key_count: int, first_token: int) -> None:
        """(Re-)widens the tokens ``first_token .. key_count-1`` (whole tiles of 128 from the tile of ``first_token``)."""
        if key_count > self.capacity:
            raise ValueError("key_count exceeds the capacity of the widened buffer")
        check(_native.lib().kvb_widen_keys(
            packed.data_ptr(), packed.stride(0), packed.stride(1), self.B, self.Hkv, int(key_count), self.capacity,
            self.C, PREFILL_ENGINES[self.engine], int(first_token), self.buffer.data_ptr(), self.buffer.numel(),
            _dev(packed), _stream(packed.device)), "kvb_widen_keys")
        self.key_count = int(key_count)


def score_prefill_blocks(qcode: torch.Tensor, qscale: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor,
                         key_count: Optional[int] = None, engine: str = "auto",
                         widened: Optional[WidenedKeys] = None) -> torch.Tensor:
    """Block scores fp32 ``[B,Hkv,Tq,ceil(Tk/64)]``: max over the GQA group and the 64 tokens of each
    key block of the dequantised int8 x int4 partial score; every query sees all ``key_count`` keys.
    ``engine``: ``auto`` (tensor-memory path on pre-widened operands: ``widened`` if given, else widened here
    for this call), ``mma`` (warp-level int8 MMA), ``i8`` / ``f16`` (tcgen05, codes widened inside every CTA;
    int8 operands and int32 accumulators / the same integers as fp16 operands with fp32 accumulators),
    ``i8w`` / ``f16w`` (tcgen05 on pre-widened operands); all produce identical bits."""
    B, Hq, Tq, C_ = qcode.shape
    Hkv = packed.shape[1]
    _check_side_cache(packed, scale, C_)
    Tk = packed.shape[2] if key_count is None else int(key_count)
    dev = qcode.device
    nblk = (Tk + PREFILL_BLOCK - 1) // PREFILL_BLOCK
    out = torch.empty((B, Hkv, Tq, nblk), dtype=torch.float32, device=dev)
    if engine in ("auto", "f16w", "i8w") or widened is not None:
        if widened is None:
            widened = WidenedKeys(packed, Tk, "i8" if engine == "i8w" else "f16", capacity=Tk)
        if widened.key_count < Tk or widened.C != C_:
            raise ValueError("the widened operands do not cover the keys asked for")
        check(_native.lib().kvb_score_prefill_blocks_widened(
            qcode.contiguous().data_ptr(), qscale.contiguous().data_ptr(), widened.buffer.data_ptr(),
            widened.buffer.numel(), widened.capacity, scale.data_ptr(), scale.stride(0), scale.stride(1),
            B, Hq, Hkv, Tq, Tk, C_, PREFILL_BLOCK, out.data_ptr(), PREFILL_ENGINES[widened.engine], _dev(qcode),
            _stream(dev)), "kvb_score_prefill_blocks_widened")
        return out
    check(_native.lib().kvb_score_prefill_blocks_engine(
        qcode.contiguous().data_ptr(), qscale.contiguous().data_ptr(),
        packed.data_ptr(), packed.stride(0), packed.stride(1),
        scale.data_ptr(), scale.stride(0), scale.stride(1),
        B, Hq, Hkv, Tq, Tk, C_, PREFILL_BLOCK, out.data_ptr(), PREFILL_ENGINES[engine], _dev(qcode), _stream(dev)),
        "kvb_score_prefill_blocks_engine")
    return out


def block_topk(block_scores: torch.Tensor, k: int, return_scores: bool = False):
    """The ``min(k, nblk)`` best blocks of every row ``[..., nblk]`` ordered by (score desc, block asc),
    int32 ``[..., kk]``."""
    lead, nblk = block_scores.shape[:-1], block_scores.shape[-1]
    s2 = block_scores.reshape(-1, nblk)
    if s2.stride(-1) != 1:
        s2 = s2.contiguous()
    R, kk = s2.shape[0], min(int(k), nblk)
    dev = block_scores.device
    idx = torch.empty((R, kk), dtype=torch.int32, device=dev)
    val = torch.empty((R, kk), dtype=torch.float32, device=dev) if return_scores else None
    check(_native.lib().kvb_block_topk(s2.data_ptr(), s2.stride(0), R, nblk, int(k), idx.data_ptr(), _ptr(val),
                                       _dev(block_scores), _stream(dev)), "kvb_block_topk")
    idx = idx.reshape(*lead, kk)
    return (idx, val.reshape(*lead, kk)) if return_scores else idx


def prefill_select_blocks(query: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor, channel_idx: torch.Tensor,
                          key_count: int, top_blocks: int = 32):
    """Query chunk ``[B,Hq,Tq,D]`` -> ``(block_idx int32 [B,Hkv,Tq,top_blocks], block_scores)``."""
    qcode, qscale = quantize_query_tokens(query, channel_idx)
    bs = score_prefill_blocks(qcode, qscale, packed, scale, key_count)
    return block_topk(bs, top_blocks), bs


# ------------------------------------------------------------------------------------------
# requests of different lengths over paged K/V: plan, append, attend
# ------------------------------------------------------------------------------------------

@dataclass
class PagePlan:
    """One serving step's bookkeeping (``page_plan``); everything is on the device."""
    cu_q: torch.Tensor          # int32 [B+1] first new token of every request; cu_q[B] is their number
    kv_len: torch.Tensor        # int32 [B] tokens held once the new ones are stored
    free_count: torch.Tensor    # int32 [1] pages left on the free stack
    slot: torch.Tensor          # int64 [capacity] page * page_tokens + row of every new token, -1 behind the last
    position: torch.Tensor      # int32 [capacity] position in its request, -1 behind the last
    request: torch.Tensor       # int32 [capacity] the request it belongs to, -1 behind the last
    status: torch.Tensor        # int32 [4] all 0, or why nothing was planned (see page_plan)


def _device_ints(name: str, t: torch.Tensor, n: int, index: int, dtype=torch.int32) -> None:
    if t.dtype != dtype or t.dim() != 1 or (n >= 0 and t.shape[0] != n) or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a dense {str(dtype).split('.')[-1]} vector" + ("" if n < 0 else f" of {n}"))
    if t.get_device() != index:
        raise RuntimeError(f"{name} must be on the same device as the other operands")


def _check_page_table(page_table: torch.Tensor, batch: int, index: int) -> int:
    """Checks int32 ``[B,W]`` with dense rows; returns the row stride."""
    if page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise RuntimeError("page_table must be int32 [B, pages] with dense rows")
    (B, W), (s0, s1) = page_table.shape, page_table.stride()
    if B != batch or W < 1 or (s1 != 1 and W > 1) or (B > 1 and s0 < W):
        raise RuntimeError("page_table must be int32 [B, pages] with dense rows")
    if page_table.get_device() != index:
        raise RuntimeError("page_table must be on the same device as the other operands")
    return max(s0, W)


def page_plan(kv_len: torch.Tensor, q_len: torch.Tensor, page_table: torch.Tensor, free_pages: torch.Tensor,
              free_count: torch.Tensor, page_tokens: int, capacity: int, *, finished: Optional[torch.Tensor] = None,
              in_place: bool = False, out: Optional[PagePlan] = None) -> PagePlan:
    """Gives the ``q_len[b]`` new tokens of every request a page and a row, on the device.

    Request ``b`` holds ``kv_len[b]`` tokens in the pages ``page_table[b]`` (int32 ``[B, W]``), or starts over where
    ``finished[b]`` (bool or uint8) is set: its pages then go back on the free stack ``free_pages[:free_count]`` before
    new ones are taken, all in request order. ``page_table`` and ``free_pages`` are updated in place; the lengths and the
    count are returned, and with ``in_place`` written to ``kv_len`` and ``free_count`` themselves (a captured step).
    ``capacity``: size of the per-token outputs, at least the number of new tokens.

    A page belongs to one request: several table rows may name it for ``paged_attend`` (a shared prefix), but only one of
    them may ever finish.

    ``status`` of the result: pages lacking, tokens beyond ``capacity``, requests whose table row is too short, 1 if
    the stack or a finished length cannot be. Unless all are 0 nothing is changed and no token has a slot."""
    dev = kv_len.get_device()
    B = kv_len.shape[0] if kv_len.dim() == 1 else -1
    if B < 1 or B > 8192:
        raise RuntimeError("page_plan takes 1 to 8192 requests")
    _device_ints("kv_len", kv_len, B, dev)
    _device_ints("q_len", q_len, B, dev)
    table_stride = _check_page_table(page_table, B, dev)
    _device_ints("free_pages", free_pages, -1, dev)
    _device_ints("free_count", free_count, 1, dev)
    page_tokens, capacity = int(page_tokens), int(capacity)
    if page_tokens < 1 or page_tokens & (page_tokens - 1):
        raise RuntimeError("page_tokens must be a power of two")
    if capacity < 1 or free_pages.shape[0] < 1:
        raise RuntimeError("capacity and the number of pages must be positive")
    if finished is not None:
        if finished.dtype not in (torch.bool, torch.uint8) or finished.shape != (B,) or not finished.is_contiguous() \
                or finished.get_device() != dev:
            raise RuntimeError("finished must be a dense bool or uint8 vector, one element per request")
    if dev < 0:
        _dev(kv_len)
    if out is None:
        # one allocation for all outputs (the 64-bit one first): seven would take longer than the kernel
        ints = kv_len.new_empty(2 * B + 6 + 4 * capacity)
        slot, cu, now, left, pos, req, status = torch.split_with_sizes(ints, (2 * capacity, B + 1, B, 1, capacity, capacity, 4))
        out = PagePlan(cu, kv_len if in_place else now, free_count if in_place else left, slot.view(torch.int64), pos, req, status)
    else:
        if in_place and (out.kv_len is not kv_len or out.free_count is not free_count):
            raise RuntimeError("in_place needs the plan's own kv_len and free_count")
        for name, n in (("cu_q", B + 1), ("kv_len", B), ("free_count", 1), ("position", capacity), ("request", capacity),
                        ("status", 4)):
            _device_ints(name, getattr(out, name), n, dev)
        _device_ints("slot", out.slot, capacity, dev, torch.int64)
    check(_native.lib().kvb_page_plan(
        kv_len.data_ptr(), q_len.data_ptr(), None if finished is None else finished.data_ptr(), B, page_table.data_ptr(),
        table_stride, page_table.shape[1], free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), page_tokens,
        capacity, out.cu_q.data_ptr(), out.kv_len.data_ptr(), out.free_count.data_ptr(), out.slot.data_ptr(),
        out.position.data_ptr(), out.request.data_ptr(), out.status.data_ptr(), dev, _raw_stream(dev)), "kvb_page_plan")
    return out


def _check_pools(key_pool: torch.Tensor, value_pool: torch.Tensor, index: int):
    """Checks two page pools; returns their shape and strides."""
    shape = key_pool.shape
    if len(shape) != 4 or value_pool.shape != shape or value_pool.dtype != key_pool.dtype:
        raise RuntimeError("key_pool and value_pool must be [num_pages,Hkv,page_tokens,D] of equal shape and type")
    if key_pool.dtype != torch.bfloat16 and key_pool.dtype != torch.float16:
        raise RuntimeError("pools must be bf16 or fp16")
    if shape[2] < 1 or shape[2] & (shape[2] - 1):
        raise RuntimeError("page_tokens must be a power of two")
    if key_pool.get_device() != index or value_pool.get_device() != index:
        raise RuntimeError("pools must be on the same device as the other operands")
    ks, vs = key_pool.stride(), value_pool.stride()
    if ks[3] != 1 or vs[3] != 1 or (ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) & 7 \
            or (key_pool.data_ptr() | value_pool.data_ptr()) & 15:
        raise RuntimeError("pool rows must be contiguous and 16-byte aligned, strides multiples of 8 elements")
    return shape, ks, vs


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """``[N,H,D]`` with contiguous D and 16-byte aligned rows, copied only when it is not."""
    s = t.stride()
    return t if s[2] == 1 and not (s[0] | s[1]) & 7 and not t.data_ptr() & 15 else t.contiguous()


def paged_append(key_rows: torch.Tensor, value_rows: torch.Tensor, slot: torch.Tensor, key_pool: torch.Tensor,
                 value_pool: torch.Tensor) -> None:
    """Stores new K and V rows ``[N,Hkv,D]`` (any token and head strides) at their ``slot`` (int64 ``[N]`` of
    ``page_plan``) in the pools ``[num_pages,Hkv,page_tokens,D]``; rows whose slot is -1 are skipped. A slot that
    appears twice receives one of its rows, which one is not defined."""
    dev = key_pool.get_device()
    if key_rows.dim() != 3 or value_rows.shape != key_rows.shape:
        raise RuntimeError("key_rows and value_rows must be [N,Hkv,D] of equal shape")
    (num_pages, Hkv, P, D), ks, vs = _check_pools(key_pool, value_pool, dev)
    N, H, Dr = key_rows.shape
    if H != Hkv or Dr != D or key_rows.dtype != key_pool.dtype or value_rows.dtype != key_pool.dtype:
        raise RuntimeError("rows and pools must have the same heads, head size and type")
    if key_rows.get_device() != dev or value_rows.get_device() != dev:
        raise RuntimeError("rows must be on the same device as the pools")
    _device_ints("slot", slot, N, dev, torch.int64)
    if dev < 0:
        _dev(key_pool)
    if N == 0:
        return
    k, v = _aligned_rows(key_rows), _aligned_rows(value_rows)
    (k0, k1, _), (v0, v1, _) = k.stride(), v.stride()
    check(_native.lib().kvb_paged_append(
        k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, slot.data_ptr(), N, Hkv, D, key_pool.data_ptr(), ks[0], ks[1], ks[2],
        value_pool.data_ptr(), vs[0], vs[1], vs[2], num_pages, P, dev, _raw_stream(dev)), "kvb_paged_append")


@lru_cache(maxsize=4096)
def _paged_workspace_bytes(*shape: int) -> int:
    return _native.lib().kvb_paged_attend_workspace_bytes(*shape)


def paged_attend(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, page_table: torch.Tensor,
                 kv_len: torch.Tensor, *, cu_q: Optional[torch.Tensor] = None, max_q: int = 0,
                 scaling: Optional[float] = None, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None,
                 window: int = 0, prefix_len: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                 return_lse: bool = False):
    """Softmax attention of the new tokens of every request over all ``kv_len[b]`` tokens it holds in paged K/V, the
    new ones included (``paged_append`` them first). ``query`` is ``[N,Hq,D]``, the requests' tokens one after the
    other: rows ``cu_q[b] .. cu_q[b+1]`` (int32 ``[B+1]``) are the last tokens of request ``b``; without ``cu_q`` every
    request has one. Rows behind ``cu_q[B]`` (a padded, captured batch) are left as they are. Returns ``[N,Hq,D]``.

    Token at position ``p`` sees the keys ``j <= p``, and those below ``prefix_len[b]`` whatever ``p`` is, but none at or
    below ``p - window`` when a window is given. Scores are ``scaling * q.k`` (default ``D ** -0.5``), capped to
    ``softcap * tanh(. / softcap)`` when ``softcap > 0``, less ``slopes[head] * |p - j|`` when ``slopes`` (fp32 ``[Hq]``) are given.
    ``return_lse`` also returns the fp32 ``[N,Hq]`` logarithm of each row's sum of exponentials. A row that sees no key
    is zero, its logarithm -inf. ``max_q``: the largest number of new tokens of one request when the caller knows it;
    it chooses the kernel and never the result. K and V rows that some token of their request sees must be finite."""
    dev = query.get_device()
    if query.dim() != 3:
        raise RuntimeError("query must be [N,Hq,D]")
    (num_pages, Hkv, P, Dk), ks, vs = _check_pools(key_pool, value_pool, dev)
    N, Hq, D = query.shape
    dtype = query.dtype
    if dtype != key_pool.dtype:
        raise RuntimeError("query and pools must have the same type")
    if Dk != D or D not in (64, 128):
        raise RuntimeError("head size must be 64 or 128, the same for query and pools")
    if Hq < 1 or Hq % Hkv:
        raise RuntimeError("the number of query heads must be a multiple of the number of KV heads")
    B = kv_len.shape[0] if kv_len.dim() == 1 else -1
    if B < 1 or B > 8192:
        raise RuntimeError("paged_attend takes 1 to 8192 requests")
    _device_ints("kv_len", kv_len, B, dev)
    table_stride = _check_page_table(page_table, B, dev)
    if cu_q is not None:
        _device_ints("cu_q", cu_q, B + 1, dev)
    elif N != B:
        raise RuntimeError("without cu_q every request has one token: query must have one row per request")
    if prefix_len is not None:
        _device_ints("prefix_len", prefix_len, B, dev)
    if slopes is not None:
        _device_ints("slopes", slopes, Hq, dev, torch.float32)
    scaling = float(D) ** -0.5 if scaling is None else float(scaling)
    softcap, window, max_q = float(softcap), int(window), int(max_q)
    if not 0.0 < scaling < 3.0e38 or not 0.0 <= softcap < 3.0e38 or window < 0 or max_q < 0 \
            or (softcap and scaling > 3.0e38 * softcap):
        raise RuntimeError("scaling must be positive and finite, softcap, window and max_q not negative")
    if out is not None and (out.shape != query.shape or out.dtype != dtype or not out.is_contiguous()
                            or out.get_device() != dev or out.data_ptr() & 15):
        raise RuntimeError("out must be a dense, 16-byte aligned tensor of the query's shape and type")
    if dev < 0:
        _dev(query)
    query = _aligned_rows(query)
    device = query.device
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    lse = torch.empty_strided((N, Hq), (Hq, 1), dtype=torch.float32, device=device) if return_lse else None
    if N == 0:
        return (out, lse) if return_lse else out
    lib = _native.lib()
    W = page_table.shape[1]
    ws_bytes = _paged_workspace_bytes(N, B, Hq, Hkv, W, P, D, max_q)
    if ws_bytes == 0:
        raise RuntimeError("kvb_paged_attend: unsupported shape")
    ws = torch.empty_strided((ws_bytes,), (1,), dtype=torch.uint8, device=device)
    q0, q1, _ = query.stride()
    p = PagedAttendParams(                               # in the order of the struct
        query.data_ptr(), q0, q1, key_pool.data_ptr(), ks[0], ks[1], ks[2], value_pool.data_ptr(), vs[0], vs[1], vs[2],
        page_table.data_ptr(), table_stride, kv_len.data_ptr(), None if cu_q is None else cu_q.data_ptr(),
        None if prefix_len is None else prefix_len.data_ptr(), None if slopes is None else slopes.data_ptr(),
        0 if dtype == torch.bfloat16 else 1, N, B, Hq, Hkv, D, W, num_pages, P, max_q, window, scaling, softcap,
        out.data_ptr(), None if lse is None else lse.data_ptr(), ws.data_ptr(), ws_bytes)
    check(lib.kvb_paged_attend(C.byref(p), dev, _raw_stream(dev)), "kvb_paged_attend")
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------------------------------
# fused decode step
# ------------------------------------------------------------------------------------------

class DecodeStep:
    """One layer's decode step (append, score, select, final list, attend) through
    ``kvb_decode_step`` with a workspace that is allocated once and reused."""

    def __init__(self, top_k: int, protect_sink: int = 0, protect_recent: int = 0, keep_self: bool = True,
                 append_protected: bool = False, append_self: bool = True, ordered_selection: bool = True):
        """``ordered_selection=False`` lets the step emit (and attend to) the selected ids in any order: the
        same exact set, a few microseconds faster, but not reproducible to the last bit."""
        self.ordered_selection = bool(ordered_selection)
        self.top_k = int(top_k)
        self.protect_sink = int(protect_sink)
        self.protect_recent = int(protect_recent)
        self.keep_self = bool(keep_self)
        self.append_protected = bool(append_protected)
        self.append_self = bool(append_self)
        self._ws: Optional[torch.Tensor] = None

    def workspace(self, B: int, Hq: int, Hkv: int, history_count: int, device, top_k: Optional[int] = None) -> torch.Tensor:
        need = _native.lib().kvb_decode_step_workspace_bytes(
            B, Hq, Hkv, history_count, self.top_k if top_k is None else top_k, self.protect_sink, self.protect_recent,
            int(self.keep_self))
        if self._ws is None or self._ws.numel() < need or self._ws.device != torch.device(device):
            # headroom so that a growing history does not reallocate every step
            self._ws = torch.empty(int(need * 1.25) + 4096, dtype=torch.uint8, device=device)
        return self._ws

    def __call__(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, packed: torch.Tensor,
                 scale: torch.Tensor, channel_idx: torch.Tensor, scaling: Optional[float] = None,
                 attention_mask: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                 selected_out: Optional[torch.Tensor] = None, history_dev: Optional[torch.Tensor] = None,
                 advance_history: bool = False,
                 new_rows: Optional[tuple[torch.Tensor, torch.Tensor]] = None,
                 top_k: Optional[int] = None,
                 kv_pages: Optional[tuple[torch.Tensor, int]] = None) -> torch.Tensor:
        """``key``/``value`` hold history+1 rows (the last is the token being decoded); the side
        cache holds the history rows. Returns bf16 ``[B,1,Hq,D]``. ``top_k`` overrides the count given at
        construction for this call (a policy whose count follows the history length keeps ONE step object
        and one workspace).

        With ``history_dev`` (int32 device tensor of one element) the history length is read on
        the device and ``key``/``value`` are the whole cache (capacity rows): the same launch
        sequence then serves every step of a CUDA-graph replayed decode loop; ``advance_history``
        makes the step add one to it when it is done. ``new_rows = (k_row, v_row)`` (bf16 ``[B,Hkv,D]``
        dense): the step first stores them as row ``history`` of ``key`` / ``value``.

        ``kv_pages = (page_table, history)``: ``key`` / ``value`` are page pools ``[num_pages,Hkv,P,D]`` (P a power of
        two) and ``page_table`` (int32 ``[B, pages_per_sequence]``) maps token t of batch row b to page
        ``page_table[b, t // P]``; ``history`` is the history length (the decoded token is row ``history``)."""
        query = _query3(query)
        B, Hq, D = query.shape
        Hkv, key_count = key.shape[1], key.shape[2]
        if kv_pages is not None:
            page_table, paged_history = kv_pages
            if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B or not page_table.is_contiguous():
                raise RuntimeError("page_table must be a dense int32 [B, pages] tensor")
            if not (key.is_contiguous() and value.is_contiguous() and key.shape == value.shape):
                raise RuntimeError("paged K/V pools must be dense [num_pages,Hkv,P,D] tensors of one shape")
            key_count = int(paged_history) + 1
        T = key_count - 1
        if T < 1:
            raise RuntimeError("the fused step needs at least one history token")
        C_ = int(channel_idx.shape[-1])
        _check_side_cache(packed, scale, C_)
        if self.append_self and packed.shape[2] < key_count:
            raise RuntimeError("side cache has no room for the appended row")
        key = _rows_contiguous(key)
        value = _rows_contiguous(value)
        dev = query.device
        k_now = self.top_k if top_k is None else int(top_k)
        ws = self.workspace(B, Hq, Hkv, T, dev, k_now)
        if out is None:
            out = torch.empty((B, 1, Hq, D), dtype=torch.bfloat16, device=dev)
        mask = _mask_rows(attention_mask, B, key_count)
        p = DecodeStepParams()
        p.query, p.q_sb, p.q_sh = query.data_ptr(), query.stride(0), query.stride(1)
        p.key, p.k_sb, p.k_sh, p.k_st = key.data_ptr(), key.stride(0), key.stride(1), key.stride(2)
        p.value, p.v_sb, p.v_sh, p.v_st = value.data_ptr(), value.stride(0), value.stride(1), value.stride(2)
        p.packed, p.packed_sb, p.packed_sh = packed.data_ptr(), packed.stride(0), packed.stride(1)
        p.scale, p.scale_sb, p.scale_sh = scale.data_ptr(), scale.stride(0), scale.stride(1)
        p.channel_idx = channel_idx.data_ptr()
        p.mask, p.mask_sb = (_ptr(mask), 0 if mask is None else mask.stride(0))
        p.B, p.Hq, p.Hkv, p.D, p.C = B, Hq, Hkv, D, C_
        p.history_count = T
        p.top_k = k_now
        p.protect_sink, p.protect_recent = self.protect_sink, self.protect_recent
        p.keep_self, p.append_protected = int(self.keep_self), int(self.append_protected)
        p.append_self = int(self.append_self)
        p.scaling = float(D) ** -0.5 if scaling is None else float(scaling)
        p.out = out.data_ptr()
        p.sel_idx_out = _ptr(selected_out)
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
        p.history_count_dev = _ptr(history_dev)
        p.advance_history = int(advance_history)
        p.selected_any_order = 0 if self.ordered_selection else 1
        if kv_pages is not None:
            p.kv_page_table, p.kv_page_table_stride = page_table.data_ptr(), page_table.stride(0)
            p.kv_page_tokens = int(key.shape[2])
        if new_rows is not None:
            k_row, v_row = new_rows
            if not (k_row.is_contiguous() and v_row.is_contiguous() and k_row.dtype == v_row.dtype == torch.bfloat16
                    and k_row.numel() == v_row.numel() == B * Hkv * D):
                raise RuntimeError("new_rows must be two dense bf16 [B,Hkv,D] tensors")
            p.new_key_row, p.new_value_row = k_row.data_ptr(), v_row.data_ptr()
        check(_native.lib().kvb_decode_step(C.byref(p), _dev(query), _stream(dev)), "kvb_decode_step")
        return out


class GraphedDecode:
    """A decode loop step as ONE CUDA graph: copies of the step's inputs (query, new K row, new V
    row) from pinned host buffers, their scatter into the cache at the device-side position, the
    fused step, and the copy of the output back to a pinned host buffer. The history length lives
    on the device (``self.history``), so the same graph serves every step until the cache is full.

        g = GraphedDecode(DecodeStep(k), key_cache, value_cache, packed, scale, channel_idx, history=T)
        g.h_query.copy_(q); g.h_key_row.copy_(k_new); g.h_value_row.copy_(v_new)
        out = g()            # pinned host tensor [B,1,Hq,D]; history has advanced by one
    """

    def __init__(self, step: DecodeStep, key: torch.Tensor, value: torch.Tensor, packed: torch.Tensor,
                 scale: torch.Tensor, channel_idx: torch.Tensor, history: int, q_heads: int,
                 advance: bool = True, scaling: Optional[float] = None, zero_copy: bool = False):
        """``zero_copy``: the step's kernels read the new K/V rows from, and write the output to, the pinned host
        buffers themselves (pinned memory is addressable from the device), which takes the device-to-host copy node
        and a third of the host-to-device one out of the graph; only the query, which three kernels read, is still
        copied to the device first."""
        dev = key.device
        B, Hkv, rows, D = key.shape
        if history + 1 > rows:
            raise RuntimeError("the cache has no room for the decoded token")
        self.step, self.advance = step, advance
        self.history = torch.tensor([history], dtype=torch.int32, device=dev)
        # one pinned staging buffer and one device buffer: a single host-to-device copy per step
        nq, nkv = B * q_heads * D, B * Hkv * D
        self.h_in = torch.empty((nq + 2 * nkv,), dtype=torch.bfloat16).pin_memory()
        self.h_query = self.h_in[:nq].view(B, q_heads, D)
        self.h_key_row = self.h_in[nq:nq + nkv].view(B, Hkv, 1, D)
        self.h_value_row = self.h_in[nq + nkv:].view(B, Hkv, 1, D)
        self.h_out = torch.empty((B, 1, q_heads, D), dtype=torch.bfloat16).pin_memory()
        self._in = torch.empty((nq + 2 * nkv,), dtype=torch.bfloat16, device=dev)
        self._q = self._in[:nq].view(B, q_heads, D)
        self._k = self._in[nq:nq + nkv].view(B, Hkv, D)
        self._v = self._in[nq + nkv:].view(B, Hkv, D)
        self._out = torch.empty((B, 1, q_heads, D), dtype=torch.bfloat16, device=dev)
        self.stream = torch.cuda.Stream(dev)
        # warm-up contents: a well-spread query (an all-zero one would tie every score and send every row
        # through the slow exact-refinement path), zero K/V rows
        self.h_in.zero_()
        self.h_query.copy_(torch.randn((B, q_heads, D), generator=torch.Generator().manual_seed(0)).to(torch.bfloat16))

        self.zero_copy = bool(zero_copy)

        def body():
            if self.zero_copy:
                self._in[:nq].copy_(self.h_in[:nq], non_blocking=True)
                step(self._q, key, value, packed, scale, channel_idx, scaling=scaling, out=self.h_out,
                     history_dev=self.history, advance_history=advance,
                     new_rows=(self.h_key_row.view(B, Hkv, D), self.h_value_row.view(B, Hkv, D)))
                return
            self._in.copy_(self.h_in, non_blocking=True)
            # the step itself stores the new rows at the device-side position
            step(self._q, key, value, packed, scale, channel_idx, scaling=scaling, out=self._out,
                 history_dev=self.history, advance_history=advance, new_rows=(self._k, self._v))
            self.h_out.copy_(self._out, non_blocking=True)

        with torch.cuda.stream(self.stream):
            saved = self.history.clone()
            for _ in range(2):                       # warm-up outside capture (first-call set-up, workspace)
                body()
                self.history.copy_(saved)
            self.stream.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph, stream=self.stream):
                body()
            self.history.copy_(saved)                # capture does not run the work; start from `history`
            self.stream.synchronize()

    def __call__(self) -> torch.Tensor:
        with torch.cuda.stream(self.stream):
            self.graph.replay()
        self.stream.synchronize()
        return self.h_out
