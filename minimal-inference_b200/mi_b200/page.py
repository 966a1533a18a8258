"""KV append (kernel 1): drop-in for ``flashinfer.page.append_paged_kv_cache``.

Same arguments and in-place semantics as the call at model.py:207-216
(FlashInfer page.py:280-290, NHD layout). Keyword-only extensions fuse the
RoPE of model.py:169-170 into the same launch: pass the model's cos/sin
tables and the raw (un-rotated) K; pass ``q``/``q_out`` to rotate the
queries too.
"""
from __future__ import annotations

import torch

from . import capi
from ._tensor import (check_pool, check_scores, dtype_code, need_i32, need_on, on_device_of, ptr,
                      stream_of)


def append_paged_kv_cache(append_key: torch.Tensor, append_value: torch.Tensor,
                          batch_indices: torch.Tensor, positions: torch.Tensor,
                          paged_kv_cache: torch.Tensor, kv_indices: torch.Tensor,
                          kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor,
                          kv_layout: str = "NHD", *, rope_cos: torch.Tensor | None = None,
                          rope_sin: torch.Tensor | None = None,
                          rope_positions: torch.Tensor | None = None,
                          q: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                          scratch_page: int = -1, status: torch.Tensor | None = None) -> None:
    """Append ``append_key``/``append_value`` ``[nnz, Hkv, D]`` into the pages.

    Token ``i`` of request ``batch_indices[i]`` at ``positions[i]`` lands on
    page ``kv_indices[kv_indptr[b] + pos // ps]``, slot ``pos % ps``. With
    ``rope_cos``/``rope_sin`` (``[max_pos, D]``, model dtype) K is rotated on
    the way (bit-identical to ``apply_rotary_emb``); with ``q``/``q_out``
    (``[nnz, Hq, D]``) the queries are rotated into ``q_out``.
    """
    if kv_layout != "NHD":
        raise ValueError("only the NHD layout (the reference's) is supported")
    dev = paged_kv_cache.device
    num_pages, ps, hkv, d = check_pool(paged_kv_cache)
    nnz = append_key.shape[0]
    if append_key.shape != (nnz, hkv, d) or append_value.shape != (nnz, hkv, d):
        raise ValueError(f"append_key/value must be [nnz, {hkv}, {d}], got "
                         f"{tuple(append_key.shape)} / {tuple(append_value.shape)}")
    if append_key.stride(-1) != 1 or append_value.stride(-1) != 1:
        raise ValueError("append_key/value need a unit stride on head_dim")
    dt = paged_kv_cache.dtype
    for name, t in (("append_key", append_key), ("append_value", append_value)):
        if t.dtype != dt or t.device != dev:
            raise ValueError(f"{name} must be {dt} on {dev}")
    for name, t in (("batch_indices", batch_indices), ("positions", positions),
                    ("kv_indices", kv_indices), ("kv_indptr", kv_indptr)):
        need_i32(name, t, dev)
    if batch_indices.numel() < nnz or positions.numel() < nnz:
        raise ValueError("batch_indices/positions shorter than nnz")
    rope_max = 0
    if rope_cos is not None or rope_sin is not None:
        if rope_cos is None or rope_sin is None:
            raise ValueError("pass both rope_cos and rope_sin")
        if rope_cos.dtype != dt or rope_sin.dtype != dt or rope_cos.shape[-1] != d:
            raise ValueError("rope tables must be [max_pos, head_dim] in the pool dtype")
        if not (rope_cos.is_contiguous() and rope_sin.is_contiguous()):
            raise ValueError("rope tables must be contiguous")
        need_on("rope_cos", rope_cos, dev)
        need_on("rope_sin", rope_sin, dev)
        rope_max = rope_cos.shape[0]
    if rope_positions is not None:
        need_i32("rope_positions", rope_positions, dev)
    hq = 0
    if q is not None:
        if q_out is None or rope_max == 0:
            raise ValueError("query rotation needs q_out and the rope tables")
        hq = q.shape[1]
        if q.shape != (nnz, hq, d) or q_out.shape != (nnz, hq, d):
            raise ValueError("q/q_out must be [nnz, Hq, D]")
        if q.stride(-1) != 1 or q_out.stride(-1) != 1 or q.dtype != dt or q_out.dtype != dt:
            raise ValueError("q/q_out need the pool dtype and a unit stride on head_dim")
        need_on("q", q, dev)
        need_on("q_out", q_out, dev)
    if status is not None:
        need_i32("status", status, dev)
    capi.call(
        "mi_append_paged_kv_cache",
        append_key.data_ptr(), append_key.stride(0), append_key.stride(1),
        append_value.data_ptr(), append_value.stride(0), append_value.stride(1),
        batch_indices.data_ptr(), positions.data_ptr(), nnz,
        paged_kv_cache.data_ptr(), num_pages, ps, hkv, d, dtype_code(dt),
        kv_indices.data_ptr(), kv_indptr.data_ptr(), kv_indptr.numel() - 1,
        ptr(rope_cos), ptr(rope_sin), rope_max, ptr(rope_positions),
        ptr(q), q.stride(0) if q is not None else 0, q.stride(1) if q is not None else 0,
        ptr(q_out), q_out.stride(0) if q is not None else 0,
        q_out.stride(1) if q is not None else 0, hq,
        scratch_page, ptr(status), stream_of(paged_kv_cache))


def evict_paged_kv_cache(paged_kv_cache: torch.Tensor, scores: torch.Tensor,
                         kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                         kv_last_page_len: torch.Tensor, budget: int, *, recent: int = 0,
                         sinks: int = 0, max_len: int | None = None, return_kept: bool = False,
                         status: torch.Tensor | None = None) -> torch.Tensor | None:
    """Cut every request with more than ``budget`` cached tokens to ``budget``,
    in place, by accumulated attention weight (``mi_kv_evict``).

    ``paged_kv_cache`` is one layer's pool ``[P, 2, ps, Hkv, D]`` with
    ``scores [P, Hkv, ps]``, or the layers' pools in one tensor ``[L, P, 2,
    ps, Hkv, D]`` with ``scores [L, P, Hkv, ps]``; layers and KV heads choose
    by themselves. Kept are the first ``sinks`` slots, the last ``recent`` ones
    and the best-scored between them (equal scores: the lowest slot).
    Afterwards the kept tokens fill slots ``0 .. budget - 1``, the recent ones
    last and in order, the others in no particular order; scores move along and
    are 0 behind. The page table tensors are not changed.

    ``max_len``: an upper bound of the requests' lengths (default: all of
    ``kv_indices``' slots; at most 819200). It sizes the shared memory: with a
    large page table the longest request's length is the faster one to pass.
    Returns, with ``return_kept``, int32
    ``[(L,) B, Hkv, budget]``: the slot each kept token came from (-1: none)."""
    stacked = paged_kv_cache.dim() == 6
    layers = paged_kv_cache.shape[0] if stacked else 1
    if stacked and not paged_kv_cache.is_contiguous():
        raise ValueError("paged kv cache must be contiguous")
    if stacked and layers == 0:
        raise ValueError("no layers")
    kv = paged_kv_cache[0] if stacked else paged_kv_cache
    num_pages, ps, hkv, d = check_pool(kv)
    dev = paged_kv_cache.device
    if stacked:
        if scores.dim() != 4 or scores.shape[0] != layers or not scores.is_contiguous():
            raise ValueError(f"scores must be a contiguous [{layers}, {num_pages}, {hkv}, {ps}]")
        check_scores(scores[0], kv, dev)
    else:
        check_scores(scores, kv, dev)
    for name, t in (("kv_indices", kv_indices), ("kv_indptr", kv_indptr),
                    ("kv_last_page_len", kv_last_page_len)):
        need_i32(name, t, dev)
    batch = kv_indptr.numel() - 1
    if batch < 0 or kv_last_page_len.numel() < batch:
        raise ValueError("kv_indptr needs batch + 1 entries and kv_last_page_len batch")
    if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError(f"need 0 <= recent + sinks <= budget, got {recent} + {sinks}, {budget}")
    if max_len is None:
        max_len = max(1, kv_indices.numel() * ps)
    if max_len < 1:
        raise ValueError(f"max_len must be positive, got {max_len}")
    if status is not None:
        need_i32("status", status, dev)
    stream = stream_of(paged_kv_cache)
    kept = None
    if return_kept:
        shape = (batch, hkv, budget)
        kept = torch.empty((layers, *shape) if stacked else shape, dtype=torch.int32, device=dev)
    if kv_indices.numel() == 0:  # no request holds a page
        return kept.fill_(-1) if return_kept else None
    with on_device_of(paged_kv_cache):
        capi.call("mi_kv_evict", None, paged_kv_cache.data_ptr(),
                  paged_kv_cache.stride(0) if stacked else 0, scores.data_ptr(), layers,
                  num_pages, ps, hkv, d, dtype_code(paged_kv_cache.dtype), kv_indptr.data_ptr(),
                  kv_indices.data_ptr(), kv_last_page_len.data_ptr(), batch,
                  min(max_len, 2 ** 31 - 1), budget, recent, sinks, ptr(kept), ptr(status),
                  stream)
    return kept
