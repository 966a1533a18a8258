"""Token sampling on the device: temperature, top-k, top-p and min-p.

``sample_tokens`` chooses one token per row of logits in one launch, with one
given random number per row (the reference samples with torch softmax and
multinomial, temperature only; scheduler.py:310-343). It never synchronises
and can be captured into a CUDA graph.
"""
from __future__ import annotations

import torch

from . import capi
from ._tensor import dtype_code, need_on, on_device_of, ptr, stream_of

MAX_VOCAB = 1 << 18


def _setting(name: str, value, rows: int, dtype: torch.dtype, device):
    """A per-row device tensor -> (pointer, unused scalar); a number -> (None, it)."""
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {value.dtype}")
        if value.shape != (rows,) or not value.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [{rows}] tensor or a number, got "
                             f"{tuple(value.shape)}")
        need_on(name, value, device)
        return value.data_ptr(), 0
    return None, value


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, top_k=0,
                  top_p=1.0, min_p=0.0, *, out: torch.Tensor | None = None,
                  logprobs: torch.Tensor | None = None, return_logprobs: bool = False,
                  status: torch.Tensor | None = None):
    """One token per row of ``logits [rows, vocab]`` -> int32 ``[rows]``.

    ``uniform`` is fp32 ``[rows]`` in [0, 1). Each setting is a number or a
    per-row tensor (fp32; int32 for ``top_k``). The filters apply in the order
    top-k, top-p (of the mass top-k left), min-p (relative to the likeliest
    token); equal logits rank by index; the draw runs over the kept tokens by
    index. ``temperature <= 0`` takes the largest logit. ``top_k <= 0``,
    ``top_p >= 1`` and ``min_p <= 0`` are off. A row with no logit above -inf
    (NaN counts as -inf) gives -1 and flags NO_TOKEN in ``status``.

    With ``return_logprobs`` (or ``logprobs``, an fp32 ``[rows]`` output) also
    the token's log-probability under the unscaled, unfiltered logits, as
    ``(tokens, logprobs)``."""
    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, vocab], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"vocab {vocab} outside [1, {MAX_VOCAB}]")
    if logits.stride(1) != 1 and vocab > 1:
        raise ValueError("logits rows must be contiguous")
    if rows > 1 and logits.stride(0) < vocab:
        raise ValueError("logits rows overlap")
    dev = logits.device
    code = dtype_code(logits.dtype)
    if uniform.dtype != torch.float32 or uniform.shape != (rows,) or not uniform.is_contiguous():
        raise ValueError(f"uniform must be a contiguous float32 [{rows}]")
    need_on("uniform", uniform, dev)
    t_ptr, t_all = _setting("temperature", temperature, rows, torch.float32, dev)
    k_ptr, k_all = _setting("top_k", top_k, rows, torch.int32, dev)
    p_ptr, p_all = _setting("top_p", top_p, rows, torch.float32, dev)
    m_ptr, m_all = _setting("min_p", min_p, rows, torch.float32, dev)
    for name, t, dt in (("out", out, torch.int32), ("logprobs", logprobs, torch.float32)):
        if t is not None:
            if t.dtype != dt or t.shape != (rows,) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dt} [{rows}]")
            need_on(name, t, dev)
    if status is not None:
        if status.dtype != torch.int32 or status.numel() < 1:
            raise ValueError("status must be an int32 word")
        need_on("status", status, dev)
    stream = stream_of(logits)
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=dev)
    if logprobs is None and return_logprobs:
        logprobs = torch.empty(rows, dtype=torch.float32, device=dev)
    with on_device_of(logits):
        capi.call("mi_sample_tokens", logits.data_ptr(), logits.stride(0), rows, vocab, code,
                  uniform.data_ptr(), t_ptr, float(t_all), k_ptr, min(max(int(k_all), 0), MAX_VOCAB),
                  p_ptr, float(p_all), m_ptr, float(m_all), out.data_ptr(), ptr(logprobs),
                  ptr(status), stream)
    return (out, logprobs) if logprobs is not None else out
