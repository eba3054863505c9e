"""Logits of a decode step: penalties for repeated tokens, biases, temperature and a
grammar mask in one pass over the logits (``kvb_process_logits``).

The reference samples from ``softmax(logits / max(temperature, 1e-5))`` with nothing in
between; here the steps a serving loop needs before it come in one launch, in the order

    x = logits (float32)
    x = x / r if x > 0 else x * r       for every token seen in the prompt or the output
    x = x - frequency * count - presence * (count > 0)    count: occurrences in the output
    x = x + bias                        for each entry of the row's bias list
    x = x / max(temperature, 1e-5)
    x = -inf                            where the grammar mask's bit is 0
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .paged_decode import _allocator, _check_int32, _launch

_LOGIT_DTYPES = {torch.bfloat16: _lib.KVB_DTYPE_BF16, torch.float16: _lib.KVB_DTYPE_FP16,
                 torch.float32: _lib.KVB_DTYPE_FP32}


def _per_row(name: str, t: Optional[torch.Tensor], batch: int, device, dtype) -> int:
    """Address of a row parameter, 0 for one that is not given."""
    if t is None:
        return 0
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is not dtype or t.device != device or t.dim() != 1 or t.numel() != batch \
            or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous {dtype} tensor of {batch} entries on {device}")
    return t.data_ptr()


def process_logits(logits: torch.Tensor, token_ids: Optional[torch.Tensor] = None,
                   prompt_lens: Optional[torch.Tensor] = None,
                   total_lens: Optional[torch.Tensor] = None,
                   repetition_penalty: Optional[torch.Tensor] = None,
                   frequency_penalty: Optional[torch.Tensor] = None,
                   presence_penalty: Optional[torch.Tensor] = None,
                   bias_ids: Optional[torch.Tensor] = None,
                   bias_values: Optional[torch.Tensor] = None,
                   allowed_mask: Optional[torch.Tensor] = None,
                   temperature: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalised, biased and masked logits ``[B, V]``, float32 (or into ``out``).

    logits: ``[B, V]`` bfloat16, float16 or float32 with contiguous rows.  ``token_ids``:
    int32 ``[B, L]``, each row's prompt then output tokens, of which the first
    ``total_lens[b]`` count and the first ``prompt_lens[b]`` (default 0) are the prompt.
    The penalties and the temperature: float32 ``[B]``.  ``bias_ids`` int32 / ``bias_values``
    float32 ``[B, N]``: entries added to the row's logits, negative ids are padding, an id
    given twice adds twice.  ``allowed_mask``: int32 ``[B, >= ceil(V / 32)]``, bit ``v % 32`` of
    word ``v // 32`` set where token v is allowed; a row that allows nothing is all -inf.
    Every part is optional.  Ids outside the vocabulary are ignored.  ``out``: float32 or
    the logits' dtype; ``out=logits`` works in place, an ``out`` that overlaps them otherwise is
    refused.
    """
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a torch.Tensor")
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _LOGIT_DTYPES:
        raise RuntimeError("logits must be a [B, V] bfloat16, float16 or float32 tensor on CUDA, "
                           f"got {logits.dim()}-D {logits.dtype} on {logits.device}")
    B, V = logits.shape
    dev = logits.device
    if V < 1 or (logits.stride(1) != 1 and V > 1):
        raise RuntimeError("logits must have contiguous, non-empty rows")
    if out is None:
        out = _allocator(dev)((B, V), (V, 1), torch.float32)
    elif out.shape != logits.shape or out.device != dev or (out.stride(1) != 1 and V > 1) \
            or out.dtype not in (torch.float32, logits.dtype):
        raise RuntimeError("out must be float32 or the logits' dtype, of their shape and device, "
                           "with contiguous rows")
    f32 = torch.float32
    rep = _per_row("repetition_penalty", repetition_penalty, B, dev, f32)
    freq = _per_row("frequency_penalty", frequency_penalty, B, dev, f32)
    pres = _per_row("presence_penalty", presence_penalty, B, dev, f32)
    temp = _per_row("temperature", temperature, B, dev, f32)
    L = history_stride = 0
    if token_ids is not None:
        _check_int32("token_ids", token_ids, 2, dev)
        rows, L = token_ids.shape
        if rows != B or total_lens is None:
            raise RuntimeError(f"token_ids must be [{B}, L] with total_lens")
        history_stride = token_ids.stride()[0] if B > 1 else L
        if history_stride < L:
            raise RuntimeError("token_ids rows must not overlap")
    elif prompt_lens is not None or total_lens is not None or rep or freq or pres:
        raise RuntimeError("lengths and penalties need token_ids")
    prompt = _per_row("prompt_lens", prompt_lens, B, dev, torch.int32)
    total = _per_row("total_lens", total_lens, B, dev, torch.int32)
    N = 0
    if (bias_ids is None) != (bias_values is None):
        raise RuntimeError("bias_ids and bias_values come together")
    if bias_ids is not None:
        _check_int32("bias_ids", bias_ids, 2, dev)
        if bias_ids.shape[0] != B or not bias_ids.is_contiguous() or not isinstance(
                bias_values, torch.Tensor) or bias_values.dtype != torch.float32 \
                or bias_values.shape != bias_ids.shape or bias_values.device != dev \
                or not bias_values.is_contiguous():
            raise RuntimeError(f"bias_ids (int32) and bias_values (float32) must be contiguous [{B}, N]")
        N = bias_ids.shape[1]
    mask_stride = 0
    if allowed_mask is not None:
        _check_int32("allowed_mask", allowed_mask, 2, dev)
        words = (V + 31) // 32
        rows, width = allowed_mask.shape
        if rows != B or width < words:
            raise RuntimeError(f"allowed_mask must be [{B}, >= {words}]")
        mask_stride = allowed_mask.stride()[0] if B > 1 else width
        if mask_stride < words:
            raise RuntimeError("allowed_mask rows must not overlap")
    if B == 0:
        return out
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    ls, os_ = (logits.stride()[0], out.stride()[0]) if B > 1 else (V, V)
    if ls < V or os_ < V:
        raise RuntimeError("rows of logits and out must not overlap")
    p = _lib.pack_logits(
        _LOGIT_DTYPES[logits.dtype], _LOGIT_DTYPES[out.dtype], B, V, L, N, logits.data_ptr(),
        out.data_ptr(), ls, os_, ptr(token_ids), history_stride, prompt, total, rep, freq, pres,
        temp, ptr(bias_ids), ptr(bias_values), ptr(allowed_mask), mask_stride)
    _launch(_lib.load().kvb_process_logits, p, dev, "kvb_process_logits")
    return out
