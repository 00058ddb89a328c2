"""Verification of drafted tokens against the target model's logits (speculative sampling: Leviathan, Kalman,
Matias 2023; Chen et al. 2023), from random numbers the caller gives, so a step is reproducible and can be
captured in a CUDA graph. The logits come from int8_linear or any other head.

No counterpart in the reference; it stands beside the reductions over given logits of
fast_reduction/cute_cross_entropy.py:583-735.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _native as nat
from . import ops

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _ids(t: Tensor, name: str) -> Tensor:
    if t.dim() != 1:
        raise ValueError(f"{name} must be 1-D, got shape {tuple(t.shape)}")
    if t.dtype != torch.int64:
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
        t = t.to(torch.int64)
    return t.contiguous()


def _rows(t: Tensor, name: str) -> Tensor:
    if t.dtype not in _FLOATS:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def verify_drafts(
    target_logits: Tensor,
    draft_tokens: Tensor,
    cu_drafts: Tensor,
    uniforms: Tensor,
    final_uniforms: Tensor,
    draft_probs: Optional[Tensor] = None,
    temperature: Union[float, Tensor] = 1.0,
) -> Tuple[Tensor, Tensor, Tensor]:
    """Which drafted tokens stand, and the token each sequence emits after them.

    Sequence b of B has drafts draft_tokens[cu_drafts[b]:cu_drafts[b + 1]] (n of them, possibly none) and the
    n + 1 logits rows from row cu_drafts[b] + b: row i is the target's distribution for the token at place i.
    With p_i = softmax(row i / temperature), draft i is accepted while
        uniforms[draft] * draft_probs[draft, token] < p_i(token)
    (without draft_probs: uniforms[draft] < p_i(token), for drafts that were looked up or chosen greedily). The
    next token is drawn from max(p - q, 0) at the first rejected draft's row (without draft_probs: from p with
    the rejected token taken out; from p when nothing is left), or from the last row's p: the first j whose
    running sum of weights passes final_uniforms[b] times their total.

    target_logits   [N + B, V] bf16 / fp16 / fp32; NaN counts as -inf, +inf as the largest finite
                    value (of fp32 for fp32 logits, of bf16 for 16-bit ones)
    draft_tokens    [N] int32 / int64; an id outside [0, V) is rejected and sets FRX_STATUS_BAD_TARGET
    cu_drafts       [B + 1] int32 / int64 on the GPU, from 0, non-decreasing; its last entry may be below N (a
                    padded batch: rows behind the last sequence's are not read)
    uniforms        [N] fp32 in [0, 1), final_uniforms [B] fp32 in [0, 1)
    draft_probs     optional [N, V] bf16 / fp16 / fp32
    temperature     a number or fp32 [B]; below 1e-6 is greedy (accepted while equal to the argmax, lowest
                    index of a tie; the argmax is emitted)

    Returns (accepted int64 [B], tokens int64 [N + B], log_probs fp32 [N + B]): at the logits rows, the tokens
    emitted there and their log p_i (greedy: at temperature 1); -1 and 0 where nothing is emitted. A row that
    leaves nothing to draw emits -1 with log-probability -inf. Decisions are taken in 64 bits (in a draw, p below e^-680 of
    the row's largest counts as 0); log_probs come from sums in fp32. No host synchronisation. Nothing here is
    differentiable: logits or draft_probs that require a gradient (while gradients are enabled) or have a forward-mode
    tangent are refused."""
    drafts, cu = _ids(draft_tokens, "draft_tokens"), _ids(cu_drafts, "cu_drafts")
    n, batch = drafts.numel(), cu.numel() - 1
    if batch < 0:
        raise ValueError("cu_drafts must hold at least one offset")
    ops.refuse_grad("verify_drafts", target_logits, draft_probs)
    logits = _rows(target_logits, "target_logits")
    rows, vocab = logits.shape
    if rows != n + batch or vocab < 1 or (batch == 0 and n):
        raise ValueError(f"target_logits must have at least one column and a row for each of {n} drafts and {batch} "
                         f"sequences, got {tuple(logits.shape)}")
    if draft_probs is not None:
        draft_probs = _rows(draft_probs, "draft_probs")
    temps = None
    if isinstance(temperature, Tensor):
        temps, temperature = temperature.contiguous(), 1.0
    dev = logits.device
    accepted = torch.empty(batch, device=dev, dtype=torch.int64)
    tokens = torch.empty(rows, device=dev, dtype=torch.int64)
    log_probs = torch.empty(rows, device=dev, dtype=torch.float32)
    workspace = torch.empty(4 * rows * ((vocab + 6) // nat.FRX_VERIFY_CHUNK + 1), device=dev, dtype=torch.float32)
    ops.verify_drafts(logits, drafts, cu, uniforms.contiguous(), final_uniforms.contiguous(), draft_probs, temps,
                      float(temperature), workspace, accepted, tokens, log_probs)
    return accepted, tokens, log_probs
