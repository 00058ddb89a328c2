"""The vocabulary head in 8-bit integers: hidden states quantised per token, a weight quantised per
vocabulary row, products on the int8 tensor cores.

    codes, scale = quantize_int8(weight)                               once
    logits = int8_linear(hidden, codes, scale)                         serving: logits for the sampler
    ce, entropy, log_probs = int8_ce_entropy(hidden, codes, scale, target)
                                                                       scoring: no logits in HBM

Quantisation is symmetric: scale_r = max |x_r| / 127 (fp32), code = the integer nearest to x / scale_r.
The sums of code products are exact (int32); scales and bias are applied in fp32 and each output is
rounded once. Nothing here is differentiable: the results carry no gradient, and inputs that require one
(while gradients are enabled) or have a forward-mode tangent are refused.

No counterpart in the reference, whose head is bf16 / fp16 / fp32 (fast_reduction/gemm_kernel.py:276-356);
int8_ce_entropy returns what its gemm_fused_ce_entropy does.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _native as nat
from . import gemm_kernel as gk
from . import ops

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _codes_like(rows: int, cols: int, device: torch.device) -> Tensor:
    """Uninitialised [rows, cols] int8 codes whose rows start on 16-byte boundaries."""
    return torch.empty(rows, ops.round_up(max(cols, 1), 16), device=device, dtype=torch.int8)[:, :cols]


def _aligned_codes(codes: Tensor) -> Tensor:
    """`codes` itself when its rows start on 16-byte boundaries, else a copy laid out that way."""
    row, unit = codes.stride()
    if unit == 1 and not row & 15 and row >= codes.shape[1] and not codes.data_ptr() & 15:
        return codes
    out = _codes_like(codes.shape[0], codes.shape[1], codes.device)
    out.copy_(codes)
    return out


def _rows_2d(x: Tensor) -> Tensor:
    """x as a matrix of its rows, with unit column stride and rows that do not overlap."""
    if x.dim() != 2:
        x = x.reshape(x.shape[:-1].numel(), x.shape[-1])
    row, unit = x.stride()
    return x if unit == 1 and row >= x.shape[1] else x.contiguous()


def quantize_int8(x: Tensor) -> Tuple[Tensor, Tensor]:
    """8-bit codes of the rows of ``x`` [..., K] (bf16, fp16 or fp32): (codes int8 [..., K], scale fp32 [...])
    with x ~ codes * scale[..., None]. scale = max |row| / 127; each code is the integer nearest to x / scale,
    ties to even. A row with a NaN or an infinity gets scale NaN and codes 0 (what is computed from it is
    NaN); a row whose scale would be below 2^-120 gets scale 0 and codes 0.

    For 2-D ``x`` the codes are a view of rows padded to a multiple of 16 bytes, the layout int8_linear
    reads in place."""
    if x.dtype not in _FLOATS:
        raise TypeError(f"quantize_int8 takes bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("quantize_int8 needs at least one dimension")
    ops.refuse_grad("quantize_int8", x)
    ops._require_cuda(x)
    rows = _rows_2d(x) if x.numel() else x.new_empty(x.shape[:-1].numel(), x.shape[-1])
    codes = _codes_like(rows.shape[0], rows.shape[1], x.device)
    scale = torch.empty(rows.shape[0], device=x.device, dtype=torch.float32)
    ops.quantize_i8(rows, codes, scale)
    return codes if x.dim() == 2 else codes.reshape(x.shape), scale.view(x.shape[:-1])


def _prepare(hidden: Tensor, weight_codes: Tensor, weight_scale: Tensor, bias: Optional[Tensor],
             hidden_scale: Optional[Tensor]):
    """Operands as the kernels read them, (hidden [M, H], hidden scale [M] or None, weight codes, weight scale, bias);
    what does not concern the layout is checked at the launch (ops)."""
    shape = weight_codes.shape
    if len(shape) != 2 or weight_codes.dtype is not torch.int8:
        raise TypeError(f"weight_codes must be int8 [V, H], got {weight_codes.dtype} {tuple(weight_codes.shape)}")
    V, H = shape
    if V < 1 or H < 1:
        raise ValueError(f"weight_codes must not be empty, got {tuple(weight_codes.shape)}")
    if H > nat.FRX_I8_MAX_K:
        raise NotImplementedError(f"hidden size {H} > {nat.FRX_I8_MAX_K} could overflow the int32 sums")
    shape = hidden.shape
    if not shape or shape[-1] != H:
        raise ValueError(f"hidden size mismatch: hidden {tuple(hidden.shape)} vs weight_codes {tuple(weight_codes.shape)}")
    ops.refuse_grad("the int8 head", hidden, weight_scale, bias, hidden_scale)
    if hidden_scale is not None:
        if hidden_scale.shape != shape[:-1] or hidden.dtype is not torch.int8:
            raise ValueError(f"hidden_scale goes with int8 tokens, float32 {tuple(shape[:-1])}; got {hidden_scale.dtype} "
                             f"{tuple(hidden_scale.shape)}")
        hidden_scale = hidden_scale.reshape(-1).contiguous()
    x = _rows_2d(hidden)
    if hidden_scale is not None:
        x = _aligned_codes(x)
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    return x, hidden_scale, _aligned_codes(weight_codes), weight_scale.contiguous(), bias


def int8_linear(
    hidden: Tensor,
    weight_codes: Tensor,
    weight_scale: Tensor,
    bias: Optional[Tensor] = None,
    *,
    hidden_scale: Optional[Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
    out: Optional[Tensor] = None,
) -> Tensor:
    """Logits [..., V] = hidden @ dequantised(weight).T (+ bias) with hidden quantised per token.

    hidden        [..., H] bf16 / fp16 / fp32 (quantised here), or int8 codes with ``hidden_scale`` [...]
    weight_codes  [V, H] int8 and weight_scale [V] fp32, e.g. from quantize_int8(weight). Codes whose rows do
                  not start on 16-byte boundaries are copied on every call; quantize_int8 lays them out so
    bias          optional [V] bf16 / fp16 / fp32
    out_dtype     bf16, fp16 or fp32; default: hidden's type, bf16 for int8 hidden
    out           optional [rows, V] output (any row stride, unit column stride), instead of a new tensor
    """
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else (torch.bfloat16 if hidden.dtype == torch.int8 else hidden.dtype)
    if out_dtype not in _FLOATS:
        raise TypeError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    if out is not None:
        ops.refuse_grad("int8_linear", out)
        rows, V = hidden.shape[:-1].numel(), weight_codes.shape[0]
        if out.dtype != out_dtype or out.shape != (rows, V) or (V > 1 and out.stride(1) != 1) \
                or (rows > 1 and out.stride(0) < V):
            raise ValueError(f"out must be {out_dtype} [{rows}, {V}] with unit column stride and rows that do not "
                             f"overlap, got {out.dtype} {tuple(out.shape)} stride {out.stride()}")
    x, x_scale, w, w_scale, bias = _prepare(hidden, weight_codes, weight_scale, bias, hidden_scale)
    rows, V = x.shape[0], w.shape[0]
    y = torch.empty(rows, V, device=x.device, dtype=out_dtype) if out is None else out
    workspace = None if x_scale is not None else torch.empty(ops.i8_workspace_bytes(x), device=x.device,
                                                             dtype=torch.uint8)
    ops.gemm_i8(x, x_scale, w, w_scale, y, workspace, bias=bias)
    return y if out is not None or hidden.dim() == 2 else y.view(*hidden.shape[:-1], V)


def int8_ce_entropy(
    hidden: Tensor,
    weight_codes: Tensor,
    weight_scale: Tensor,
    target: Tensor,
    bias: Optional[Tensor] = None,
    chunk_size: int = 4096,
    ignore_index: int = gk.IGNORE_INDEX,
    *,
    hidden_scale: Optional[Tensor] = None,
) -> Tuple[Tensor, Tensor, Tensor]:
    """(ce_loss, entropy, log_probs), each fp32 and shaped like ``hidden.shape[:-1]``, of the logits
    int8_linear would give in fp32 (but for the order of the two scales' products, a step or two of fp32), which never
    reach HBM. Operands as in int8_linear; target, chunk_size and
    ignore_index as in gemm_fused_ce_entropy (ignored rows: ce = log_probs = 0, entropy kept; a target
    outside [0, V) gives NaN and sets FRX_STATUS_BAD_TARGET). A bias of -inf masks its vocabulary entry,
    as do all logits below -1e38; others are expected below 1e38, also before ``hidden_scale`` is multiplied in."""
    x, x_scale, w, w_scale, bias = _prepare(hidden, weight_codes, weight_scale, bias, hidden_scale)
    B = x.shape[0]
    if target.numel() != B:
        raise ValueError(f"target has {target.numel()} elements, expected {B}")
    if target.dtype != torch.int64:
        if target.dtype.is_floating_point or target.dtype.is_complex or target.dtype == torch.bool:
            raise TypeError(f"target must be an integer tensor, got {target.dtype}")
        target = target.to(torch.int64)
    target = target.contiguous()
    chunk = gk._chunk_rows(chunk_size, B)
    dev = x.device
    # three tensors: views of one would share a version counter, and each would keep the memory of all
    ce = torch.empty(B, device=dev, dtype=torch.float32)
    ent, logp = torch.empty_like(ce), torch.empty_like(ce)
    if B:
        V = w.shape[0]
        if B <= nat.FRX_I8_FEW_ROWS:
            partials = (V + 127) // 128 * B
        else:
            tiles = ops.n_vocab_tiles(V)
            chunk = gk._launch_rows(chunk, B, tiles)
            partials = tiles * chunk
        workspace = torch.empty(ops.i8_workspace_bytes(x) + 16 * partials, device=dev, dtype=torch.uint8)
        ops.i8_ce_entropy(x, x_scale, w, w_scale, target, ce, ent, logp, workspace, launch_rows=chunk,
                          ignore_index=ignore_index, bias=bias)
    if hidden.dim() == 2:
        return ce, ent, logp
    shape = hidden.shape[:-1]
    return ce.view(shape), ent.view(shape), logp.view(shape)
