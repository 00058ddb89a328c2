"""Tensor-level wrappers over the libfrx C ABI (one function per entry point).

These functions take torch tensors, validate them, and pass raw device pointers plus sizes
to libfrx on the tensors' current CUDA stream. Outputs are written into caller-provided
tensors, as in the reference's custom ops (`mutates_args`, e.g.
fast_reduction/gemm_ce_entropy_finalize.py:123-148, cute_dlogits.py:121-159).
"""

from __future__ import annotations

import contextlib
import os

import torch
from torch.autograd import forward_ad

from . import _native as nat

VOCAB_TILE = nat.FRX_VOCAB_TILE
# Never equal to a real target id: disables the ignore_index rule.
NO_IGNORE = -(2**63)

# Optional launch observer (used by bench.py to time each libfrx kernel with CUDA events on the
# launching stream): an object with before(name, device) / after(name, device), or None.
_observer = None


def set_launch_observer(observer):
    """Installs `observer` (or None) and returns the previous one."""
    global _observer
    prev, _observer = _observer, observer
    return prev


# NVTX ranges (visible in Nsight Systems / Nsight Compute timelines): one per libfrx launch, named
# "frx.<entry point>", inside the phase ranges of the Python layer. FRX_NVTX=0 turns them off.
_NVTX = os.environ.get("FRX_NVTX", "1") != "0"


def _nvtx_push(name: str) -> bool:
    if not _NVTX:
        return False
    try:
        torch.cuda.nvtx.range_push(name)
        return True
    except Exception:  # a torch build without NVTX
        return False


@contextlib.contextmanager
def phase(name: str):
    """NVTX range around one phase of the path (e.g. "frx.train.dhidden")."""
    pushed = _nvtx_push(name)
    try:
        yield
    finally:
        if pushed:
            torch.cuda.nvtx.range_pop()


def _launch(name: str, dev: torch.device, call) -> int:
    pushed = _nvtx_push("frx." + name)
    try:
        obs = _observer
        if obs is None:
            return call()
        obs.before(name, dev)
        rc = call()
        obs.after(name, dev)
        return rc
    finally:
        if pushed:
            torch.cuda.nvtx.range_pop()


def n_vocab_tiles(vocab_shard: int) -> int:
    return (vocab_shard + VOCAB_TILE - 1) // VOCAB_TILE


def round_up(x: int, m: int) -> int:
    return (x + m - 1) // m * m


# Operand types of the tcgen05 GEMMs (kind::f16: both operands bf16, or both fp16).
_GEMM_DTYPES = {torch.bfloat16: nat.FRX_DTYPE_BF16, torch.float16: nat.FRX_DTYPE_F16}
_OUT_DTYPES = {**_GEMM_DTYPES, torch.float32: nat.FRX_DTYPE_F32}


def _gemm_dtype(*tensors: torch.Tensor) -> int:
    """FRX dtype code shared by the GEMM operands; raises unless all are bf16 or all fp16."""
    dts = {t.dtype for t in tensors}
    if len(dts) != 1 or next(iter(dts)) not in _GEMM_DTYPES:
        raise TypeError(f"GEMM operands must all be bfloat16 or all float16, got {sorted(map(str, dts))}")
    return _GEMM_DTYPES[next(iter(dts))]


def _require_cuda(*tensors: torch.Tensor | None) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("fast_reduction (B200 engine) requires CUDA tensors; got a tensor on " + str(t.device))
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"all tensors must be on one device, got {dev} and {t.device}")
    return dev


def _row_major(t: torch.Tensor, name: str) -> int:
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be a 2-D tensor with unit column stride, got shape {tuple(t.shape)} "
                         f"stride {t.stride()}")
    return t.stride(0)


def fwd_partials(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    target: torch.Tensor | None,
    partials: torch.Tensor,
    tile_stride: int,
    vocab_offset: int = 0,
    logits: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    logits_rel: torch.Tensor | None = None,
) -> None:
    """partials[t, r] <- (m, s, u, zt) of z = hidden @ weight.T (+ bias) over vocab tile t (see include/frx.h).

    Optionally also writes every logit: fp32 ``logits`` (frx_fwd_partials), or fp16 ``logits_rel`` =
    z - m of the logit's tile (frx_fwd_partials_tilerel, half the bytes)."""
    dev = _require_cuda(hidden, weight, target, partials, logits, bias, logits_rel)
    ldh = _row_major(hidden, "hidden")
    ldw = _row_major(weight, "weight")
    rows, hdim = hidden.shape
    vshard = weight.shape[0]
    if weight.shape[1] != hdim:
        raise ValueError(f"hidden dim mismatch: hidden {tuple(hidden.shape)} vs weight {tuple(weight.shape)}")
    dt = _gemm_dtype(hidden, weight)
    if target is not None and (target.dtype != torch.int64 or not target.is_contiguous() or target.numel() < rows):
        raise ValueError("target must be a contiguous int64 tensor with one id per row")
    if partials.dtype != torch.float32 or not partials.is_contiguous():
        raise ValueError("partials must be contiguous float32")
    if tile_stride < rows or partials.numel() < 4 * ((n_vocab_tiles(vshard) - 1) * tile_stride + rows):
        raise ValueError("partials buffer too small")
    if bias is not None and (bias.dtype != hidden.dtype or not bias.is_contiguous() or bias.numel() != vshard):
        raise ValueError("bias must be a contiguous tensor of the weight's dtype with one value per vocabulary row "
                         "of the shard")
    ldl = 0
    if logits is not None:
        ldl = _row_major(logits, "logits")
        if logits.dtype != torch.float32 or logits.shape[0] < rows or logits.shape[1] < vshard:
            raise ValueError("logits must be float32 [rows, >= vocab_shard]")
    lib = nat.load()
    if logits_rel is not None:
        if logits is not None:
            raise ValueError("pass at most one of logits and logits_rel")
        ldr = _row_major(logits_rel, "logits_rel")
        if logits_rel.dtype != torch.float16 or logits_rel.shape[0] < rows or logits_rel.shape[1] < vshard:
            raise ValueError("logits_rel must be float16 [rows, >= vocab_shard]")
        rc = _launch("fwd_partials", dev, lambda: lib.frx_fwd_partials_tilerel(
            hidden.data_ptr(), ldh, weight.data_ptr(), ldw, dt, nat.ptr(bias), nat.ptr(target), rows, vshard, hdim,
            vocab_offset, partials.data_ptr(), tile_stride, logits_rel.data_ptr(), ldr,
            nat.status_word(dev).data_ptr(), nat.stream_of(dev),
        ))
        nat.check(rc, "frx_fwd_partials_tilerel")
        return
    rc = _launch("fwd_partials", dev, lambda: lib.frx_fwd_partials(
        hidden.data_ptr(), ldh, weight.data_ptr(), ldw, dt, nat.ptr(bias), nat.ptr(target), rows, vshard, hdim,
        vocab_offset,
        partials.data_ptr(), tile_stride, nat.ptr(logits), ldl, nat.status_word(dev).data_ptr(), nat.stream_of(dev),
    ))
    nat.check(rc, "frx_fwd_partials")


def finalize(
    partials: torch.Tensor,
    n_tiles: int,
    rows: int,
    tile_stride: int,
    *,
    ref_layout: bool = False,
    ignore_negative: bool = False,
    target: torch.Tensor | None = None,
    vocab_size: int = 0,
    ignore_index: int = NO_IGNORE,
    ce: torch.Tensor | None = None,
    entropy: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    log_probs: torch.Tensor | None = None,
    merged: torch.Tensor | None = None,
) -> None:
    """Merges [n_tiles, tile_stride] float4 partials into per-row outputs (any may be None)."""
    dev = _require_cuda(partials, target, ce, entropy, lse, log_probs, merged)
    if partials.dtype != torch.float32 or not partials.is_contiguous():
        raise ValueError("partials must be contiguous float32")
    if partials.numel() < 4 * n_tiles * tile_stride or tile_stride < rows:
        raise ValueError("partials buffer smaller than n_tiles * tile_stride float4")
    for name, t in (("ce", ce), ("entropy", entropy), ("lse", lse), ("log_probs", log_probs)):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.numel() < rows):
            raise ValueError(f"{name} must be contiguous float32 with >= rows elements")
    if merged is not None and (merged.dtype != torch.float32 or not merged.is_contiguous()
                               or merged.numel() < 4 * rows):
        raise ValueError("merged must be contiguous float32 [rows, 4]")
    if target is not None and (target.dtype != torch.int64 or not target.is_contiguous() or target.numel() < rows):
        raise ValueError("target must be a contiguous int64 tensor with one id per row")
    lib = nat.load()
    rc = _launch("finalize", dev, lambda: lib.frx_finalize(
        partials.data_ptr(), n_tiles, rows, tile_stride,
        (nat.FRX_PARTIALS_REF_LAYOUT if ref_layout else 0)
        | (nat.FRX_IGNORE_NEGATIVE_TARGETS if ignore_negative else 0),
        nat.ptr(target), vocab_size, ignore_index, nat.ptr(ce), nat.ptr(entropy), nat.ptr(lse), nat.ptr(log_probs),
        nat.ptr(merged), nat.status_word(dev).data_ptr(), nat.stream_of(dev),
    ))
    nat.check(rc, "frx_finalize")


def dlogits(
    logits: torch.Tensor,
    target: torch.Tensor | None,
    lse: torch.Tensor,
    entropy: torch.Tensor,
    out: torch.Tensor,
    *,
    rows: int,
    vocab_shard: int,
    g_ce: torch.Tensor | None = None,
    g_ent: torch.Tensor | None = None,
    ce_weight: float = 1.0,
    ent_weight: float = -1.0,
    vocab_offset: int = 0,
    ignore_index: int = NO_IGNORE,
) -> None:
    """out[r, j] <- d(sum g_ce*ce + g_ent*H)/dz[r, j] from fp32 logits (bf16, fp16 or fp32 out)."""
    dev = _require_cuda(logits, target, lse, entropy, out, g_ce, g_ent)
    ldl = _row_major(logits, "logits")
    ldo = _row_major(out, "dlogits")
    if logits.dtype != torch.float32:
        raise TypeError("logits must be float32")
    odt = _OUT_DTYPES.get(out.dtype)
    if odt is None:
        raise TypeError("dlogits output must be bfloat16, float16 or float32")
    if logits.shape[0] < rows or out.shape[0] < rows or logits.shape[1] < vocab_shard or out.shape[1] < vocab_shard:
        raise ValueError("logits/out smaller than [rows, vocab_shard]")
    for name, t in (("lse", lse), ("entropy", entropy), ("g_ce", g_ce), ("g_ent", g_ent)):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.numel() < rows):
            raise ValueError(f"{name} must be contiguous float32 with >= rows elements")
    if target is not None and (target.dtype != torch.int64 or not target.is_contiguous() or target.numel() < rows):
        raise ValueError("target must be a contiguous int64 tensor with one id per row")
    lib = nat.load()
    rc = _launch("dlogits", dev, lambda: lib.frx_dlogits(
        logits.data_ptr(), ldl, nat.ptr(target), lse.data_ptr(), entropy.data_ptr(), nat.ptr(g_ce), nat.ptr(g_ent),
        float(ce_weight), float(ent_weight), out.data_ptr(), ldo, odt, rows, vocab_shard, vocab_offset, ignore_index,
        nat.stream_of(dev),
    ))
    nat.check(rc, "frx_dlogits")


def dlogits_tilerel(
    logits_rel: torch.Tensor,
    partials: torch.Tensor,
    tile_stride: int,
    target: torch.Tensor | None,
    lse: torch.Tensor,
    entropy: torch.Tensor,
    out: torch.Tensor,
    *,
    rows: int,
    vocab_shard: int,
    g_ce: torch.Tensor | None = None,
    g_ent: torch.Tensor | None = None,
    ce_weight: float = 1.0,
    ent_weight: float = -1.0,
    vocab_offset: int = 0,
    ignore_index: int = NO_IGNORE,
) -> None:
    """dlogits (as `dlogits`) from fp16 tile-relative logits z - m_t and the partials holding each tile's
    maximum m_t (the outputs of one fwd_partials launch with logits_rel)."""
    dev = _require_cuda(logits_rel, partials, target, lse, entropy, out, g_ce, g_ent)
    ldl = _row_major(logits_rel, "logits_rel")
    ldo = _row_major(out, "dlogits")
    if logits_rel.dtype != torch.float16:
        raise TypeError("logits_rel must be float16")
    odt = _OUT_DTYPES.get(out.dtype)
    if odt is None:
        raise TypeError("dlogits output must be bfloat16, float16 or float32")
    if (logits_rel.shape[0] < rows or out.shape[0] < rows or logits_rel.shape[1] < vocab_shard
            or out.shape[1] < vocab_shard):
        raise ValueError("logits_rel/out smaller than [rows, vocab_shard]")
    if partials.dtype != torch.float32 or not partials.is_contiguous() or tile_stride < rows or \
            partials.numel() < 4 * ((n_vocab_tiles(vocab_shard) - 1) * tile_stride + rows):
        raise ValueError("partials must be contiguous float32 covering every tile of the launch")
    for name, t in (("lse", lse), ("entropy", entropy), ("g_ce", g_ce), ("g_ent", g_ent)):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.numel() < rows):
            raise ValueError(f"{name} must be contiguous float32 with >= rows elements")
    if target is not None and (target.dtype != torch.int64 or not target.is_contiguous() or target.numel() < rows):
        raise ValueError("target must be a contiguous int64 tensor with one id per row")
    lib = nat.load()
    rc = _launch("dlogits", dev, lambda: lib.frx_dlogits_tilerel(
        logits_rel.data_ptr(), ldl, partials.data_ptr(), tile_stride, nat.ptr(target), lse.data_ptr(),
        entropy.data_ptr(), nat.ptr(g_ce), nat.ptr(g_ent), float(ce_weight), float(ent_weight), out.data_ptr(), ldo,
        odt, rows, vocab_shard, vocab_offset, ignore_index, nat.stream_of(dev),
    ))
    nat.check(rc, "frx_dlogits_tilerel")


def _out_dtype(t: torch.Tensor, accumulate: bool = False) -> int:
    if t.dtype not in _OUT_DTYPES:
        raise TypeError("GEMM output must be bfloat16, float16 or float32")
    if accumulate:
        if t.dtype != torch.float32:
            raise TypeError("accumulating GEMM output must be float32")
        return _OUT_DTYPES[t.dtype] | nat.FRX_OUT_ACCUMULATE
    return _OUT_DTYPES[t.dtype]


# bf16x6 emulation of an fp32 product (Henry, Tang, Heinecke, ARITH 2019): the left operand's parts
# in this order times the right operand's parts in the other order sum to the product up to the
# mid*lo, lo*mid and lo*lo terms.
SPLIT_LEFT = (nat.FRX_PART_HI, nat.FRX_PART_HI, nat.FRX_PART_MID, nat.FRX_PART_HI, nat.FRX_PART_LO, nat.FRX_PART_MID)
SPLIT_RIGHT = (nat.FRX_PART_HI, nat.FRX_PART_MID, nat.FRX_PART_HI, nat.FRX_PART_LO, nat.FRX_PART_HI, nat.FRX_PART_MID)


def split_f32(x: torch.Tensor, out: torch.Tensor, parts, *, part_stride: int) -> None:
    """out (bf16, row stride out.stride(0)) + p * part_stride <- part parts[p] (hi / mid / lo) of the
    fp32 matrix x [rows, cols]: x = hi + mid + lo to ~24 bits (frx_split_f32)."""
    dev = _require_cuda(x, out)
    if x.dtype != torch.float32 or out.dtype != torch.bfloat16:
        raise TypeError("split_f32 takes a float32 matrix and writes bfloat16 parts")
    ldx = _row_major(x, "x")
    ldo = _row_major(out, "out")
    rows, cols = x.shape
    code = 0
    for p, sel in enumerate(parts):
        code |= int(sel) << (2 * p)
    lib = nat.load()
    rc = _launch("split_f32", dev, lambda: lib.frx_split_f32(
        x.data_ptr(), ldx, rows, cols, code, len(parts), out.data_ptr(), ldo, part_stride, nat.stream_of(dev)))
    nat.check(rc, "frx_split_f32")


def gemm_dhidden(dz: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, *, rows: int, vocab_shard: int,
                 accumulate: bool = False) -> None:
    """out[rows, H] <- dz[rows, vocab_shard] @ weight[vocab_shard, H] (``accumulate``: fp32 out +=)."""
    dev = _require_cuda(dz, weight, out)
    dt = _gemm_dtype(dz, weight)
    ldz = _row_major(dz, "dz")
    ldw = _row_major(weight, "weight")
    ldo = _row_major(out, "d_hidden")
    hdim = weight.shape[1]
    if out.shape[0] < rows or out.shape[1] < hdim or weight.shape[0] < vocab_shard or dz.shape[1] < vocab_shard:
        raise ValueError("shape mismatch in gemm_dhidden")
    lib = nat.load()
    rc = _launch("gemm_dhidden", dev, lambda: lib.frx_gemm_dhidden(
        dz.data_ptr(), ldz, weight.data_ptr(), ldw, dt, out.data_ptr(), ldo, _out_dtype(out, accumulate), rows, hdim,
        vocab_shard,
        nat.status_word(dev).data_ptr(), nat.stream_of(dev),
    ))
    nat.check(rc, "frx_gemm_dhidden")


def gemm_dweight(dz: torch.Tensor, hidden: torch.Tensor, out: torch.Tensor, *, rows: int, vocab_shard: int,
                 accumulate: bool = False, max_sms: int = 0) -> None:
    """out[vocab_shard, H] <- dz[rows, vocab_shard]^T @ hidden[rows, H] (``accumulate``: fp32 out +=), on at
    most ``max_sms`` SMs when it is positive (frx_gemm_dweight_sms)."""
    dev = _require_cuda(dz, hidden, out)
    dt = _gemm_dtype(dz, hidden)
    ldz = _row_major(dz, "dz")
    ldh = _row_major(hidden, "hidden")
    ldo = _row_major(out, "d_weight")
    hdim = hidden.shape[1]
    if out.shape[0] < vocab_shard or out.shape[1] < hdim or hidden.shape[0] < rows or dz.shape[0] < rows:
        raise ValueError("shape mismatch in gemm_dweight")
    lib = nat.load()
    if max_sms > 0:
        rc = _launch("gemm_dweight", dev, lambda: lib.frx_gemm_dweight_sms(
            dz.data_ptr(), ldz, hidden.data_ptr(), ldh, dt, out.data_ptr(), ldo, _out_dtype(out, accumulate),
            vocab_shard, hdim, rows, int(max_sms), nat.status_word(dev).data_ptr(), nat.stream_of(dev),
        ))
        nat.check(rc, "frx_gemm_dweight_sms")
        return
    rc = _launch("gemm_dweight", dev, lambda: lib.frx_gemm_dweight(
        dz.data_ptr(), ldz, hidden.data_ptr(), ldh, dt, out.data_ptr(), ldo, _out_dtype(out, accumulate), vocab_shard,
        hdim, rows,
        nat.status_word(dev).data_ptr(), nat.stream_of(dev),
    ))
    nat.check(rc, "frx_gemm_dweight")


_LOGITS_DTYPES = {torch.bfloat16: nat.FRX_DTYPE_BF16, torch.float16: nat.FRX_DTYPE_F16,
                  torch.float32: nat.FRX_DTYPE_F32}


def logits_partials(logits: torch.Tensor, target: torch.Tensor | None, partials: torch.Tensor, tile_cols: int,
                    tile_stride: int) -> None:
    """partials[t, r] <- (m, s, u, zt) of logits[r, t*tile_cols : (t+1)*tile_cols] (any float dtype)."""
    dev = _require_cuda(logits, target, partials)
    ld = _row_major(logits, "logits")
    if logits.dtype not in _LOGITS_DTYPES:
        raise TypeError(f"logits must be bfloat16, float16 or float32, got {logits.dtype}")
    rows, cols = logits.shape
    if target is not None and (target.dtype != torch.int64 or not target.is_contiguous() or target.numel() < rows):
        raise ValueError("target must be a contiguous int64 tensor with one id per row")
    n_tiles = (cols + tile_cols - 1) // tile_cols
    if partials.dtype != torch.float32 or not partials.is_contiguous() or partials.numel() < 4 * n_tiles * tile_stride:
        raise ValueError("partials must be contiguous float32 with n_tiles * tile_stride float4")
    lib = nat.load()
    rc = _launch("logits_partials", dev, lambda: lib.frx_logits_partials(
        logits.data_ptr(), _LOGITS_DTYPES[logits.dtype], ld, rows, cols, nat.ptr(target), tile_cols,
        partials.data_ptr(), tile_stride, nat.stream_of(dev),
    ))
    nat.check(rc, "frx_logits_partials")


def column_sums(x: torch.Tensor, out: torch.Tensor, *, rows: int, cols: int) -> None:
    """out[c] <- sum_r x[r, c] for a bf16 / fp16 [rows, >= cols] matrix, fp32 out (deterministic order)."""
    dev = _require_cuda(x, out)
    ld = _row_major(x, "x")
    if x.dtype not in _GEMM_DTYPES:
        raise TypeError("column_sums input must be bfloat16 or float16")
    if out.dtype != torch.float32 or not out.is_contiguous() or out.numel() < cols:
        raise ValueError("out must be contiguous float32 with >= cols elements")
    lib = nat.load()
    rc = _launch("column_sums", dev, lambda: lib.frx_column_sums(
        x.data_ptr(), _GEMM_DTYPES[x.dtype], ld, rows, cols, out.data_ptr(), nat.stream_of(dev)))
    nat.check(rc, "frx_column_sums")


def gemm_dhidden_multicast(dz: torch.Tensor, weight: torch.Tensor, mc_ptr: int, ld_out: int, *, rows: int,
                           vocab_shard: int, device: torch.device) -> None:
    """Adds dz[rows, vocab_shard] @ weight[vocab_shard, H] into the fp32 matrix behind the NVLS
    multicast address `mc_ptr` (row stride ld_out): the cross-rank d_hidden sum inside the GEMM."""
    dev = _require_cuda(dz, weight)
    dt = _gemm_dtype(dz, weight)
    if not mc_ptr:
        raise ValueError("a multicast address is required")
    ldz = _row_major(dz, "dz")
    ldw = _row_major(weight, "weight")
    hdim = weight.shape[1]
    lib = nat.load()
    rc = _launch("gemm_dhidden", dev, lambda: lib.frx_gemm_dhidden_multicast(
        dz.data_ptr(), ldz, weight.data_ptr(), ldw, dt, mc_ptr, ld_out, rows, hdim, vocab_shard,
        nat.status_word(dev).data_ptr(), nat.stream_of(dev),
    ))
    nat.check(rc, "frx_gemm_dhidden_multicast")


def loss_sum(ce: torch.Tensor | None, entropy: torch.Tensor | None, loss: torch.Tensor, *, rows: int,
             ce_weight: float, ent_weight: float) -> None:
    """loss (0-d fp32) <- ce_weight * sum(ce[:rows]) + ent_weight * sum(entropy[:rows]) (deterministic)."""
    dev = _require_cuda(ce, entropy, loss)
    for name, t in (("ce", ce), ("entropy", entropy)):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.numel() < rows):
            raise ValueError(f"{name} must be contiguous float32 with >= rows elements")
    if loss.dtype != torch.float32 or loss.numel() != 1:
        raise ValueError("loss must be a one-element float32 tensor")
    lib = nat.load()
    rc = _launch("loss_sum", dev, lambda: lib.frx_loss_sum(
        nat.ptr(ce), nat.ptr(entropy), rows, float(ce_weight), float(ent_weight), loss.data_ptr(), nat.stream_of(dev)))
    nat.check(rc, "frx_loss_sum")


def scale_inplace(x: torch.Tensor, scale: torch.Tensor) -> None:
    """x *= scale[0] on the device (a no-op kernel when the scale is exactly 1; no host synchronisation)."""
    dev = _require_cuda(x, scale)
    if not x.is_contiguous() or x.dtype not in _OUT_DTYPES:
        raise ValueError("x must be a contiguous bfloat16, float16 or float32 tensor")
    if scale.dtype != torch.float32 or scale.numel() != 1:
        raise ValueError("scale must be a one-element float32 tensor")
    lib = nat.load()
    rc = _launch("scale_inplace", dev, lambda: lib.frx_scale_inplace(
        x.data_ptr(), _OUT_DTYPES[x.dtype], x.numel(), scale.data_ptr(), nat.stream_of(dev)))
    nat.check(rc, "frx_scale_inplace")


_I8_X_DTYPES = {**_OUT_DTYPES, torch.int8: nat.FRX_DTYPE_I8}


def _call(name: str, entry: str, dev: torch.device, *args) -> None:
    """One libfrx call on the tensors' device, whatever the current one is, with its status word and stream last."""
    fn = getattr(nat.load(), entry)
    index = dev.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _call(name, entry, dev, *args)
    status, stream = nat.status_word(dev).data_ptr(), nat.stream_of(dev)
    if _observer is None and not _NVTX:
        rc = fn(*args, status, stream)
    else:
        rc = _launch(name, dev, lambda: fn(*args, status, stream))
    if rc:
        nat.check(rc, entry)


def _one_device(first: torch.Tensor, *rest: torch.Tensor | None) -> torch.device:
    """_require_cuda, with its loop left to the case that it refuses (a device's number is read in half the time of a
    torch.device; the CPU's is -1)."""
    index = first.get_device()
    if index >= 0:
        for t in rest:
            if t is not None and t.get_device() != index:
                break
        else:
            return first.device
    return _require_cuda(first, *rest)


def refuse_grad(what: str, *tensors: torch.Tensor | None) -> None:
    """Raises where a result without a gradient, or without a tangent, would silently end what one of the inputs takes
    part in: reverse mode (unless gradients are disabled) or forward mode (which torch.no_grad() leaves on)."""
    duals = forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()
    for t in tensors:
        if t is None:
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")
        if duals and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no gradient in forward mode either: call it on the primal")


def _is_vector(t: torch.Tensor, dtype: torch.dtype, n: int) -> bool:
    return t.dtype is dtype and t.dim() == 1 and t.numel() == n and t.is_contiguous()


def _leading(t: torch.Tensor, rows: int, cols: int, name: str) -> int:
    """Row stride of a [rows, cols] matrix for the C entry points. A dimension of one may come with any stride (torch calls that
    contiguous); otherwise columns lie next to each other and rows do not overlap."""
    ld, unit = t.stride()
    if (unit != 1 and cols > 1) or (ld < cols and rows > 1):
        raise ValueError(f"{name} must have unit column stride and rows that do not overlap, got shape {tuple(t.shape)} "
                         f"stride {t.stride()}")
    return ld if ld > cols else cols


def _room(workspace: torch.Tensor | None, dtype: torch.dtype) -> tuple[int | None, int]:
    """Address and number of elements of a workspace."""
    if workspace is None:
        return None, 0
    if workspace.dtype is not dtype or not workspace.is_contiguous():
        raise ValueError(f"the workspace must be contiguous {dtype}, got {workspace.dtype} stride {workspace.stride()}")
    return workspace.data_ptr(), workspace.numel()


def quantize_i8(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor) -> None:
    """codes (int8), scale (fp32 per row) <- symmetric 8-bit codes of the rows of x (frx_quantize_i8)."""
    dev = _require_cuda(x, codes, scale)
    if x.dtype not in _OUT_DTYPES or codes.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError("quantize_i8 takes a bfloat16, float16 or float32 matrix, int8 codes and float32 scales")
    if codes.shape != x.shape or scale.shape != x.shape[:1] or not scale.is_contiguous():
        raise ValueError("codes must have x's shape and scale one value per row")
    rows, cols = x.shape
    ldx, ldc = _leading(x, rows, cols, "x"), _leading(codes, rows, cols, "codes")
    lib = nat.load()
    with torch.cuda.device(dev):
        rc = _launch("quantize_i8", dev, lambda: lib.frx_quantize_i8(
            x.data_ptr(), _OUT_DTYPES[x.dtype], ldx, rows, cols, codes.data_ptr(), ldc, scale.data_ptr(),
            nat.stream_of(dev)))
    nat.check(rc, "frx_quantize_i8")


def i8_workspace_bytes(x: torch.Tensor) -> int:
    """Workspace of a product whose tokens are ``x`` [rows, k]: their codes and scales, unless they are codes."""
    rows, k = x.shape
    return 0 if x.dtype == torch.int8 else (rows * ((k + 15) // 16 * 16 + 4) + 15) // 16 * 16


def _i8_operands(x, x_scale, weight, weight_scale, bias, *others):
    """Checked operands of an 8-bit product: (device, rows, cols, k, the leading C arguments up to bias_dtype). ``others``
    need to be on the same device."""
    xdt = _I8_X_DTYPES.get(x.dtype)
    if xdt is None or weight.dtype is not torch.int8:
        raise TypeError(f"x must be int8, bfloat16, float16 or float32 and weight int8, got {x.dtype} and {weight.dtype}")
    rows, k = x.shape
    cols, wk = weight.shape
    if wk != k:
        raise ValueError(f"row length mismatch: x {tuple(x.shape)} vs weight {tuple(weight.shape)}")
    ldx, ldw = _leading(x, rows, k, "x"), _leading(weight, cols, k, "weight")
    if not _is_vector(weight_scale, torch.float32, cols):
        raise ValueError(f"weight_scale must be contiguous float32 [{cols}], got {weight_scale.dtype} "
                         f"{tuple(weight_scale.shape)}")
    sptr = None
    if x_scale is None:
        if xdt == nat.FRX_DTYPE_I8:
            raise ValueError("int8 tokens need their scales (hidden_scale)")
    elif xdt != nat.FRX_DTYPE_I8 or not _is_vector(x_scale, torch.float32, rows):
        raise ValueError(f"hidden_scale goes with int8 tokens, contiguous float32 [{rows}]")
    else:
        sptr = x_scale.data_ptr()
    bptr, bdt = None, 0
    if bias is not None:
        bdt = _OUT_DTYPES.get(bias.dtype)
        if bdt is None or not _is_vector(bias, bias.dtype, cols):
            raise ValueError(f"bias must be a contiguous bfloat16, float16 or float32 [{cols}], got {bias.dtype} "
                             f"{tuple(bias.shape)}")
        bptr = bias.data_ptr()
    dev = _one_device(x, x_scale, weight, weight_scale, bias, *others)
    return dev, rows, cols, k, (x.data_ptr(), xdt, ldx, sptr, weight.data_ptr(), ldw, weight_scale.data_ptr(), bptr, bdt)


def gemm_i8(x: torch.Tensor, x_scale: torch.Tensor | None, weight: torch.Tensor, weight_scale: torch.Tensor,
            out: torch.Tensor, workspace: torch.Tensor | None, *, bias: torch.Tensor | None = None) -> None:
    """out[r, j] <- (xc[r] . weight[j]) * x_scale[r] * weight_scale[j] (+ bias[j]): xc = x for int8 x, else its codes,
    which go into the uint8 ``workspace`` (frx_gemm_i8)."""
    dev, rows, cols, k, operands = _i8_operands(x, x_scale, weight, weight_scale, bias, out, workspace)
    odt = _OUT_DTYPES.get(out.dtype)
    if odt is None or out.shape != (rows, cols):
        raise ValueError(f"out must be bfloat16, float16 or float32 [{rows}, {cols}], got {out.dtype} {tuple(out.shape)}")
    _call("gemm_i8", "frx_gemm_i8", dev, *operands, rows, cols, k, *_room(workspace, torch.uint8), out.data_ptr(),
          _leading(out, rows, cols, "out"), odt)


def i8_ce_entropy(x: torch.Tensor, x_scale: torch.Tensor | None, weight: torch.Tensor, weight_scale: torch.Tensor,
                  target: torch.Tensor, ce: torch.Tensor, entropy: torch.Tensor, log_probs: torch.Tensor,
                  workspace: torch.Tensor, *, launch_rows: int, ignore_index: int,
                  bias: torch.Tensor | None = None) -> None:
    """ce, entropy, log_probs <- those of gemm_i8's fp32 logits, launch_rows rows at a time (frx_i8_ce_entropy)."""
    dev, rows, cols, k, operands = _i8_operands(x, x_scale, weight, weight_scale, bias, target, ce, entropy, log_probs,
                                                workspace)
    if target.dtype != torch.int64 or not target.is_contiguous() or target.numel() != rows:
        raise ValueError("target must be a contiguous int64 tensor with one id per row")
    for t in (ce, entropy, log_probs):
        if t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != rows:
            raise ValueError("ce, entropy and log_probs must be contiguous float32 with one value per row")
    _call("i8_ce_entropy", "frx_i8_ce_entropy", dev, *operands, target.data_ptr(), rows, cols, k, ignore_index,
          launch_rows, *_room(workspace, torch.uint8), ce.data_ptr(), entropy.data_ptr(), None, log_probs.data_ptr())


def verify_drafts(logits: torch.Tensor, drafts: torch.Tensor, cu_drafts: torch.Tensor, uniforms: torch.Tensor,
                  final_uniforms: torch.Tensor, draft_probs: torch.Tensor | None, temperature: torch.Tensor | None,
                  temperature_all: float, workspace: torch.Tensor, accepted: torch.Tensor, tokens: torch.Tensor,
                  log_probs: torch.Tensor) -> None:
    """accepted, tokens, log_probs <- the outcome of drafted tokens against target logits (frx_verify_drafts)."""
    n, batch = drafts.numel(), cu_drafts.numel() - 1
    dt = _LOGITS_DTYPES.get(logits.dtype)
    rows, vocab = logits.shape
    if dt is None or rows != n + batch:
        raise ValueError(f"logits must be bfloat16, float16 or float32 [{n + batch}, V], got {logits.dtype} "
                         f"{tuple(logits.shape)}")
    ldl = _leading(logits, rows, vocab, "logits")
    qptr, qdt, ldq = None, 0, 0
    if draft_probs is not None:
        qdt = _LOGITS_DTYPES.get(draft_probs.dtype)
        if qdt is None or draft_probs.shape != (n, vocab):
            raise ValueError(f"draft_probs must be bfloat16, float16 or float32 [{n}, {vocab}], got {draft_probs.dtype} "
                             f"{tuple(draft_probs.shape)}")
        qptr, ldq = draft_probs.data_ptr(), _leading(draft_probs, n, vocab, "draft_probs")
    if not _is_vector(drafts, torch.int64, n) or not _is_vector(cu_drafts, torch.int64, batch + 1):
        raise ValueError("drafts and cu_drafts must be contiguous int64 vectors")
    if not _is_vector(uniforms, torch.float32, n):
        raise ValueError(f"uniforms must be contiguous float32 [{n}], got {uniforms.dtype} {tuple(uniforms.shape)}")
    if not _is_vector(final_uniforms, torch.float32, batch):
        raise ValueError(f"final_uniforms must be contiguous float32 [{batch}], got {final_uniforms.dtype} "
                         f"{tuple(final_uniforms.shape)}")
    tptr = None
    if temperature is not None:
        if not _is_vector(temperature, torch.float32, batch):
            raise ValueError(f"temperature must be contiguous float32 [{batch}], got {temperature.dtype} "
                             f"{tuple(temperature.shape)}")
        tptr = temperature.data_ptr()
    if not (_is_vector(accepted, torch.int64, batch) and _is_vector(tokens, torch.int64, rows)
            and _is_vector(log_probs, torch.float32, rows)):
        raise ValueError(f"outputs must be contiguous: int64 accepted [{batch}], int64 tokens and float32 log_probs "
                         f"[{rows}]")
    dev = _one_device(logits, drafts, cu_drafts, uniforms, final_uniforms, draft_probs, temperature, workspace, accepted,
                      tokens, log_probs)
    _call("verify_drafts", "frx_verify_drafts", dev, logits.data_ptr(), dt, ldl, drafts.data_ptr(), cu_drafts.data_ptr(),
          uniforms.data_ptr(), final_uniforms.data_ptr(), qptr, qdt, ldq, tptr, temperature_all, batch, n, vocab,
          *_room(workspace, torch.float32), accepted.data_ptr(), tokens.data_ptr(), log_probs.data_ptr())
