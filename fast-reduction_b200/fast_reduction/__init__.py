"""fast_reduction (B200 engine): fused linear + cross-entropy + entropy on sm_100a.

Drop-in for the hot path of justinchiu/fast-reduction: the GEMM-epilogue forward and the
training megakernel of `fast_reduction.gemm_kernel`, exported lazily as in the reference
(fast_reduction/__init__.py:37-53). All device work runs in libfrx.so (hand-written CUDA for
sm_100a behind a C ABI, include/frx.h); there is no CPU or library fallback.
"""

__all__ = [
    "gemm_fused_ce_entropy",
    "gemm_fused_ce_entropy_v2",
    "gemm_fused_ce_entropy_differentiable",
    "gemm_fused_ce_entropy_fast",
    "gemm_megakernel_fast",
    "vocab_parallel_ce_entropy",
    "vocab_parallel_megakernel",
    "quantize_int8",
    "int8_linear",
    "int8_ce_entropy",
    "verify_drafts",
]

_GEMM_KERNEL_NAMES = {
    "gemm_fused_ce_entropy",
    "gemm_fused_ce_entropy_v2",
    "gemm_fused_ce_entropy_differentiable",
    "gemm_fused_ce_entropy_fast",
    "gemm_megakernel_fast",
}
_INT8_HEAD_NAMES = {"quantize_int8", "int8_linear", "int8_ce_entropy"}
_VOCAB_PARALLEL_NAMES = {"vocab_parallel_ce_entropy", "vocab_parallel_megakernel"}


def __getattr__(name):
    if name in _GEMM_KERNEL_NAMES:
        from fast_reduction import gemm_kernel

        return getattr(gemm_kernel, name)
    if name in _VOCAB_PARALLEL_NAMES:
        from fast_reduction import vocab_parallel

        return getattr(vocab_parallel, name)
    if name in _INT8_HEAD_NAMES:
        from fast_reduction import int8_head

        value = globals()[name] = getattr(int8_head, name)  # found directly from now on
        return value
    if name == "verify_drafts":
        from fast_reduction import draft_verify

        value = globals()[name] = draft_verify.verify_drafts
        return value
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
