"""CPU: the 8-bit head and the draft verification refuse bad arguments before any GPU work, in Python and at the
C entry points (which read nothing through the pointers they are given here)."""

import pytest
import torch

A, B, C, D = 1 << 20, 1 << 21, 1 << 22, 1 << 23  # aligned addresses that are never read


def _lib():
    from fast_reduction import _native as nat

    return nat, nat.load()


def test_quantize_entry_point():
    nat, lib = _lib()
    assert lib.frx_quantize_i8(A, 0, 8, -1, 8, B, 16, C, None) == nat.FRX_ERR_INVALID_ARG
    assert lib.frx_quantize_i8(A, 0, 7, 2, 8, B, 16, C, None) == nat.FRX_ERR_INVALID_ARG  # ld_x < cols
    assert lib.frx_quantize_i8(A, 0, 8, 2, 8, B, 7, C, None) == nat.FRX_ERR_INVALID_ARG
    assert lib.frx_quantize_i8(A, 5, 8, 2, 8, B, 16, C, None) == nat.FRX_ERR_INVALID_ARG  # dtype
    assert lib.frx_quantize_i8(A, 0, 8, 2, 8, None, 16, C, None) == nat.FRX_ERR_INVALID_ARG
    assert lib.frx_quantize_i8(A, 0, 8, 2, 8, B, 16, None, None) == nat.FRX_ERR_INVALID_ARG
    assert lib.frx_quantize_i8(None, 0, 8, 0, 8, None, 16, None, None) == nat.FRX_OK


@pytest.mark.parametrize("score", [False, True])
def test_product_entry_points(score):
    nat, lib = _lib()

    def call(x=A, xdt=nat.FRX_DTYPE_I8, ld_x=64, xs=B, w=C, ld_w=64, ws=D, bias=None, bdt=0, rows=4, cols=8, k=64,
             out=A, ld=8, odt=0, work=B, nbytes=1 << 20, target=A, step=4):
        if score:
            return lib.frx_i8_ce_entropy(x, xdt, ld_x, xs, w, ld_w, ws, bias, bdt, target, rows, cols, k, -100, step,
                                         work, nbytes, A, A, None, A, None, None)
        return lib.frx_gemm_i8(x, xdt, ld_x, xs, w, ld_w, ws, bias, bdt, rows, cols, k, work, nbytes, out, ld, odt,
                               None, None)

    bad = nat.FRX_ERR_INVALID_ARG
    assert call(rows=-1) == bad and call(cols=0) == bad and call(k=0) == bad and call(rows=1 << 31) == bad
    assert call(k=131072, ld_x=131072, ld_w=131072) == nat.FRX_ERR_UNSUPPORTED
    assert call(x=None) == bad and call(xs=None) == bad and call(w=None) == bad and call(ws=None) == bad
    assert call(x=A + 8) == bad and call(w=C + 1) == bad and call(ld_x=72) == bad and call(ld_w=48) == bad
    assert call(xdt=4) == bad and call(bias=A, bdt=7) == bad and call(bias=A, bdt=nat.FRX_DTYPE_I8) == bad
    # floating-point tokens need room for their codes (64 bytes a row here) and scales
    need = 4 * (64 + 4) + (16 * 4 if score else 0)
    assert call(xdt=0, nbytes=need - 1) == bad and b"workspace" in lib.frx_last_error()
    assert call(xdt=0, work=None) == bad and call(xdt=0, work=B + 8) == bad and call(xdt=0, ld_x=63) == bad
    assert call(rows=0) == nat.FRX_OK
    if score:
        assert call(target=None) == bad and call(step=0) == bad
        assert call(nbytes=16 * 4 - 1) == bad
    else:
        assert call(out=None) == bad and call(ld=7) == bad and call(odt=9) == bad


def test_verify_entry_point():
    nat, lib = _lib()

    def call(logits=A, dt=0, ld=100, drafts=B, cu=B, u=B, r=B, q=None, qdt=1, ldq=0, batch=2, n=3, v=100, ws=C,
             floats=20, acc=D, tok=D, lp=D):
        return lib.frx_verify_drafts(logits, dt, ld, drafts, cu, u, r, q, qdt, ldq, None, 1.0, batch, n, v, ws, floats,
                                     acc, tok, lp, None, None)

    bad = nat.FRX_ERR_INVALID_ARG
    assert call(batch=-1) == bad and call(n=-1) == bad and call(v=0) == bad and call(ld=99) == bad
    assert call(dt=4) == bad and call(q=A, qdt=8, ldq=100) == bad and call(q=A, ldq=99) == bad
    for name in ("logits", "drafts", "cu", "u", "r", "ws", "acc", "tok", "lp"):
        assert call(**{name: None}) == bad, name
    assert call(floats=19) == bad and b"workspace" in lib.frx_last_error()
    assert call(ws=C + 4) == bad
    assert call(batch=0) == bad  # drafts of no sequence
    assert call(batch=0, n=0) == nat.FRX_OK


def test_int8_head_refusals():
    from fast_reduction import int8_ce_entropy, int8_linear, quantize_int8

    x, w, s = torch.zeros(4, 32), torch.zeros(10, 32, dtype=torch.int8), torch.ones(10)  # on the CPU
    t = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        quantize_int8(x)
    with pytest.raises(TypeError):
        quantize_int8(torch.zeros(3, 4, dtype=torch.int32))
    with pytest.raises(ValueError):
        quantize_int8(torch.zeros(()))
    for fn in (lambda *a, **k: int8_linear(*a, **k), lambda h, *a, **k: int8_ce_entropy(h, *a, t, **k)):
        with pytest.raises(ValueError, match="CUDA"):
            fn(x, w, s)
        with pytest.raises(TypeError):
            fn(x, w.float(), s)
        with pytest.raises(TypeError):
            fn(x.double(), w, s)
        with pytest.raises(ValueError, match="mismatch"):
            fn(x[:, :31], w, s)
        with pytest.raises(ValueError, match="weight_scale"):
            fn(x, w, s[:9])
        with pytest.raises(ValueError, match="weight_scale"):
            fn(x, w, s.half())
        with pytest.raises(ValueError, match="bias"):
            fn(x, w, s, bias=torch.zeros(9))
        with pytest.raises(ValueError, match="hidden_scale"):
            fn(x.to(torch.int8), w, s)
        with pytest.raises(ValueError, match="hidden_scale"):
            fn(x.to(torch.int8), w, s, hidden_scale=torch.ones(3))
        with pytest.raises(ValueError, match="hidden_scale"):
            fn(x, w, s, hidden_scale=torch.ones(4))
        with pytest.raises(NotImplementedError, match="overflow"):
            fn(torch.zeros(1, 131072), torch.zeros(2, 131072, dtype=torch.int8), s[:2])
        with pytest.raises(NotImplementedError, match="gradient"):
            fn(x.clone().requires_grad_(True), w, s)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            fn(x.clone().requires_grad_(True), w, s)
        with pytest.raises(ValueError, match="empty"):
            fn(torch.zeros(4, 0), w[:, :0], s)
    with pytest.raises(TypeError, match="out_dtype"):
        int8_linear(x, w, s, out_dtype=torch.float64)
    for out in (torch.zeros(4, 9), torch.zeros(10, 4).t(), torch.zeros(1, 10).expand(4, 10), torch.zeros(3, 10)):
        with pytest.raises(ValueError, match="out must"):
            int8_linear(x, w, s, out=out)
    with pytest.raises(NotImplementedError, match="gradient"):
        int8_linear(x, w, s, out=torch.zeros(4, 10, requires_grad=True))


def test_verify_refusals():
    from fast_reduction import verify_drafts

    z, d, cu = torch.zeros(5, 20), torch.zeros(3, dtype=torch.int64), torch.tensor([0, 1, 3])
    u, r, q = torch.zeros(3), torch.zeros(2), torch.full((3, 20), 0.05)

    def call(**kw):
        a = dict(target_logits=z, draft_tokens=d, cu_drafts=cu, uniforms=u, final_uniforms=r, draft_probs=q)
        a.update(kw)
        return verify_drafts(**a)

    with pytest.raises(ValueError, match="CUDA"):
        call()
    with pytest.raises(TypeError):
        call(draft_tokens=d.float())
    with pytest.raises(ValueError):
        call(draft_tokens=d[None])
    with pytest.raises(TypeError):
        call(cu_drafts=cu.float())
    with pytest.raises(ValueError, match="offset"):
        call(cu_drafts=cu[:0])
    with pytest.raises(ValueError, match="0 sequences"):
        call(cu_drafts=cu[:1])
    with pytest.raises(ValueError, match="target_logits"):
        call(target_logits=z[:4])
    with pytest.raises(TypeError, match="target_logits"):
        call(target_logits=z.double())
    with pytest.raises(ValueError, match="column"):
        call(target_logits=z[:, :0], draft_probs=None)
    with pytest.raises(NotImplementedError, match="gradient"):
        call(target_logits=z.clone().requires_grad_(True))
    with pytest.raises(NotImplementedError, match="gradient"):
        call(draft_probs=q.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="uniforms"):
        call(uniforms=u[:2])
    with pytest.raises(ValueError, match="final_uniforms"):
        call(final_uniforms=r.double())
    with pytest.raises(ValueError, match="draft_probs"):
        call(draft_probs=q[:, :19])
    with pytest.raises(ValueError, match="temperature"):
        call(temperature=torch.ones(3))


def test_tensor_level_calls_refuse_layouts_that_pass_their_memory():
    """Rows that overlap, spread columns and spread workspaces, which the C entry points cannot see."""
    from fast_reduction import ops

    x, w, s = torch.zeros(4, 32), torch.zeros(10, 32, dtype=torch.int8), torch.ones(10)
    t, out, work = torch.zeros(4, dtype=torch.int64), torch.zeros(4, 10), torch.zeros(4096, dtype=torch.uint8)
    r = [torch.zeros(4) for _ in range(3)]

    def score(x, w, work):
        ops.i8_ce_entropy(x, None, w, s, t, *r, work, launch_rows=4, ignore_index=-100)

    def spread(rows, dtype):
        return [m.to(dtype).as_strided(*at) for m, at in ((torch.zeros(1, 32), ((rows, 32), (0, 1))),
                                                          (torch.zeros(32, rows), ((rows, 32), (1, rows))),
                                                          (torch.zeros(rows, 64), ((rows, 32), (64, 2))))]

    for bad in spread(4, torch.float32):
        for fn in (lambda: ops.gemm_i8(bad, None, w, s, out, work), lambda: score(bad, w, work)):
            with pytest.raises(ValueError, match="x must have unit"):
                fn()
    for bad in spread(10, torch.int8):
        for fn in (lambda: ops.gemm_i8(x, None, bad, s, out, work), lambda: score(x, bad, work)):
            with pytest.raises(ValueError, match="weight must have unit"):
                fn()
    for fn in (lambda: ops.gemm_i8(x, None, w, s, out, work), lambda: score(x, w, work)):
        with pytest.raises(ValueError, match="CUDA"):
            fn()
    for bad in (torch.zeros(1, dtype=torch.uint8).expand(4096), work.view(torch.float32)):
        with pytest.raises(ValueError, match="workspace"):
            ops._room(bad, torch.uint8)
    for bad in (torch.zeros(1, 10).expand(4, 10), torch.zeros(10, 4).t()):
        with pytest.raises(ValueError, match="out must"):
            ops._leading(bad, 4, 10, "out")
    z, q, d = torch.zeros(5, 20), torch.full((3, 20), 0.05), torch.zeros(3, dtype=torch.int64)
    cu, u, f, e = torch.tensor([0, 1, 3]), torch.zeros(3), torch.zeros(2), torch.zeros(20)

    def verify(z, q):
        ops.verify_drafts(z, d, cu, u, f, q, None, 1.0, e, torch.zeros(2, dtype=torch.int64),
                          torch.zeros(5, dtype=torch.int64), torch.zeros(5))

    with pytest.raises(ValueError, match="CUDA"):
        verify(z, q)
    for bad in (z[:1].expand(5, 20), torch.zeros(20, 5).t()):
        with pytest.raises(ValueError, match="logits must have unit"):
            verify(bad, q)
    with pytest.raises(ValueError, match="draft_probs must have unit"):
        verify(z, q[:1].expand(3, 20))


def test_forward_mode_tangents_are_refused():
    """A tangent that would be dropped silently: in a dual tensor (also under no_grad, which leaves forward mode on) and in
    jvp. Inputs without one pass on to the next check."""
    from torch.autograd import forward_ad

    from fast_reduction import int8_ce_entropy, int8_linear, quantize_int8, verify_drafts

    x, w, s, b = torch.zeros(4, 32), torch.zeros(10, 32, dtype=torch.int8), torch.ones(10), torch.zeros(10)
    t = torch.zeros(4, dtype=torch.int64)
    z, q = torch.zeros(5, 20), torch.full((3, 20), 0.05)
    rest = (torch.zeros(3, dtype=torch.int64), torch.tensor([0, 1, 3]), torch.zeros(3), torch.zeros(2))
    calls = [(quantize_int8, x), (lambda h: int8_linear(h, w, s), x), (lambda v: int8_linear(x, w, v), s),
             (lambda v: int8_linear(x, w, s, bias=v), b), (lambda o: int8_linear(x, w, s, out=o), torch.zeros(4, 10)),
             (lambda v: int8_linear(x.to(torch.int8), w, s, hidden_scale=v), torch.ones(4)),
             (lambda h: int8_ce_entropy(h, w, s, t), x), (lambda v: int8_ce_entropy(x, w, s, t, bias=v), b),
             (lambda v: verify_drafts(v, *rest, q), z), (lambda v: verify_drafts(z, *rest, v), q)]
    for fn, v in calls:
        with pytest.raises(NotImplementedError, match="forward mode"):
            torch.func.jvp(fn, (v,), (torch.ones_like(v),))
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(v, torch.ones_like(v))
            with pytest.raises(NotImplementedError, match="forward mode"):
                fn(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                fn(dual)
            with pytest.raises(ValueError, match="CUDA"):
                fn(v)
            with pytest.raises(ValueError, match="CUDA"):
                fn(forward_ad.unpack_dual(dual).primal)
        with pytest.raises(ValueError, match="CUDA"):
            fn(dual)


def test_sizes_shared_with_the_library():
    """The limits that size workspaces in Python are those of the header that the kernels are compiled with, and the
    library asks for the workspaces that Python makes at their borders."""
    import re
    from pathlib import Path

    nat, lib = _lib()
    header = (Path(__file__).resolve().parents[1] / "include" / "frx.h").read_text()
    for name in ("FRX_I8_MAX_K", "FRX_I8_FEW_ROWS", "FRX_VERIFY_CHUNK", "FRX_DTYPE_I8", "FRX_STATUS_CHECK_FAILED",
                 "FRX_STATUS_BAD_OFFSETS"):
        assert int(re.search(rf"#define {name} (\d+)", header).group(1)) == getattr(nat, name), name
    for rows in (nat.FRX_I8_FEW_ROWS - 1, nat.FRX_I8_FEW_ROWS, nat.FRX_I8_FEW_ROWS + 1, 300):
        per = 128 if rows <= nat.FRX_I8_FEW_ROWS else 256
        need = 16 * rows * ((1000 + per - 1) // per)
        rc = lib.frx_i8_ce_entropy(A, nat.FRX_DTYPE_I8, 64, B, C, 64, D, None, 0, A, rows, 1000, 64, -100, rows, B,
                                   need - 1, A, A, None, A, None, None)
        assert rc == nat.FRX_ERR_INVALID_ARG and f"with {need} bytes".encode() in lib.frx_last_error()
    for v in (1, nat.FRX_VERIFY_CHUNK - 7, nat.FRX_VERIFY_CHUNK - 6, 128256):
        chunks = (v + 6) // nat.FRX_VERIFY_CHUNK + 1
        rc = lib.frx_verify_drafts(A, 0, v, B, B, B, B, None, 1, 0, None, 1.0, 2, 3, v, C, 4 * 5 * chunks - 1, D, D, D, None,
                                   None)
        assert rc == nat.FRX_ERR_INVALID_ARG and f"4 * 5 * {chunks} floats".encode() in lib.frx_last_error()
