"""GPU: verify_drafts against a request-by-request 64-bit restatement.

Accepted counts and tokens are compared exactly. log_probs are (z - m) / T - log S, formed in 64 bits and rounded
once, from S summed over exponentials in fp32: each is off by 2^-22 relative plus its argument's rounding
(at most 3 * 2^-24 * D for the spread D = max |z - m| log2(e) / T of terms that matter, D <= 150: below that a term
is smaller than 2^-150), sums of 64 terms per lane (64 * 2^-24) and 5 shuffles (5 * 2^-24):
    |logp - logp64| <= 2^-22 + 450 * 2^-24 + 69 * 2^-24 + 2^-24 |logp64|  <  4e-5 + 2^-24 |logp64|
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
MAX = 3.4028234663852886e38


def reference(z, d, cu, u, r, q, temps):
    """accepted, tokens, log_probs (float64), one request at a time on the host."""
    z = z.cpu().double().numpy()
    z = np.where(np.isnan(z), -np.inf, np.minimum(z, MAX))
    q = None if q is None else np.nan_to_num(np.maximum(q.cpu().double().numpy(), 0), nan=0.0, posinf=np.inf)
    d, cu, u, r = (t.cpu().numpy() for t in (d, cu, u, r))
    v = z.shape[1]
    accepted, tokens, logps = np.zeros(len(cu) - 1, np.int64), np.full(len(z), -1, np.int64), np.zeros(len(z))
    for b in range(len(cu) - 1):
        t = float(temps[b])
        greedy = not t >= float(np.float32(1e-6))
        t = 1.0 if greedy else min(t, 1e6)
        n = int(cu[b + 1] - cu[b])
        for i in range(n + 1):
            row, at = int(cu[b]) + b + i, int(cu[b]) + i
            m = z[row].max()
            drafted = i < n
            tok = int(d[at]) if drafted and 0 <= d[at] < v else -1
            if m == -np.inf:
                tokens[row], logps[row] = -1, -np.inf
                break
            with np.errstate(over="ignore", invalid="ignore"):
                e = np.where(z[row] == -np.inf, 0.0, np.exp((z[row] - m) / t))
                s = e.sum()
                logp = (z[row] - m) / t - np.log(s)
            p = e / s
            passed = False
            if greedy:
                token = int(np.argmax(z[row]))
                passed = drafted and tok == token
            else:
                if tok >= 0:
                    passed = float(u[at]) * (1.0 if q is None else q[at][tok]) < p[tok]
                if passed:
                    token = tok
                else:
                    w = p.copy()
                    if drafted and q is not None:
                        w = np.maximum(p - q[at], 0)
                    elif drafted and tok >= 0:
                        w[tok] = 0
                    if not w.sum() > 0:
                        w = p
                    c = np.cumsum(w)
                    past = np.nonzero((c > float(r[b]) * c[-1]) & (w > 0))[0]
                    token = int(past[0]) if len(past) else int(np.nonzero(w > 0)[0][-1])
            tokens[row], logps[row] = token, logp[token]
            if not passed:
                break
            accepted[b] += 1
    return accepted, tokens, logps


def check(z, d, cu, u, r, q=None, temps=1.0):
    from fast_reduction import verify_drafts

    got = verify_drafts(z, d, cu, u, r, draft_probs=q, temperature=temps)
    b = cu.numel() - 1
    t = temps.cpu().numpy() if isinstance(temps, torch.Tensor) else [np.float32(temps)] * b
    acc, tok, lp = reference(z, d, cu, u, r, q, t)
    assert got[0].dtype == torch.int64 and got[1].dtype == torch.int64 and got[2].dtype == torch.float32
    assert got[0].cpu().numpy().tolist() == acc.tolist()
    assert got[1].cpu().numpy().tolist() == tok.tolist()
    mine = got[2].cpu().double().numpy()
    inf = np.isinf(lp)
    assert (mine[inf] == lp[inf]).all()
    assert (np.abs(mine - lp)[~inf] <= 4e-5 + 2.0**-24 * np.abs(lp[~inf])).all()
    for a, b2 in zip(got, verify_drafts(z, d, cu, u, r, draft_probs=q, temperature=temps)):
        assert torch.equal(a, b2)
    return got


def make(counts, v, dtype, seed, probs=torch.float32, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n, b = sum(counts), len(counts)
    cu = torch.tensor([0] + list(np.cumsum(counts)), device=DEV)
    z = spread * torch.randn(n + b, v, device=DEV, generator=g)
    z.scatter_add_(1, torch.randint(0, v, (n + b, 3), device=DEV, generator=g),
                   3 + 6 * torch.rand(n + b, 3, device=DEV, generator=g))
    owner = torch.repeat_interleave(torch.arange(b, device=DEV), torch.tensor(counts, device=DEV))
    zd = z[torch.arange(n, device=DEV) + owner] + 0.6 * torch.randn(n, v, device=DEV, generator=g)
    q = torch.softmax(zd, -1)
    d = torch.multinomial(q, 1, generator=g)[:, 0] if n else torch.zeros(0, dtype=torch.int64, device=DEV)
    u, r = torch.rand(n, device=DEV, generator=g), torch.rand(b, device=DEV, generator=g)
    if probs is None:
        q, d = None, torch.where(u < 0.7, zd.argmax(-1), d) if n else d
    else:
        q = q.to(probs)
    return z.to(dtype), d, cu, u, r, q


@pytest.fixture(autouse=True)
def _status_clean():
    from fast_reduction import _native as nat

    nat.read_status(torch.device(DEV))
    yield
    torch.cuda.synchronize()
    nat.raise_on_status(torch.device(DEV))


@pytest.mark.parametrize("dtype,probs", [(torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16),
                                         (torch.float32, torch.float16), (torch.bfloat16, None), (torch.float32, None)])
@pytest.mark.parametrize("counts,v", [([0], 1), ([1], 2), ([3], 7), ([0, 0, 0], 100), ([4], 32000), ([2, 0, 5, 1], 3001),
                                      ([8, 9, 17], 2048), ([1, 2, 3], 2049), ([3, 3], 16385), ([4, 1], 128256),
                                      ([40, 3], 600)])
def test_matches_64_bits(dtype, probs, counts, v):
    for seed in range(3):
        check(*make(counts, v, dtype, seed + v, probs))


@pytest.mark.parametrize("v", [333, 4096])
def test_temperatures(v):
    counts = [3, 2, 4, 1, 5, 2, 0, 3, 2]
    z, d, cu, u, r, q = make(counts, v, torch.float32, 5)
    temps = torch.tensor([1.0, 0.0, 0.7, 1.7, -1.0, float("nan"), 0.0, 1e9, 0.05], device=DEV)
    got = check(z, d, cu, u, r, q, temps)
    # the greedy ones emit their rows' argmax
    for b in (1, 4, 5, 6):
        row = int(cu[b]) + b + int(got[0][b])
        assert got[1][row] == z[row].argmax()
    check(z, d, cu, u, r, q, 0.0)
    check(z, d, cu, u, r, q, 0.6)
    check(z, d, cu, u, r, None, temps)


def test_greedy_ties_take_the_lowest_index():
    v = 5000
    z = torch.zeros(5, v, device=DEV)
    z[0, [17, 2100, 4999]] = 3.0
    z[1, [4096, 4097]] = 1.0
    z[3, 4999] = float("inf")
    z[3, 4000] = MAX  # +inf counts as this
    z[4, 3:] = -float("inf")
    z[4, :3] = torch.tensor([float("nan"), -1.0, -1.0], device=DEV)
    cu = torch.tensor([0, 2, 3], device=DEV)
    d = torch.tensor([17, 4097, 0], device=DEV)
    acc, tok, _ = check(z, d, cu, torch.zeros(3, device=DEV), torch.zeros(2, device=DEV), None, 0.0)
    assert acc.tolist() == [1, 0] and tok.tolist() == [17, 4096, -1, 4000, -1]
    d[2] = 4000
    acc, tok, _ = check(z, d, cu, torch.zeros(3, device=DEV), torch.zeros(2, device=DEV), None, 0.0)
    assert acc.tolist() == [1, 1] and tok.tolist() == [17, 4096, -1, 4000, 1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("probs", [True, False])
def test_masked_rows(dtype, probs):
    """Masks of -inf, of the type's lowest value and NaN; rows whose mask leaves one token or none; +inf."""
    v = 2500
    counts = [2, 2, 2, 2, 2, 1]
    z, d, cu, u, r, q = make(counts, v, torch.float32, 9)
    inf, low = float("inf"), torch.finfo(dtype).min
    z[0, 100:] = -inf
    z[1, ::2] = float("nan")
    z[3] = -inf  # nothing left at the first draft
    z[6, :] = low  # every token at the lowest value: uniform
    z[7, 5:] = low
    z[9] = -inf
    z[9, 2400] = 1.0  # one token left
    z[10, 7] = inf
    z[10, 9] = inf
    z[12, 1:] = float("nan")
    z[12, 0] = -inf
    z[15] = -inf  # nothing left after the last draft
    d[0] = 3
    u[0] = 0.0
    d[6] = 2400
    u[7:] = 0.0
    check(z.to(dtype), d, cu, u, r, q if probs else None)


def test_ends_of_the_random_range():
    for v in (1, 5, 300, 3000, 9000):
        z, d, cu, u, r, q = make([1, 2, 0, 3], v, torch.bfloat16, 70 + v)
        for val in (0.0, 1.0, 1 - 2.0**-24, 1e-30):
            u.fill_(val)
            r.fill_(val)
            check(z, d, cu, u, r, q)
            check(z, d, cu, u, r, None)


def test_residual_with_nothing_left_falls_back_to_the_target():
    z, d, cu, u, r, q = make([2, 1], 700, torch.float32, 3)
    p = torch.softmax(z.double(), -1).float()
    q = (p[[0, 1, 3]] * 1.5).contiguous()  # above p everywhere
    u.fill_(0.999)
    acc, _, _ = check(z, d, cu, u, r, q)
    assert acc.tolist() == [0, 0]
    # without draft probabilities, and the rejected token the only one left
    z[:, 1:] = -float("inf")
    d.zero_()
    u.fill_(1.0)
    acc, tok, _ = check(z, d, cu, u, r, None)
    assert acc.tolist() == [0, 0] and tok[0] == 0


def test_bad_draft_ids_are_rejected_and_reported():
    from fast_reduction import _native as nat

    for probs in (torch.float32, None):
        for bad in (-1, 901, 2**40, -(2**62)):
            z, d, cu, u, r, q = make([3, 2], 900, torch.bfloat16, 12, probs)
            u.fill_(0.0)
            d[1] = bad
            acc, _, _ = check(z, d, cu, u, r, q)
            assert acc.tolist() == [1, 2]
            assert nat.read_status(torch.device(DEV)) == nat.FRX_STATUS_BAD_TARGET
            check(z, d, cu, u, r, q, 0.0)
            nat.read_status(torch.device(DEV))


def test_padded_batch_and_bad_offsets():
    from fast_reduction import _native as nat
    from fast_reduction import verify_drafts

    z, d, cu, u, r, q = make([2, 3], 800, torch.float32, 13)
    pad = 4
    z2 = torch.cat([z, torch.full((pad, 800), float("nan"), device=DEV)])
    d2 = torch.cat([d, torch.full((pad,), 10**9, device=DEV)])
    u2 = torch.cat([u, torch.full((pad,), float("nan"), device=DEV)])
    q2 = torch.cat([q, torch.full((pad, 800), float("nan"), device=DEV)])
    want, got = verify_drafts(z, d, cu, u, r, q), verify_drafts(z2, d2, cu, u2, r, q2)
    assert torch.equal(want[0], got[0])
    assert torch.equal(want[1], got[1][:7]) and (got[1][7:] == -1).all()
    assert torch.equal(want[2], got[2][:7]) and (got[2][7:] == 0).all()
    assert nat.read_status(torch.device(DEV)) == 0
    for bad in ([0, 6, 5], [1, 2, 5], [0, -3, 5], [0, 2, 99], [2**60, -(2**60), 2**61]):
        out = verify_drafts(z, d, torch.tensor(bad, device=DEV), u, r, q)
        assert nat.read_status(torch.device(DEV)) & nat.FRX_STATUS_BAD_OFFSETS
        assert ((out[1] >= -1) & (out[1] < 800)).all() or bad == [0, 6, 5]


def _same_outcome(a, b):
    """The same decisions; log_probs of rows that start at other 16-byte offsets are summed in another order, so each
    is within check()'s bound of the exact value and they are within twice that of each other."""
    return torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and \
        bool(((a[2].double() - b[2].double()).abs() <= 2 * (4e-5 + 2.0**-24 * a[2].double().abs())).all())


def test_strided_inputs_and_id_types():
    from fast_reduction import verify_drafts

    z, d, cu, u, r, q = make([3, 0, 2], 1003, torch.bfloat16, 15, torch.bfloat16)
    want = verify_drafts(z, d, cu, u, r, q, 0.9)
    wide_z = torch.zeros(8, 1100, device=DEV, dtype=torch.bfloat16)
    wide_q = torch.zeros(5, 1100, device=DEV, dtype=torch.bfloat16)
    for off in (0, 1, 8):
        wide_z[:, off:off + 1003] = z
        wide_q[:, off:off + 1003] = q
        got = verify_drafts(wide_z[:, off:off + 1003], d.int(), cu.int(), u, r, wide_q[:, off:off + 1003],
                            torch.full((3,), 0.9, device=DEV))
        assert _same_outcome(want, got)
    got = verify_drafts(z.t().contiguous().t(), d, cu, torch.stack([u, u], 1)[:, 0], r, q, 0.9)
    assert _same_outcome(want, got)
    one = verify_drafts(z[:1].expand(8, 1003), d, cu, u, r, q)  # row stride 0
    ref = verify_drafts(z[:1].repeat(8, 1), d, cu, u, r, q)
    assert _same_outcome(one, ref)


def test_empty_batch():
    from fast_reduction import verify_drafts

    e = torch.empty(0, device=DEV)
    ids = torch.empty(0, device=DEV, dtype=torch.int64)
    acc, tok, lp = verify_drafts(torch.empty(0, 10, device=DEV), ids, torch.zeros(1, device=DEV, dtype=torch.int64), e, e)
    assert acc.shape == tok.shape == lp.shape == (0,)


def test_offsets_past_32_bits():
    """Rows whose element offsets pass 2^31: the last sequence's rows lie behind them."""
    from fast_reduction import verify_drafts

    v, b = 131072, 17000  # 2.2e9 logits, 4.5 GB
    z = torch.zeros(b, v, device=DEV, dtype=torch.bfloat16)
    hot = torch.randint(0, v, (b,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    z.scatter_(1, hot[:, None], 60.0)  # p(hot) = 1 - 1e-21
    ids = torch.empty(0, device=DEV, dtype=torch.int64)
    acc, tok, lp = verify_drafts(z, ids, torch.zeros(b + 1, device=DEV, dtype=torch.int64), torch.empty(0, device=DEV),
                                 torch.rand(b, device=DEV))
    assert torch.equal(tok, hot) and (acc == 0).all() and (lp.abs() < 1e-6).all()


def test_head_product_verification_and_scores_together():
    """As a serving step runs them: logits of the 8-bit head, verification of the drafts, then the
    log-probabilities of what was emitted, which the scoring path gives too; eager, and captured in a graph
    whose replays follow new inputs. Two graphs, replayed in turn, keep their own workspaces.

    int8_linear's fp32 logits and the scores' differ by at most 2 * 4 * 2^-24 of a logit below 64 in size (3.1e-5),
    log_probs by 4e-5 more, scores by 2^-13 + 2^-17 + ... < 1.4e-4 (see test_int8_head_gpu.py)."""
    from fast_reduction import int8_ce_entropy, int8_linear, quantize_int8, verify_drafts

    counts, k, v = [3, 0, 4, 1], 512, 5003
    n, b = sum(counts), len(counts)
    cu = torch.tensor([0] + list(np.cumsum(counts)), device=DEV)
    codes, scale = quantize_int8(torch.randn(v, k, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0)) * 0.1)

    def inputs(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        h = torch.randn(n + b, k, device=DEV, generator=g).to(torch.bfloat16)
        p = torch.softmax(int8_linear(h, codes, scale, out_dtype=torch.float32), -1)
        rows = [i + s for s, c in enumerate(counts) for i in range(sum(counts[:s]), sum(counts[:s]) + c)]
        q = torch.softmax(torch.log(p[rows]) + 0.3 * torch.randn(n, v, device=DEV, generator=g), -1)
        d = torch.multinomial(q, 1, generator=g)[:, 0]
        return [h, d, torch.rand(n, device=DEV, generator=g), torch.rand(b, device=DEV, generator=g), q]

    def step(h, d, u, r, q):
        z = int8_linear(h, codes, scale, out_dtype=torch.float32)
        acc, tok, lp = verify_drafts(z, d, cu, u, r, q)
        ce, ent, score = int8_ce_entropy(h, codes, scale, tok, ignore_index=-1)
        return z, acc, tok, lp, score

    graphs = []
    for seed in (1, 2):
        static = inputs(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(*static)
        graphs.append((graph, static, outs))
    for seed in range(3, 9):
        graph, static, outs = graphs[seed % 2]
        fresh = inputs(seed)
        for a, f in zip(static, fresh):
            a.copy_(f)
        graphs[0][0].replay()
        graphs[1][0].replay()
        z, acc, tok, lp, score = step(*fresh)
        for a, e in zip(outs, (z, acc, tok, lp, score)):
            assert torch.equal(a, e)
        want = reference(z, fresh[1], cu, fresh[2], fresh[3], fresh[4], [1.0] * b)
        assert acc.tolist() == want[0].tolist() and tok.tolist() == want[1].tolist()
        assert ((lp - score).abs() <= 3.1e-5 + 4e-5 + 1.4e-4).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_greedy_takes_the_first_of_several_infinities(dtype):
    """+inf counts as one finite value, so several tie, also where one thread reads them one after the other."""
    z, d, cu, u, r, _ = make([2, 1, 0], 9001, dtype, 21, probs=None)
    for row, cols in enumerate([[5, 1029, 2053], [2047, 2048], [8999, 4104, 8200], [7, 8], [1024, 0], [3, 515, 4611]]):
        z[row, cols] = float("inf")
    first = torch.tensor([5, 2047, 4104, 7, 0, 3], device=DEV)
    d = first[torch.tensor([0, 1, 3], device=DEV)].clone()
    d[1] = 2048
    accepted, tokens, _ = check(z, d, cu, u, r, temps=0.0)
    assert accepted.tolist() == [1, 1, 0] and tokens.tolist() == [5, 2047, -1, 7, 0, 3]


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("temp", [1e-6, 2e-6, 3e-5])
@pytest.mark.parametrize("level", [1500.0, -1500.0, 10000.0, 70.0, 1e6])
def test_low_temperatures_and_logits_a_few_steps_apart(level, temp, probs):
    """The coldest temperatures that are not greedy, with logits of one size: neighbouring fp32 values are up to tens of
    thousands of T apart, and the cutoff below which a weight is 0 falls between two of them."""
    counts = [3, 0, 2, 1, 4]
    step = float(np.spacing(np.float32(abs(level) * (1 - 2.0**-20))))
    for v in (7, 500, 9001):
        z, d, cu, u, r, q = make(counts, v, torch.float32, v)
        g = torch.Generator(device=DEV).manual_seed(v)
        z = level - step * torch.randint(0, 9, z.shape, device=DEV, generator=g).float()
        z[1, :-1] -= 2 * step  # one token at the maximum
        rows = torch.arange(len(d), device=DEV) + torch.repeat_interleave(torch.arange(5, device=DEV),
                                                                          torch.tensor(counts, device=DEV))
        d[::2] = z[rows].argmax(-1)[::2]
        u[::3] = 0.0
        check(z, d, cu, u, r, q if probs else None, temp)


@pytest.mark.parametrize("dtype,probs", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16),
                                         (torch.float16, None), (torch.float32, None)])
@pytest.mark.parametrize("v,b", [(3, 200), (2051, 300), (32000, 30), (128256, 8)])
def test_acceptance_next_to_its_border(v, b, dtype, probs):
    """Numbers a few fp32 steps (6e-8 to 1.2e-7 each) either side of p(d) / q(d). The border is known to 1e-11 (an exponential of
    1.6e-12, sums of 64 bits), so numbers closer to it than that are moved by a step first."""
    for drafts in (1, 3):
        z, d, cu, u, r, q = make([drafts] * b, v, dtype, v + drafts, probs, spread=1.0)
        rows = torch.arange(len(d), device=DEV) + torch.arange(len(d), device=DEV) // drafts
        for temp in (1.0, 0.7):
            p = torch.softmax(z[rows].double() / float(np.float32(temp)), -1).gather(1, d[:, None])[:, 0]
            qd = torch.ones_like(p) if q is None else q.double().gather(1, d[:, None])[:, 0]
            near = (p / qd).float()
            for steps in (-2, -1, 0, 1, 2):
                bits = near.view(torch.int32) + steps
                x = bits.view(torch.float32)
                x = torch.where((x.double() * qd / p - 1).abs() < 1e-11, (bits + 1).view(torch.float32), x)
                check(z, d, cu, x, r, q, temp)


def test_strides_of_dimensions_of_one():
    """One row, or one token, whose stride torch does not care for."""
    from fast_reduction import verify_drafts

    e, ids = torch.empty(0, device=DEV), torch.empty(0, device=DEV, dtype=torch.int64)
    row = torch.randn(90, 1, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    z = row.t()
    assert z.shape == (1, 90) and z.stride(0) != 90
    check(z, ids, torch.tensor([0, 0], device=DEV), e, torch.tensor([0.4], device=DEV))
    z, d, cu, u, r, q = make([2, 1], 1, torch.float32, 3)
    flat_z, flat_q = z.reshape(1, 5).t(), q.reshape(1, 3).t()
    assert flat_z.stride(1) == 5 and flat_q.stride(1) == 3
    got, want = verify_drafts(flat_z, d, cu, u, r, flat_q), verify_drafts(z, d, cu, u, r, q)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tensor_level_call_refuses_tensors_of_the_host():
    from fast_reduction import ops

    z, d, cu, u, r, q = make([2, 1], 50, torch.float32, 3)
    ids = [torch.empty(n, device=DEV, dtype=torch.int64) for n in (2, 5)]
    good = [z, d, cu, u, r, q, torch.ones(2, device=DEV), 1.0, torch.empty(20, device=DEV), *ids,
            torch.empty(5, device=DEV)]
    ops.verify_drafts(*good)
    for i in (0, 1, 2, 3, 4, 5, 6, 8, 9, 10, 11):
        args = list(good)
        args[i] = args[i].cpu()
        with pytest.raises(ValueError, match="CUDA"):
            ops.verify_drafts(*args)
    with pytest.raises(ValueError, match="workspace"):
        ops.verify_drafts(*good[:8], torch.empty(1, device=DEV).expand(20), *good[9:])


@pytest.mark.parametrize("batch,v", [(56, 9001), (64, 9001), (120, 4500), (128, 4500), (240, 2100), (256, 2100), (600, 300)])
def test_batches_at_the_borders_of_the_cluster_sizes(batch, v):
    """One temperature for all and the same one for each take clusters of other sizes; the decisions are the same."""
    counts = [(5 * b + 3) % 4 for b in range(batch)]
    for probs in (torch.float32, None):
        args = make(counts, v, torch.bfloat16, batch, probs)
        one = check(*args, temps=0.7)
        each = check(*args, temps=torch.full((batch,), 0.7, device=DEV))
        assert torch.equal(one[0], each[0]) and torch.equal(one[1], each[1])


def test_two_threads_and_streams_at_once():
    """Two host threads, each on its own stream, verify batches that share the GPU, one of them beside the head's product."""
    import threading

    from fast_reduction import int8_linear, quantize_int8, verify_drafts

    work = [make([4, 0, 7, 2] * n, v, torch.bfloat16, n, probs) for n, v, probs in
            ((3, 20000, torch.float32), (40, 5000, None))]
    temps = [0.8, torch.tensor([0.0, 0.6, 1.0, 1.3] * 40, device=DEV)]
    g = torch.Generator(device=DEV).manual_seed(1)
    codes, scale = quantize_int8(torch.randn(9000, 256, device=DEV, generator=g))
    h = torch.randn(200, 256, device=DEV, generator=g)
    want = [check(*w, temps=t) for w, t in zip(work, temps)]
    logits = int8_linear(h, codes, scale)
    torch.cuda.synchronize()
    bad = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(40):
                y = int8_linear(h, codes, scale) if i else logits
                got = verify_drafts(*work[i], temperature=temps[i])
                if not (torch.equal(y, logits) and all(torch.equal(a, b) for a, b in zip(got, want[i]))):
                    bad.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(120)
    assert not bad
