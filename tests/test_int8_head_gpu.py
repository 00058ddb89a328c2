"""GPU: the 8-bit head (quantize_int8, int8_linear, int8_ce_entropy) against plain 64-bit computations.

Tolerances. Codes and scales are compared exactly: the scale is one fp32 division, a code the integer
nearest to the real quotient. A logit is an exact integer sum turned into fp32 (half a step, 2^-24), times two
scales (2^-24 each), plus a bias (2^-24 of the sum), rounded to the output type (half a step of it):
    |y - y64| <= finfo(out).eps / 2 * |y64| + 4 * 2^-24 * (|product| + |bias|) * (1 + 2^-8) + smallest subnormal.
For the reductions, with L = max |z| of the row and D = max z - min z: a logit is off by at most 4 * 2^-24 * L',
L' = |product| + |bias|; a base-2 exponential by 2^-22 relative plus its argument's rounding (2 * 2^-24 * D); sums
of 128 terms in fp32 in each tile half (128 * 2^-24), then at most 512 merges of 2^-22 each:
    rel = 2^-22 + 2^-23 * D + 2^-17 + 2^-13      (of S; of U the same, times its terms |z - m| <= D)
    |ce - ce64| <= rel + 8 * 2^-24 * L' + 2^-23 * |ce64|,   |H - H64| <= rel * (2 + 2 * D) + 8 * 2^-24 * L' * (1 + D).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
FLOATS = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _status_clean():
    from fast_reduction import _native as nat

    nat.read_status(torch.device(DEV))
    yield
    torch.cuda.synchronize()
    nat.raise_on_status(torch.device(DEV))


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ref_quantize(x):
    """Codes (float64 integers) and scales (float32) by definition."""
    x64 = x.double()
    amax = x.float().abs().amax(-1) if x.shape[-1] else x.new_zeros(x.shape[:-1], dtype=torch.float32)
    scale = (amax.double() / 127).float()  # 24-bit operands: rounding the 64-bit quotient once is the fp32 division
    bad = ~torch.isfinite(amax)
    scale = torch.where(scale < 2.0**-120, torch.zeros_like(scale), scale)
    live = (scale > 0) & ~bad
    scale = torch.where(bad, torch.full_like(scale, float("nan")), scale)
    codes = torch.round(x64 / torch.where(live, scale, torch.ones_like(scale)).double()[..., None])
    return torch.where(live[..., None], codes, torch.zeros_like(codes)), scale


def ref_logits(codes, scale, wcodes, wscale, bias):
    prod = (codes.double() @ wcodes.double().t()) * scale.double()[:, None] * wscale.double()[None, :]
    b = torch.zeros(wcodes.shape[0], device=DEV, dtype=torch.float64) if bias is None else bias.double()
    return prod + b, prod.abs() + b.abs()


def assert_logits(y, z, mag):
    fi = torch.finfo(y.dtype)
    tol = fi.eps / 2 * z.abs() + 4 * 2.0**-24 * mag * (1 + 2.0**-8) + fi.smallest_normal * fi.eps
    bad = ~((y.double() - z).abs() <= tol) & ~(torch.isnan(z) & torch.isnan(y))
    assert not bad.any(), (int(bad.sum()), y[bad][:4], z[bad][:4])


def make(rows, k, v, dtype, seed, bias=None):
    from fast_reduction import quantize_int8

    g = _gen(seed)
    x = torch.randn(rows, k, device=DEV, generator=g).to(dtype)
    codes, scale = quantize_int8((torch.randn(v, k, device=DEV, generator=g) * k**-0.5))
    b = None if bias is None else torch.randn(v, device=DEV, generator=g).to(bias)
    return x, codes, scale, b


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 17), (2, 16), (5, 1000), (1, 4096), (1300, 520), (257, 4096),
                                       (2, 20001), (1201, 72), (1, 131072)])
def test_quantize_matches_definition(dtype, rows, cols):
    from fast_reduction import quantize_int8

    x = (torch.randn(rows, cols, device=DEV, generator=_gen(rows + cols)) * 3).to(dtype)
    codes, scale = quantize_int8(x)
    c, s = ref_quantize(x)
    assert codes.dtype == torch.int8 and codes.stride(0) % 16 == 0
    assert torch.equal(scale, s)
    assert torch.equal(codes.double(), c)


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_halves_and_extreme_rows(dtype):
    from fast_reduction import quantize_int8

    k = 512
    x = torch.randn(12, k, device=DEV, generator=_gen(1))
    big = torch.finfo(dtype).max
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 4] = float("nan")
    x[3, 5] = -float("inf")
    # every quotient a half or next to one: the maximum is 127, so the scale is 1
    x[4] = (torch.arange(k, device=DEV) % 127).float() + 0.5
    x[4, 0] = 127
    x[5] = -x[4]
    x[6] = torch.where(torch.arange(k, device=DEV) % 2 == 0, 4.0, 2.0)  # max and half of it
    x[7] = x[7].clamp(-1, 1) * 1e-30  # subnormal or zero in fp16
    x[8] = x[8].clamp(-1, 1) * 1e-38
    x[9] = x[9].clamp(-1, 1)
    x = x.to(dtype)
    x[9, 7] = big
    x[10] = big
    x[11] = -big
    codes, scale = quantize_int8(x)
    c, s = ref_quantize(x)
    assert torch.equal(scale.isnan(), s.isnan()) and torch.equal(scale.nan_to_num(-1), s.nan_to_num(-1))
    assert torch.equal(codes.double(), c)
    assert s[[1, 2, 3]].isnan().all() and s[0] == 0


def test_quantize_strided_and_many_dimensions():
    from fast_reduction import quantize_int8

    base = torch.randn(40, 131, device=DEV, generator=_gen(2)).to(torch.bfloat16)
    for x in (base[:, 1:130], base[::3], base[:, ::2], base.t(), base.view(5, 8, 131), base[0]):
        codes, scale = quantize_int8(x)
        c, s = ref_quantize(x)
        assert codes.shape == x.shape and torch.equal(codes.double(), c) and torch.equal(scale, s)
    for shape in ((0, 5), (3, 0), (2, 0, 4), (0,)):
        codes, scale = quantize_int8(torch.empty(shape, device=DEV))
        assert codes.shape == shape and scale.shape == shape[:-1] and (scale == 0).all()


@pytest.mark.parametrize("dtype,out,bias", [(torch.bfloat16, torch.bfloat16, None),
                                            (torch.float16, torch.float32, torch.float16),
                                            (torch.float32, torch.float16, torch.float32),
                                            (torch.bfloat16, torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("rows,k,v", [(1, 16, 1), (1, 1, 5), (1, 1024, 3001), (2, 4096, 640), (7, 100, 129), (16, 256, 256),
                                      (17, 1000, 127), (37, 1000, 3001), (64, 4096, 1280), (100, 520, 333),
                                      (128, 128, 128), (129, 129, 515), (256, 384, 257), (300, 4096, 1000),
                                      (515, 65, 700)])
def test_linear_matches_64_bits(dtype, out, bias, rows, k, v):
    from fast_reduction import int8_linear

    x, w, ws, b = make(rows, k, v, dtype, rows * 7 + k + v, bias)
    y = int8_linear(x, w, ws, bias=b, out_dtype=out)
    assert y.dtype == out and y.shape == (rows, v)
    c, s = ref_quantize(x)
    assert_logits(y, *ref_logits(c, s, w, ws, b))
    assert torch.equal(y, int8_linear(x, w, ws, bias=b, out_dtype=out))  # deterministic


@pytest.mark.parametrize("rows", [1, 30, 400])
def test_linear_sums_are_exact_at_the_limits(rows):
    """Codes of +-127 and -128 over the longest row: the largest sums, which fp32 accumulation could not hold exactly."""
    from fast_reduction import int8_linear

    k, v = 131071, 200
    g = _gen(5)
    x = torch.full((rows, k), 127, device=DEV, dtype=torch.int8)
    w = torch.full((v, k), 127, device=DEV, dtype=torch.int8)
    x[:, ::9] = torch.randint(-127, 128, x[:, ::9].shape, device=DEV, generator=g, dtype=torch.int8)
    w[1::2] *= -1
    one = torch.ones(rows, device=DEV)
    y = int8_linear(x, w, torch.ones(v, device=DEV), hidden_scale=one, out_dtype=torch.float32)
    exact = x.double() @ w.double().t()
    assert torch.equal(y, exact.float())
    x.fill_(-128)
    w.fill_(-128)
    y = int8_linear(x, w, torch.ones(v, device=DEV), hidden_scale=one, out_dtype=torch.float32)
    assert (y == 131071 * 16384).all()


def test_linear_operand_layouts():
    from fast_reduction import int8_linear, quantize_int8

    x, w, ws, _ = make(24, 144, 300, torch.bfloat16, 11)
    y = int8_linear(x, w, ws)
    assert torch.equal(int8_linear(x.view(2, 3, 4, 144), w, ws), y.view(2, 3, 4, 300))
    assert torch.equal(int8_linear(x[3], w, ws), y[3])
    wide = torch.zeros(24, 300, device=DEV, dtype=torch.bfloat16)
    wide[:, 7:151] = x
    assert torch.equal(int8_linear(wide[:, 7:151], w, ws), y)
    assert torch.equal(int8_linear(x.t().contiguous().t(), w, ws), y)
    # codes that do not start on 16-byte boundaries, and a strided scale
    odd = torch.zeros(300, 147, device=DEV, dtype=torch.int8)
    odd[:, 2:146] = w
    ws2 = torch.stack([ws, ws], 1)[:, 0]
    assert torch.equal(int8_linear(x, odd[:, 2:146], ws2), y)
    # int8 hidden states, 8 tokens per group
    c, s = quantize_int8(x.view(3, 8, 144))
    assert torch.equal(int8_linear(c, w, ws, hidden_scale=s), y.view(3, 8, 300))
    # an output with longer rows: the rest of it stays as it was
    for dt in FLOATS:
        for off in (0, 1, 5):
            buf = torch.full((26, 311), 7.0, device=DEV, dtype=dt)
            got = int8_linear(x, w, ws, out=buf[1:25, off:off + 300])
            assert got.data_ptr() == buf[1:25, off:].data_ptr()
            assert torch.equal(got, int8_linear(x, w, ws, out_dtype=dt))
            rest = buf.clone()
            rest[1:25, off:off + 300] = 7.0
            assert (rest == 7.0).all()
    assert int8_linear(x[:0], w, ws).shape == (0, 300)


@pytest.mark.parametrize("rows", [3, 200])
def test_bad_tokens_and_weights_stay_in_their_row_and_column(rows):
    from fast_reduction import int8_linear, quantize_int8

    x, _, _, _ = make(rows, 256, 4, torch.float32, 3)
    wf = torch.randn(300, 256, device=DEV, generator=_gen(8))
    good = int8_linear(x, *quantize_int8(wf))
    x2, wf2 = x.clone(), wf.clone()
    x2[1, 5] = float("nan")
    wf2[70, 9] = float("inf")
    wf2[71] = 0
    y = int8_linear(x2, *quantize_int8(wf2))
    assert y[1].isnan().all() and y[:, 70].isnan().all()
    rows = [r for r in range(rows) if r != 1]
    cols = [c for c in range(300) if c not in (70, 71)]
    assert torch.equal(y[rows][:, cols], good[rows][:, cols]) and (y[rows, 71] == 0).all()


def ref_score(z, mag, t):
    lse = torch.logsumexp(z, -1)
    ls = z - lse[:, None]
    ent = -(ls.exp() * ls).sum(-1)
    ok = t >= 0
    ce = torch.where(ok, lse - z.gather(1, t.clamp(min=0)[:, None])[:, 0], torch.zeros_like(lse))
    big, d = mag.amax(-1), z.amax(-1) - z.amin(-1)
    rel = 2.0**-22 + 2.0**-23 * d + 2.0**-17 + 2.0**-13
    return ce, ent, rel + 8 * 2.0**-24 * big + 2.0**-23 * ce.abs(), rel * (2 + 2 * d) + 8 * 2.0**-24 * big * (1 + d)


@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, None), (torch.float16, torch.float16),
                                        (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("rows,k,v", [(1, 16, 1), (1, 1024, 3001), (3, 17, 20), (64, 512, 257), (130, 129, 1000),
                                      (300, 1000, 5000), (517, 256, 32000)])
def test_score_matches_64_bits(dtype, bias, rows, k, v):
    from fast_reduction import int8_ce_entropy

    x, w, ws, b = make(rows, k, v, dtype, rows + k + v, bias)
    x = x * 3
    t = torch.randint(0, v, (rows,), device=DEV, generator=_gen(4))
    t[::5] = -100
    if rows > 2:
        t[1] = v - 1
    ce, ent, lp = int8_ce_entropy(x, w, ws, t, bias=b)
    c, s = ref_quantize(x)
    z, mag = ref_logits(c, s, w, ws, b)
    ce_r, ent_r, tol_ce, tol_ent = ref_score(z, mag, t)
    assert ((ce.double() - ce_r).abs() <= tol_ce).all()
    assert ((ent.double() - ent_r).abs() <= tol_ent).all()
    assert torch.equal(lp, -ce) and (ce[t < 0] == 0).all()


def test_score_chunks_shapes_and_int8_hidden():
    from fast_reduction import int8_ce_entropy, quantize_int8

    x, w, ws, b = make(600, 384, 2001, torch.bfloat16, 21, torch.float32)
    t = torch.randint(0, 2001, (600,), device=DEV, generator=_gen(6))
    whole = int8_ce_entropy(x, w, ws, t, bias=b)
    for chunk in (1, 77, 256, 600):
        for a, e in zip(int8_ce_entropy(x, w, ws, t, bias=b, chunk_size=chunk), whole):
            assert torch.equal(a, e)
    c, s = quantize_int8(x.view(20, 30, 384))
    for a, e in zip(int8_ce_entropy(c, w, ws, t.view(20, 30).int(), bias=b, hidden_scale=s), whole):
        assert a.shape == (20, 30) and torch.equal(a.reshape(-1), e)
    for a in int8_ce_entropy(x[:0], w, ws, t[:0]):
        assert a.shape == (0,)


def test_score_bad_target_sets_status_and_nan():
    from fast_reduction import _native as nat
    from fast_reduction import int8_ce_entropy

    x, w, ws, _ = make(8, 64, 300, torch.bfloat16, 2)
    t = torch.tensor([0, 299, 300, 5, -1, 7, 8, -100], device=DEV)
    ce, ent, _ = int8_ce_entropy(x, w, ws, t)
    assert nat.read_status(torch.device(DEV)) == nat.FRX_STATUS_BAD_TARGET
    assert ce[[2, 4]].isnan().all() and ce[[0, 1, 3, 5, 6, 7]].isfinite().all() and ent.isfinite().all()


def test_other_stream_and_two_streams_at_once():
    from fast_reduction import int8_ce_entropy, int8_linear

    x, w, ws, _ = make(48, 2048, 4000, torch.bfloat16, 31)
    t = torch.randint(0, 4000, (48,), device=DEV, generator=_gen(6))
    want = int8_linear(x, w, ws)
    score = int8_ce_entropy(x, w, ws, t)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append((int8_linear(x, w, ws), int8_ce_entropy(x, w, ws, t)))
    torch.cuda.synchronize()
    for y, sc in got:
        assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(sc, score))


@pytest.mark.parametrize("rows", [5, 200])
def test_zero_negative_and_uneven_scales(rows):
    """Zero rows and weights, and the caller's own scales: negative, zero, and far apart."""
    from fast_reduction import int8_ce_entropy, int8_linear

    g = _gen(14)
    k, v = 80, 1100
    x = torch.randint(-127, 128, (rows, k), device=DEV, generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (v, k), device=DEV, generator=g, dtype=torch.int8)
    x[0] = 0
    w[:3] = 0
    xs = torch.logspace(-4, 0, rows, device=DEV) * 1e-3
    xs[1], xs[2], xs[3] = -xs[1], 0.0, -1e-3
    ws = (torch.rand(v, device=DEV, generator=g) + 0.5) * 0.1
    ws[700:] = -ws[700:]
    t = torch.randint(0, v, (rows,), device=DEV, generator=g)
    for bias in (None, torch.randn(v, device=DEV, generator=g)):
        z, mag = ref_logits(x, xs, w, ws, bias)
        assert_logits(int8_linear(x, w, ws, bias=bias, hidden_scale=xs, out_dtype=torch.float32), z, mag)
        ce, ent, _ = int8_ce_entropy(x, w, ws, t, bias=bias, hidden_scale=xs)
        ce_r, ent_r, tol_ce, tol_ent = ref_score(z, mag, t)
        assert ((ce.double() - ce_r).abs() <= tol_ce).all()
        assert ((ent.double() - ent_r).abs() <= tol_ent).all()


@pytest.mark.parametrize("rows", [3, 64, 65, 300])
@pytest.mark.parametrize("v", [97, 513, 3000])
def test_bias_of_minus_infinity_masks_its_column(rows, v):
    """Masked vocabulary entries take no part in CE and entropy; a masked target has CE +inf; a row whose mask leaves
    nothing has NaN."""
    from fast_reduction import int8_ce_entropy, int8_linear

    x, w, ws, b = make(rows, 96, v, torch.float32, rows + v, torch.float32)
    masked = torch.rand(v, device=DEV, generator=_gen(1)) < 0.5
    masked[0], masked[v - 1] = False, True
    if v > 600:
        masked[256:512] = True  # a whole tile, and half of another
        masked[640:768] = True
    b[masked] = -float("inf")
    t = torch.randint(0, v, (rows,), device=DEV, generator=_gen(2))
    t[0] = 0
    ce, ent, lp = int8_ce_entropy(x, w, ws, t, bias=b)
    c, s = ref_quantize(x)
    keep = ~masked
    z, mag = ref_logits(c, s, w[keep], ws[keep], b[keep])
    at = torch.cumsum(keep, 0)[t] - 1
    ce_r, ent_r, tol_ce, tol_ent = ref_score(z, mag, at)
    hit = masked[t]
    assert (ce[hit] == float("inf")).all() and (lp[hit] == -float("inf")).all()
    assert ((ce.double() - ce_r).abs() <= tol_ce)[~hit].all()
    assert ((ent.double() - ent_r).abs() <= tol_ent).all()
    y = int8_linear(x, w, ws, bias=b)
    assert (y[:, masked] == -float("inf")).all() and y[:, keep].isfinite().all()
    b.fill_(-float("inf"))
    ce, ent, _ = int8_ce_entropy(x, w, ws, t, bias=b)
    assert ce.isnan().all() and ent.isnan().all()


@pytest.mark.parametrize("bias", [None, torch.float32])
@pytest.mark.parametrize("rows", [5, 200])
def test_nan_in_the_last_column_alone_in_its_warp(rows, bias):
    from fast_reduction import int8_ce_entropy

    for v in (97, 129, 257, 385):
        x, w, ws, b = make(rows, 64, v, torch.bfloat16, v, bias)
        t = torch.zeros(rows, device=DEV, dtype=torch.int64)
        ws[v - 1] = float("nan")
        ce, ent, _ = int8_ce_entropy(x, w, ws, t, bias=b)
        assert ce.isnan().all() and ent.isnan().all()
        x2, w2, ws2, _ = make(rows, 64, v, torch.bfloat16, v, bias)
        x2[1, 3] = float("nan")
        ce, ent, _ = int8_ce_entropy(x2, w2, ws2, t, bias=b)
        other = [r for r in range(rows) if r != 1]
        assert ce[1].isnan() and ent[1].isnan() and ce[other].isfinite().all() and ent[other].isfinite().all()


def test_offsets_past_32_bits():
    """More than 2^31 values in, and more than 2^31 logits out: the last rows lie behind offsets of 32 bits."""
    from fast_reduction import int8_linear, quantize_int8

    rows, k = 140000, 16384  # 2.3e9 values, 4.6 GB
    x = torch.zeros(rows, k, device=DEV, dtype=torch.bfloat16)
    last = torch.randn(50, k, device=DEV, generator=_gen(3)).to(torch.bfloat16)
    x[-50:] = last
    codes, scale = quantize_int8(x)
    c, s = ref_quantize(last)
    assert torch.equal(codes[-50:].double(), c) and torch.equal(scale[-50:], s)
    assert (scale[:-50] == 0).all() and int(codes[-51].abs().max()) == 0
    del x, codes, scale
    v, m = 131072, 17000  # 2.2e9 logits
    x, w, ws, _ = make(m, 64, v, torch.bfloat16, 1)
    y = int8_linear(x, w, ws)
    c, s = ref_quantize(x[-40:])
    assert_logits(y[-40:], *ref_logits(c, s, w, ws, None))
    assert torch.equal(y[-40:], int8_linear(x[-40:], w, ws))


def test_two_threads_at_once():
    """Two host threads, each on its own stream, get what serial calls get."""
    import threading

    from fast_reduction import int8_ce_entropy, int8_linear

    work = [make(rows, 512, 3000, torch.bfloat16, rows) for rows in (20, 200)]
    t = [torch.randint(0, 3000, (x.shape[0],), device=DEV, generator=_gen(2)) for x, _, _, _ in work]
    want = [(int8_linear(x, w, ws), int8_ce_entropy(x, w, ws, tt)) for (x, w, ws, _), tt in zip(work, t)]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        x, w, ws, _ = work[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                y, sc = int8_linear(x, w, ws), int8_ce_entropy(x, w, ws, t[i])
                if not (torch.equal(y, want[i][0]) and all(torch.equal(a, b) for a, b in zip(sc, want[i][1]))):
                    bad.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(120)
    assert not bad


@pytest.mark.parametrize("fill", [-float("inf"), torch.finfo(torch.float32).min, -1e37, -3e36])
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("rows", [1, 40, 65, 300])
def test_masked_stretch_before_live_columns(rows, codes, fill):
    """Stretches of masked entries of every length that the reductions work in (16 columns, 32, a tile's half, whole
    tiles), each followed by live ones. What is masked has a weight of 0 in 64 bits too; the bounds are those of
    ref_score over the live entries."""
    from fast_reduction import int8_ce_entropy

    v = 1600
    for stretch in ([0, 16], [0, 100], [16, 48], [0, 128], [128, 200], [64, 256], [0, 256], [0, 1040], [0, v - 1]):
        x, w, ws, b = make(rows, 96, v, torch.float32, rows + stretch[1], torch.float32)
        masked = torch.zeros(v, device=DEV, dtype=torch.bool)
        masked[stretch[0]:stretch[1]] = True
        b[masked] = fill
        keep = ~masked
        live = keep.nonzero()[:, 0]
        t = live[torch.randint(0, len(live), (rows,), device=DEV, generator=_gen(3))]
        c, s = ref_quantize(x)
        if codes:
            ce, ent, lp = int8_ce_entropy(c.to(torch.int8), w, ws, t, bias=b, hidden_scale=s)
        else:
            ce, ent, lp = int8_ce_entropy(x, w, ws, t, bias=b)
        z, mag = ref_logits(c, s, w[keep], ws[keep], b[keep])
        ce_r, ent_r, tol_ce, tol_ent = ref_score(z, mag, torch.cumsum(keep, 0)[t] - 1)
        assert ((ce.double() - ce_r).abs() <= tol_ce).all(), stretch
        assert ((ent.double() - ent_r).abs() <= tol_ent).all(), stretch
        assert torch.equal(lp, -ce)


@pytest.mark.parametrize("rows,k", [(129, 16), (300, 64), (700, 200)])
def test_score_of_many_tiles_per_cta(rows, k):
    """Short sums and a long vocabulary: the epilogue's two halves hand over through the same slots up to 20 times a CTA,
    with nothing else to wait for."""
    from fast_reduction import int8_ce_entropy

    v = 128256
    x, w, ws, b = make(rows, k, v, torch.bfloat16, rows, torch.float32)
    t = torch.randint(0, v, (rows,), device=DEV, generator=_gen(4))
    for bias in (None, b):
        c, s = ref_quantize(x)
        ce_r, ent_r, tol_ce, tol_ent = ref_score(*ref_logits(c, s, w, ws, bias), t)
        first = int8_ce_entropy(x, w, ws, t, bias=bias)
        assert ((first[0].double() - ce_r).abs() <= tol_ce).all()
        assert ((first[1].double() - ent_r).abs() <= tol_ent).all()
        for _ in range(20):
            for a, e in zip(int8_ce_entropy(x, w, ws, t, bias=bias), first):
                assert torch.equal(a, e)


@pytest.mark.parametrize("dtype", FLOATS)
def test_strides_of_dimensions_of_one(dtype):
    """One row, or one column, whose stride torch does not care for: a transposed column, a row of an expanded matrix, a
    column of a transposed row."""
    from fast_reduction import int8_ce_entropy, int8_linear, quantize_int8

    k = 70
    col = torch.randn(k, 1, device=DEV, generator=_gen(1)).to(dtype)
    wide = torch.randn(1, k, device=DEV, generator=_gen(2)).to(dtype)
    w, ws = quantize_int8(torch.randn(300, k, device=DEV, generator=_gen(3)))
    t = torch.tensor([7], device=DEV)
    for x in (col.t(), wide.expand(5, k)[:1], wide.expand(5, k)[2:3], wide.as_strided((1, k), (3, 1))):
        assert x.shape == (1, k) and x.stride(0) != k
        c, s = ref_quantize(x)
        codes, scale = quantize_int8(x)
        assert torch.equal(codes.double(), c) and torch.equal(scale, s)
        assert_logits(int8_linear(x, w, ws), *ref_logits(c, s, w, ws, None))
        for a, e in zip(int8_ce_entropy(x, w, ws, t), int8_ce_entropy(x.clone().view(1, k), w, ws, t)):
            assert torch.equal(a, e)
    one = torch.randn(1, 40, device=DEV, generator=_gen(4)).to(dtype)
    w1, ws1 = quantize_int8(torch.randn(300, 1, device=DEV, generator=_gen(5)))
    for x in (one.t(), one.t()[:1]):
        assert x.shape[1] == 1 and x.stride(1) == 40
        c, s = ref_quantize(x)
        codes, scale = quantize_int8(x)
        assert torch.equal(codes.double(), c) and torch.equal(scale, s)
        assert_logits(int8_linear(x, w1, ws1), *ref_logits(c, s, w1, ws1, None))
        assert torch.equal(int8_linear(codes, w1, ws1, hidden_scale=scale, out_dtype=dtype), int8_linear(x, w1, ws1))


def test_tensor_level_calls_refuse_tensors_of_the_host():
    """Every tensor of a call has to be on the GPU, outputs and workspaces too."""
    from fast_reduction import ops

    x, w, ws, b = make(4, 64, 100, torch.bfloat16, 1, torch.float32)
    t = torch.zeros(4, device=DEV, dtype=torch.int64)
    out, work = torch.empty(4, 100, device=DEV), torch.empty(1 << 16, device=DEV, dtype=torch.uint8)
    r = [torch.empty(4, device=DEV) for _ in range(3)]
    good = [x, None, w, ws, out, work]
    for i in (0, 2, 3, 4, 5):
        args = list(good)
        args[i] = args[i].cpu()
        with pytest.raises(ValueError, match="CUDA"):
            ops.gemm_i8(*args, bias=b)
    with pytest.raises(ValueError, match="overlap"):
        ops.gemm_i8(x, None, w, ws, torch.empty(1, 100, device=DEV).expand(4, 100), work)
    good = [x, None, w, ws, t, *r, work]
    for i in (0, 2, 3, 4, 5, 6, 7, 8):
        args = list(good)
        args[i] = args[i].cpu()
        with pytest.raises(ValueError, match="CUDA"):
            ops.i8_ce_entropy(*args, launch_rows=4, ignore_index=-100)
    with pytest.raises(ValueError, match="workspace"):
        ops.gemm_i8(x, None, w, ws, out, work[:1].expand(1 << 16))


@pytest.mark.parametrize("rows", [6, 200])
def test_results_of_scoring_are_tensors_of_their_own(rows):
    """Each result can be changed in place while another is saved for a backward pass, and keeps no memory but its own."""
    from fast_reduction import int8_ce_entropy

    x, w, ws, _ = make(rows, 64, 300, torch.bfloat16, 2)
    t = torch.zeros(rows, device=DEV, dtype=torch.int64)
    for hidden, shape in ((x, (rows,)), (x.view(2, rows // 2, 64), (2, rows // 2))):
        out = int8_ce_entropy(hidden, w, ws, t)
        assert len({o.untyped_storage().data_ptr() for o in out}) == 3
        assert all(o.shape == shape and o.untyped_storage().nbytes() == 4 * rows for o in out)
        a = torch.ones(shape, device=DEV, requires_grad=True)
        loss = (a * out[1]).sum()  # saves the entropy
        out[0].mul_(2)
        out[2].zero_()
        loss.backward()
        assert torch.equal(a.grad, out[1])


@pytest.mark.parametrize("rows", [1, 33, 64, 128])
@pytest.mark.parametrize("v", [37889, 128256])
@pytest.mark.parametrize("k", [100, 1000])
def test_few_tokens_with_many_tiles_per_cta(rows, v, k):
    """Above 296 tiles of 128 entries a CTA of the few-token kernels takes several, through both accumulators, a ring of K
    steps that wraps inside a tile and across tiles, and the same slots again. Without a bias and with one that masks
    whole tiles, warps' quarters of a tile and single entries."""
    from fast_reduction import int8_ce_entropy, int8_linear

    x, w, ws, b = make(rows, k, v, torch.bfloat16, rows + k, torch.float32)
    t = torch.randint(0, v, (rows,), device=DEV, generator=_gen(4))
    t[0] = v - 1
    c, s = ref_quantize(x)
    masked = torch.rand(v, device=DEV, generator=_gen(1)) < 0.3
    tile = torch.arange(v, device=DEV) // 128
    masked |= (tile % 7 == 3) | ((tile % 5 == 1) & (torch.arange(v, device=DEV) % 128 < 32))
    masked[t] = False
    b[masked] = -float("inf")
    for bias, keep in ((None, torch.ones_like(masked)), (b, ~masked)):
        y = int8_linear(x, w, ws, bias=bias, out_dtype=torch.float32)
        z, mag = ref_logits(c, s, w[keep], ws[keep], None if bias is None else bias[keep])
        assert_logits(y[:, keep], z, mag)
        assert (y[:, ~keep] == -float("inf")).all()
        assert torch.equal(y, int8_linear(x, w, ws, bias=bias, out_dtype=torch.float32))
        got = int8_ce_entropy(x, w, ws, t, bias=bias)
        ce_r, ent_r, tol_ce, tol_ent = ref_score(z, mag, torch.cumsum(keep, 0)[t] - 1)
        assert ((got[0].double() - ce_r).abs() <= tol_ce).all()
        assert ((got[1].double() - ent_r).abs() <= tol_ent).all()
        for _ in range(5):
            assert all(torch.equal(a, e) for a, e in zip(int8_ce_entropy(x, w, ws, t, bias=bias), got))


FIRST_CALL_CAPTURED = """
import torch
from fast_reduction import _native as nat, int8_ce_entropy
dev = torch.device("cuda", 0)
x, ws = torch.randn(4, 64, device=dev), torch.ones(300, device=dev)
w, t = torch.randint(-127, 128, (300, 64), device=dev, dtype=torch.int8), torch.tensor([0, 1, 2, 3], device=dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ce, _, _ = int8_ce_entropy(x, w, ws, t)
assert nat.read_status(dev) == 0
bad = t.clone()
bad[1] = 300
want = int8_ce_entropy(x, w, ws, bad)[0]
graph.replay()
assert nat.read_status(dev) == nat.FRX_STATUS_BAD_TARGET
assert nat.read_status(dev) == 0
assert torch.equal(ce[[0, 2, 3]], want[[0, 2, 3]]) and ce.isfinite().all()
t.fill_(-5)
graph.replay()
assert nat.read_status(dev) == nat.FRX_STATUS_BAD_TARGET and ce.isnan().all()
"""


def test_first_call_of_a_process_captured_in_a_graph():
    """Replays neither clear what other calls reported nor need a call before the capture."""
    import os
    import subprocess
    import sys
    from pathlib import Path

    repo = Path(__file__).resolve().parents[1]
    out = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=repo, capture_output=True, text=True, timeout=300,
                         env=dict(os.environ, PYTHONPATH=str(repo / "fast-reduction_b200")))
    assert out.returncode == 0, out.stderr[-2000:]
