"""The operators on embedding rows (proxima_b200.rows) on a GPU, against the
same formulas in 64 bits.

Every tolerance is an error bound of the arithmetic, evaluated per output:
u = 2^-24 is half a step of fp32, h half a step of the output's type. The
tensor cores' fp32 sums of n products are taken at 3 * 2^-23 of the sum of
their magnitudes per product (the bound the search certificate uses).
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACC = 3 * 2.0 ** -23
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half the smallest step
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _rand(*shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _within(got, want, bound, what=""):
    got, bound = got.double(), bound + 0 * want
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound)[bad].max())} bounds"


# ---------------------------------------------------------------- 8-bit rows

def _codes64(x):
    """Codes and scales in 64 bits: the quotient of two fp32 numbers is at
    least 2^-24 of itself away from a half it does not equal, so a 64-bit
    quotient rounds as the exact one does."""
    scales = (x.float().abs().amax(1).cpu().numpy() / np.float32(127)).astype(np.float32)
    scales = torch.from_numpy(scales).to(x.device)
    codes = (x.double() / scales.double()[:, None]).round().clamp(-127, 127)
    return torch.where(scales[:, None] == 0, 0.0, codes).to(torch.int8), scales


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", [(1, 1), (1, 768), (3, 7), (5, 38), (2, 261), (1000, 128), (77, 100), (129, 384), (13, 1000),
                                 (4, 1024), (3, 1025), (2, 5000), (2, 5001), (100_001, 16)])
def test_quantize_rows(px, dtype, n, d):
    x = _rand(n, d, seed=n + d, dtype=dtype)
    codes, scales = px.quantize_rows(x)
    want, want_scales = _codes64(x)
    assert codes.shape == (n, d) and codes.dtype == torch.int8
    assert codes.data_ptr() % 16 == 0 and (n == 1 or codes.stride(0) % 16 == 0)
    assert torch.equal(scales, want_scales)
    assert torch.equal(codes, want)
    back = px.dequantize_rows(codes, scales, dtype=dtype)
    exact = want.double() * want_scales.double()[:, None]
    _within(back, exact, exact.abs() * (HALF[dtype] + 2 * U) + TINY[dtype], "dequantize")


def test_quantize_rounds_exactly_at_halves(px):
    # Rows with a maximum of 127 * s (scale exactly s) whose values lie on and
    # one fp32 step around every half of s.
    rows = []
    for s in (1.0, 0.375, 1.1920929e-07, 3.0e-38):
        s = np.float32(s)
        half = ((np.arange(-126, 126, dtype=np.float64) + 0.5) * s).astype(np.float32)
        rows.append(np.concatenate([half, np.nextafter(half, np.float32(np.inf)), np.nextafter(half, np.float32(-np.inf)),
                                    np.float32([127 * s])]))
    x = torch.from_numpy(np.stack(rows)).cuda()
    codes, scales = px.quantize_rows(x)
    want, want_scales = _codes64(x)
    assert torch.equal(scales, want_scales) and torch.equal(codes, want)


def test_quantize_special_rows(px):
    x = _rand(8, 40, seed=3)
    x[0] = 0.0
    x[1, 39] = math.nan
    x[2, 0] = math.inf
    x[3, 5] = -math.inf
    x[4] = 1e-45  # the smallest number: its scale underflows to 0
    x[5] *= 1e-41
    x[6, 7] = 3.4e38
    codes, scales = px.quantize_rows(x)
    assert scales[0] == 0 and not codes[0].any()
    assert scales[1:4].isnan().all() and not codes[1:4].any()
    assert scales[4] == 0 and not codes[4].any()
    want, want_scales = _codes64(x)
    rest = [5, 6, 7]
    assert torch.equal(scales[rest], want_scales[rest]) and torch.equal(codes[rest], want[rest])
    assert px.dequantize_rows(codes, scales)[1].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,lead", [(1, 1, 1), (5000, 1, 3), (700, 3, 1), (3001, 33, 0), (3001, 33, 5), (1200, 130, 2), (601, 619, 7),
                                      (40, 1537, 1), (40, 2048, 0), (9, 7999, 3), (3, 16001, 1), (2, 20001, 0)])
def test_contiguous_rows_anywhere(px, dtype, n, d, lead):
    # Contiguous rows from any element on, short and long, and back; what lies
    # around them is not read.
    buf = torch.full((n * d + 32,), math.nan, dtype=dtype, device="cuda")
    x = buf[lead:lead + n * d].view(n, d)
    x.copy_(_rand(n, d, seed=n + d, dtype=dtype))
    codes, scales = px.quantize_rows(x)
    want, want_scales = _codes64(x)
    assert torch.equal(codes, want) and torch.equal(scales, want_scales)
    back = px.dequantize_rows(codes, scales, dtype)
    exact = codes.double() * scales.double()[:, None]
    _within(back, exact, (U + HALF[dtype]) * 1.001 * exact.abs() + TINY[dtype])
    # Into an output that begins anywhere: its surroundings stay.
    lib, out = px._lib.load(), torch.full((n * d + 32,), 7.0, dtype=dtype, device="cuda")
    kinds = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    px._lib.check(lib.px_dequantize_rows_device(0, codes.data_ptr(), codes.stride(0), scales.data_ptr(), n, d, kinds[dtype],
                                                out[lead:].data_ptr(), d, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[lead:lead + n * d].view(n, d), back)
    assert (out[:lead] == 7.0).all() and (out[lead + n * d:] == 7.0).all()


def test_quantize_strided_inputs(px):
    base = _rand(50, 200, seed=9)
    want = px.quantize_rows(base[:, 3:100].contiguous())
    for x in (base[:, 3:100], base.t().contiguous().t()[:, 3:100]):  # misaligned rows; strided columns
        codes, scales = px.quantize_rows(x)
        assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    one = base[:1, :97].expand(5, 97)  # rows that share memory
    codes, scales = px.quantize_rows(one)
    assert torch.equal(codes, px.quantize_rows(base[:1, :97])[0].expand(5, 97))
    # Codes with an odd pitch.
    c, s = px.quantize_rows(base)
    odd = torch.empty(50, 201, dtype=torch.int8, device="cuda")[:, 1:]
    odd.copy_(c)
    assert torch.equal(px.dequantize_rows(odd, s), px.dequantize_rows(c, s))


# ---------------------------------------------------------------- 8-bit scores

def _scores_case(m, n, d, seed, bias):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(-127, 128, (m, d), device="cuda", generator=g, dtype=torch.int8)
    x = torch.randint(-127, 128, (n, d), device="cuda", generator=g, dtype=torch.int8)
    qs = torch.rand(m, device="cuda", generator=g) + 0.01
    xs = torch.rand(n, device="cuda", generator=g) + 0.01
    b = torch.randn(n, device="cuda", generator=g) * d * 1000 if bias else None
    return q, qs, x, xs, b


def _scores64(q, qs, x, xs, b):
    dots = q.double() @ x.double().T  # whole numbers below 2^53
    s = dots * qs.double()[:, None] * xs.double()
    return s if b is None else s + b.double()


def _scores_bound(want, b, dtype):
    # The sum's conversion, the product of the scales, and the fused multiply
    # and add: u each; then the output's own half step.
    prod = (want if b is None else want - b.double()).abs()
    return (2.001 * U) * prod + (U + HALF[dtype]) * 1.001 * want.abs() + TINY[dtype]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,d", [(1, 1, 1), (1, 1000, 128), (2, 255, 16), (33, 257, 100), (64, 512, 384), (255, 513, 129),
                                   (256, 300, 768), (257, 1031, 65), (300, 640, 896), (520, 999, 1000), (5, 77, 3000)])
def test_int8_scores(px, dtype, bias, m, n, d):
    q, qs, x, xs, b = _scores_case(m, n, d, m + n + d, bias)
    got = px.int8_scores(q, qs, x, xs, bias=b, dtype=dtype)
    assert got.shape == (m, n) and got.dtype == dtype
    want = _scores64(q, qs, x, xs, b)
    if dtype == torch.float16:  # keep inside the type's range
        f = 2.0 ** -math.ceil(math.log2(float(want.abs().max()) / 30000)) if want.abs().max() > 30000 else 1.0
        b = None if b is None else b * f
        got = px.int8_scores(q, qs * f, x, xs, bias=b, dtype=dtype)
        want = want * f
    _within(got, want, _scores_bound(want, b, dtype), "scores")


def test_int8_scores_many_tiles(px):
    # More tiles than clusters, several query groups, odd row counts.
    q, qs, x, xs, b = _scores_case(700, 30_001, 200, 5, True)
    want = _scores64(q, qs, x, xs, b)
    for dtype in (torch.float32, torch.bfloat16):
        _within(px.int8_scores(q, qs, x, xs, bias=b, dtype=dtype), want, _scores_bound(want, b, dtype), str(dtype))


def test_int8_scores_longest_sums(px):
    # The most products a 32-bit sum holds, all of one sign.
    d = 131071
    q = torch.full((2, d), -128, dtype=torch.int8, device="cuda")
    x = torch.full((3, d), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(3, device="cuda")
    got = px.int8_scores(q, one[:2], x, one)
    assert torch.equal(got, torch.full((2, 3), float(np.float32(128 * 128 * d)), device="cuda"))


def test_int8_scores_special_scales(px):
    q, qs, x, xs, _ = _scores_case(3, 100, 64, 1, False)
    qs[1] = math.nan
    xs[7] = 0.0
    b = torch.zeros(100, device="cuda")
    b[9] = -math.inf
    got = px.int8_scores(q, qs, x, xs, bias=b)
    assert got[1].isnan().all() and not got[[0, 2]].isnan().any()
    assert (got[[0, 2], 7] == 0).all() and (got[[0, 2], 9] == -math.inf).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_int8_scores_out_and_strides(px, dtype):
    m, n, d = 70, 301, 90
    q, qs, x, xs, b = _scores_case(m, n, d, 4, True)
    qs, b = qs / 100, b / 100
    want = px.int8_scores(q, qs, x, xs, bias=b, dtype=dtype)
    # A strided output: what lies around it stays.
    for lead, pitch in ((0, 304), (1, 305), (3, 310)):
        buf = torch.full((m + 2, pitch), 7.0, dtype=dtype, device="cuda")
        out = buf[1:-1, lead:lead + n]
        assert px.int8_scores(q, qs, x, xs, bias=b, dtype=dtype, out=out) is out
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert (buf == 7.0).all()
    # Codes in other layouts.
    odd = torch.empty(n, 91, dtype=torch.int8, device="cuda")[:, 1:]
    odd.copy_(x)
    assert torch.equal(px.int8_scores(q.t().contiguous().t(), qs, odd, xs, bias=b, dtype=dtype), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_int8_scores_ragged_ends(px, dtype):
    # Every place of a row's two ends within and across tiles of 128, in rows
    # that begin anywhere; what lies around them stays.
    m, d = 19, 40
    q, qs, x, xs, _ = _scores_case(m, 400, d, 5, False)
    qs, want = qs / 100, px.int8_scores(q, qs / 100, x, xs, dtype=dtype)
    _within(want, _scores64(q, qs, x, xs, None), _scores_bound(_scores64(q, qs, x, xs, None), None, dtype))
    for n in [*range(1, 20), *range(112, 146), *range(250, 275), 391]:
        for lead, pitch in ((0, n + 9), (1 + n % 15, 401 + n % 3)):
            buf = torch.full((m, 432), 7.0, dtype=dtype, device="cuda").view(-1)
            out = buf[lead:].as_strided((m, n), (pitch, 1))
            px.int8_scores(q, qs, x[:n], xs[:n], dtype=dtype, out=out)
            assert torch.equal(out, want[:, :n]), (n, lead)
            out.fill_(7.0)
            assert (buf == 7.0).all(), (n, lead)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 9, 17, 32, 41, 49, 270])
def test_int8_scores_many_ragged_tiles(px, dtype, m):
    n, d = 100_003, 24
    q, qs, x, xs, b = _scores_case(m, n, d, 6, True)
    qs, b = qs / 100, b / 100
    want = _scores64(q, qs, x, xs, b)
    _within(px.int8_scores(q, qs, x, xs, bias=b, dtype=dtype), want, _scores_bound(want, b, dtype), "scores")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [73, 81])
def test_int8_scores_large_ragged_matrices(px, dtype, m):
    # Matrices past 320 MB off 16-byte boundaries, which leave another way.
    most, d = 2_400_130, 16
    q, qs, x, xs, b = _scores_case(m, most, d, 7, True)
    qs, b = qs / 100, b / 100
    full = px.int8_scores(q, qs, x, xs, bias=b, dtype=dtype)
    for i in range(0, m, 16):
        want = _scores64(q[i:i + 16], qs[i:i + 16], x, xs, b)
        _within(full[i:i + 16], want, _scores_bound(want, b, dtype), "scores")
    buf = torch.full((m * (most + 16),), 7.0, dtype=dtype, device="cuda")
    for n in [*range(2_400_000, 2_400_129, 16), 2_400_127, 2_400_129]:
        for lead, pitch in ((0, n + 9), (1 + n % 15, n)):
            out = buf[lead:].as_strided((m, n), (pitch, 1))
            px.int8_scores(q, qs, x[:n], xs[:n], bias=b[:n], dtype=dtype, out=out)
            assert torch.equal(out, full[:, :n]), (n, lead)
            out.fill_(7.0)
            assert (buf == 7.0).all(), (n, lead)


def test_int8_scores_offsets_beyond_32_bits(px):
    # An output of more than 2^31 values, of which the last rows are checked.
    m, n, d = 2200, 1_000_003, 32
    q, qs, x, xs, _ = _scores_case(m, n, d, 8, False)
    got = px.int8_scores(q, qs, x, xs, dtype=torch.bfloat16)
    want = _scores64(q[-3:], qs[-3:], x, xs, None)
    _within(got[-3:], want, _scores_bound(want, None, torch.bfloat16), "last rows")


def test_quantized_scores_follow_a_search(px):
    """Rows cut to 8 bits and scored: the L2 order of the scores against an
    exact search, over the distance the codes' rounding allows."""
    rows, q = _rand(5000, 96, seed=1), _rand(40, 96, seed=2)
    codes, scales = px.quantize_rows(rows)
    qc, qs = px.quantize_rows(q)
    xhat, qhat = px.dequantize_rows(codes, scales), px.dequantize_rows(qc, qs)
    got = px.int8_scores(qc, qs, codes, scales, bias=-0.5 * xhat.square().sum(1))
    ids = got.topk(10, dim=1).indices
    idx = px.FlatIndex(96, px.Metric.L2)
    idx.add(rows.cpu().numpy())
    _, dist = idx.search_batch(q.cpu().numpy(), k=10)
    mine = (q[:, None].double() - rows[ids].double()).norm(dim=2).sort(1).values.cpu().numpy()
    # |q - x| and |qhat - xhat| differ by at most the two rows' rounding, so the
    # i-th nearest by codes is at most twice that farther than the i-th nearest.
    slack = float((rows - xhat).norm(dim=1).max()) + float((q - qhat).norm(dim=1).max())
    assert (mine <= dist + 2 * slack + 1e-4).all()


# ---------------------------------------------------------------- softmax loss

def _xent64(q, r, y, scale, bias, ignore, g):
    """Loss, its terms and gradients in 64 bits, and bounds on the kernels'
    errors. g: the gradient of each query's loss."""
    q, r = q.detach().double(), r.detach().double()
    t, d = q.shape
    v = r.shape[0]
    z = scale * (q @ r.T)
    mag = scale * (q.abs() @ r.abs().T)
    b = torch.zeros(v, dtype=torch.float64, device=q.device) if bias is None else bias.double()
    out = b == -math.inf
    z = torch.where(out, -math.inf, z + torch.where(out, 0.0, b))
    used = y != ignore
    inside = (y >= 0) & (y < v)
    at = torch.where(inside, y, 0)
    lse = torch.logsumexp(z, 1)
    zt = z.gather(1, at[:, None])[:, 0]
    loss = torch.where(zt == -math.inf, math.inf, lse - zt)
    loss = torch.where(used, torch.where(inside, loss, math.nan), 0.0)
    # A logit's error: the product's sum, the scale in log2 units (two
    # roundings), the multiply-add, the bias's conversion, the subtraction of
    # the maximum: within 6u of the magnitudes, times the largest in the row.
    fin = torch.where(z.isinf(), 0.0, z)
    dz = (ACC * (d + 2) * mag + 6 * U * (mag + b.abs().nan_to_num(posinf=0))).amax(1) + 2 * U * fin.abs().amax(1)
    # The sum: ex2 within 2^-22, a chain of additions of at most v/64 + 200.
    dsum = 2.0 ** -22 + (v / 64 + 200) * U
    dloss = 2 * dz + dsum + 8 * U * (fin.abs().amax(1) + torch.where(loss.isfinite(), loss, 0.0)) + 4 * U
    p = torch.exp(z - torch.where(lse == -math.inf, 0.0, lse)[:, None])
    onehot = torch.zeros_like(p)
    counted = used & inside
    onehot[torch.arange(t, device=q.device)[counted], y[counted]] = 1.0
    g = torch.where(counted, g.double(), 0.0)
    G = (p - onehot) * g[:, None]
    half = HALF[torch.bfloat16] if _xent64.dtype == torch.bfloat16 else HALF[torch.float16]
    # An entry: its probability's relative error, its rounding to 16 bits, and
    # fp16's smallest step at a lift of 2^14 below the largest gradient.
    dp = 2 * (dz + dloss + 2.0 ** -22)[:, None]
    small = float(g.abs().max()) * 2.0 ** -39 if _xent64.dtype == torch.float16 else 0.0
    dG = G.abs() * half * 1.01 + p * dp * g.abs()[:, None] + onehot * (dp + 4 * U) * G.abs() + small
    dq, dr = scale * G @ r, scale * G.T @ q
    bq = scale * ((dG + ACC * (v + 2) * G.abs()) @ r.abs()) + 4 * U * dq.abs()
    br = scale * ((dG + ACC * (t + 2) * G.abs()).T @ q.abs()) + 4 * U * dr.abs()
    tiny = TINY[_xent64.dtype]
    return loss, dloss, lse, (dq, bq + 1.01 * half * dq.abs() + tiny), (dr, br + 1.01 * half * dr.abs() + tiny)


def _xent_case(t, v, d, dtype, seed, bias=False, ignored=False, pitch=True):
    unit = 8 if pitch else 1
    width = (d + unit - 1) // unit * unit
    q = torch.empty(t, width, dtype=dtype, device="cuda")[:, :d]
    r = torch.empty(v, width, dtype=dtype, device="cuda")[:, :d]
    q.copy_(_rand(t, d, seed=seed) / math.sqrt(d))
    r.copy_(_rand(v, d, seed=seed + 1))
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    y = torch.randint(0, v, (t,), device="cuda", generator=g)
    b = None
    if bias:
        b = _rand(v, seed=seed + 3)
        b[torch.rand(v, device="cuda", generator=g) < 0.2] = -math.inf
        b[y] = b[y].nan_to_num(neginf=0.5)
    if ignored:
        y = y.masked_fill(torch.rand(t, device="cuda", generator=g) < 0.3, -100)
    return q, r, y, b


def _check_xent(px, q, r, y, b, scale=1.5, reduction="none", ignore=-100, weights=None):
    _xent64.dtype = q.dtype
    q, r = q.detach().requires_grad_(), r.detach().requires_grad_()
    used = (y != ignore)
    loss = px.softmax_cross_entropy(q, r, y, scale=scale, bias=b, ignore_index=ignore, reduction=reduction)
    t = q.shape[0]
    if reduction == "none":
        g = torch.ones(t, device="cuda") if weights is None else weights
        (loss * g).sum().backward()
    else:
        g = torch.full((t,), 0.75 / (float(used.sum()) if reduction == "mean" else 1.0), device="cuda")
        (loss * 0.75).backward()
    want, dloss, _, (dq, bq), (dr, br) = _xent64(q, r, y, scale, b, ignore, g)
    if reduction == "none":
        assert loss.shape == (t,) and loss.dtype == torch.float32
        fin = want.isfinite()
        assert torch.equal(loss[~fin].isnan(), want[~fin].isnan()) and torch.equal(loss.isinf(), want.isinf())
        _within(loss[fin], want[fin], dloss[fin], "loss")
        assert (loss[~used] == 0).all()
    else:
        total = want.sum() / (float(used.sum()) if reduction == "mean" else 1.0)
        assert loss.shape == ()
        _within(loss, total, (dloss * used).sum() / (used.sum() if reduction == "mean" else 1) + 2 * U * total.abs(), "total")
    assert q.grad.dtype == q.dtype and r.grad.shape == r.shape
    _within(q.grad, dq, bq, "grad of queries")
    _within(r.grad, dr, br, "grad of rows")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,v,d", [(1, 1, 8), (1, 1000, 64), (3, 2, 16), (2, 31, 1), (128, 256, 64), (129, 257, 65),
                                   (256, 255, 128), (300, 700, 100), (257, 5000, 200), (40, 3000, 384), (65, 513, 520),
                                   (1000, 300, 32), (30, 100, 1030)])
def test_softmax_cross_entropy(px, dtype, t, v, d):
    _check_xent(px, *_xent_case(t, v, d, dtype, t + v + d))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("t,v,d", [(5, 40, 24), (300, 1001, 96)])
def test_softmax_bias_ignored_and_reductions(px, dtype, reduction, t, v, d):
    _check_xent(px, *_xent_case(t, v, d, dtype, 7, bias=True, ignored=True), reduction=reduction)


def test_softmax_weighted_queries(px):
    q, r, y, b = _xent_case(200, 500, 64, torch.bfloat16, 11, ignored=True)
    w = torch.linspace(-2, 3, 200, device="cuda")
    _check_xent(px, q, r, y, b, weights=w)
    _check_xent(px, q, r, y, b, weights=torch.zeros(200, device="cuda"))


@pytest.mark.parametrize("v", [230_007, 520_009])
def test_softmax_several_pieces(px, v):
    # Bases of one and of several pieces of the gradient's buffer, the last ragged.
    t, d = 300, 16
    ws = px._lib.load().px_softmax_xent_workspace_bytes(0, t, v, d, 1)
    assert (ws < 2 * t * v) == (v == 520_009)
    _check_xent(px, *_xent_case(t, v, d, torch.bfloat16, 21), reduction="mean")


def test_softmax_several_pieces_with_shared_targets(px):
    # Every third query has the same target, in the second piece; the others
    # share theirs by twos and threes.
    t, v, d = 300, 520_009, 16
    q, r, y, b = _xent_case(t, v, d, torch.float16, 22, bias=True, ignored=True)
    y[::3] = 400_001
    y[1:40] = y[1:40] // 1000 * 1000
    y[50:56] = 7
    b[y[y >= 0]] = 0.25
    _check_xent(px, q, r, y, b, weights=torch.linspace(0.5, 2, t, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,v,d", [(1, 1, 8), (5, 70, 40), (65, 250, 64), (200, 5001, 100), (333, 520_009, 16)])
def test_softmax_results_do_not_depend_on_what_workspaces_held(px, monkeypatch, dtype, t, v, d):
    # All logits near -1000, so that a logit of 0 past the base's end would
    # weigh infinitely much.
    q = _rand(t, d, seed=71, dtype=dtype) * 0.05 + 8
    r = _rand(v, d, seed=72, dtype=dtype) * 0.05 - 1000 / 8 / d
    y = torch.arange(t, device="cuda") * 7 % v
    real = torch.empty

    def step(bits):
        def filled(*args, **kw):
            x = real(*args, **kw)
            if x.is_cuda:
                x.fill_(bits if x.dtype == torch.uint8 else math.nan if bits else 0.0)
            return x

        monkeypatch.setattr(torch, "empty", filled)
        a, b = q.clone().requires_grad_(), r.clone().requires_grad_()
        loss = px.softmax_cross_entropy(a, b, y)
        loss.backward()
        monkeypatch.setattr(torch, "empty", real)
        return loss, a.grad, b.grad

    want = step(0)
    assert all(x.isfinite().all() for x in want)
    assert all(torch.equal(x, w) for x, w in zip(step(255), want))


def test_softmax_unpitched_and_strided_operands(px):
    q, r, y, b = _xent_case(70, 300, 50, torch.bfloat16, 31, bias=True)
    q2, r2, _, _ = _xent_case(70, 300, 50, torch.bfloat16, 31, bias=True, pitch=False)  # rows of 100 bytes
    rt = r.t().contiguous().t()
    want = px.softmax_cross_entropy(q, r, y, bias=b, reduction="none")
    assert torch.equal(px.softmax_cross_entropy(q2, r2, y, bias=b, reduction="none"), want)
    assert torch.equal(px.softmax_cross_entropy(q2, rt, y, bias=b, reduction="none"), want)
    odd = torch.empty(301, device="cuda")[1:]
    odd.copy_(b)
    assert torch.equal(px.softmax_cross_entropy(q, r, y, bias=odd, reduction="none"), want)
    _check_xent(px, q2, rt, y, odd)


@pytest.mark.parametrize("d", [1, 50, 65, 100])
def test_padding_is_neither_read_nor_written(px, d):
    """What lies behind the columns of a padded row, and behind the last row:
    NaN there reaches no result, and stays."""
    t, v = 140, 300
    q, r, y, b = _xent_case(t, v, d, torch.bfloat16, 35, bias=True)
    width = (d + 7) // 8 * 8 + 8

    def padded(a, rows):
        buf = torch.full((rows + 1, width), math.nan, dtype=a.dtype, device="cuda")
        buf[:rows, :d] = a
        return buf, buf[:rows, :d]

    (qb, q2), (rb, r2) = padded(q, t), padded(r, v)
    _check_xent(px, q2, r2, y, b)
    # The gradients into padded arrays, through the C ABI.
    lib, L = px._lib.load(), px._lib
    loss, lse = torch.empty(t, device="cuda"), torch.empty(t, device="cuda")
    ws = torch.empty(max(lib.px_softmax_xent_workspace_bytes(0, t, v, d, k) for k in (0, 1)), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    common = (0, q2.data_ptr(), width, t, r2.data_ptr(), width, v, d, 2, y.data_ptr(), -100, 1.5, b.data_ptr())
    L.check(lib.px_softmax_xent_device(*common, 0, loss.data_ptr(), lse.data_ptr(), None, None, ws.data_ptr(), ws.numel(), stream))
    one = torch.ones(1, device="cuda")
    outs = [padded(torch.zeros_like(q), t), padded(torch.zeros_like(r), v)]
    L.check(lib.px_softmax_xent_backward_device(
        *common, loss.data_ptr(), lse.data_ptr(), one.data_ptr(), 0, None, outs[0][1].data_ptr(), width,
        outs[1][1].data_ptr(), width, ws.data_ptr(), ws.numel(), stream))
    q1, r1 = q.detach().requires_grad_(), r.detach().requires_grad_()
    want = torch.autograd.grad(px.softmax_cross_entropy(q1, r1, y, scale=1.5, bias=b, reduction="sum"), (q1, r1))
    for (buf, view), w, rows in zip(outs, want, (t, v)):
        assert torch.equal(view, w)
        assert buf[:, d:].isnan().all() and buf[rows].isnan().all()
    # Codes: padding that would change the sums.
    c1, s1, c2, s2, _ = _scores_case(t, v, d, 36, False)
    bufs = [torch.full((rows + 1, (d + 15) // 16 * 16 + 16), 99, dtype=torch.int8, device="cuda") for rows in (t, v)]
    for buf, c in zip(bufs, (c1, c2)):
        buf[:-1, :d] = c
    got = px.int8_scores(bufs[0][:-1, :d], s1, bufs[1][:-1, :d], s2)
    assert torch.equal(got, px.int8_scores(c1.contiguous(), s1, c2.contiguous(), s2))
    x, codes = torch.full((5, 40), math.nan, device="cuda"), torch.full((5, 48), 77, dtype=torch.int8, device="cuda")
    x[:, :33] = 1.0
    scales = torch.empty(5, device="cuda")
    L.check(lib.px_quantize_rows_device(0, x.data_ptr(), 0, 5, 33, 40, codes.data_ptr(), 48, scales.data_ptr(), stream))
    assert (codes[:, :33] == 127).all() and (codes[:, 33:] == 77).all() and (scales == np.float32(1) / np.float32(127)).all()


def test_softmax_confident_targets(px):
    # The target holds nearly the whole softmax: the loss is far below an fp32
    # step of the logits, which subtracting them would lose.
    d = 64
    q = torch.zeros(16, d, dtype=torch.bfloat16, device="cuda")
    r = torch.zeros(50, d, dtype=torch.bfloat16, device="cuda")
    for i in range(16):
        q[i, i] = r[i, i] = 4.0
    y = torch.arange(16, device="cuda")
    loss = px.softmax_cross_entropy(q, r, y, scale=1.5, reduction="none")
    want = math.log1p(49 * math.exp(-24.0))
    assert ((loss.double() - want).abs() <= want * (2.0 ** -21 + 30 * U + 8 * U * 24)).all()
    _check_xent(px, q, r, y, None)


def test_softmax_lowest_bias_leaves_rows_out(px):
    q, r, y, b = _xent_case(40, 300, 32, torch.bfloat16, 43, bias=True)
    q, r = q.requires_grad_(), r.requires_grad_()

    def step(bias):
        loss = px.softmax_cross_entropy(q, r, y, bias=bias, reduction="none")
        return (loss, *torch.autograd.grad(loss.sum(), (q, r)))

    want = step(b)
    out = b == -math.inf
    for lowest in (torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min, -3e31):
        assert all(torch.equal(x, w) for x, w in zip(step(b.masked_fill(out, lowest)), want))
    assert not want[2][out].any()


def test_softmax_common_offset_changes_nothing_much(px):
    # Biases far from zero but alike: the softmax is that of their differences,
    # to the accuracy of fp32 numbers of that size.
    q, r, y, b = _xent_case(40, 300, 32, torch.bfloat16, 44)
    off = torch.full((300,), -10_000.0, device="cuda")
    a = px.softmax_cross_entropy(q, r, y, bias=off, reduction="none").double()
    w = px.softmax_cross_entropy(q, r, y, reduction="none").double()
    # Logits of 14427 in log2 units have steps of 2^-10; three roundings.
    assert ((a - w).abs() <= 4 * 2.0 ** -10).all()


def test_softmax_rows_left_out(px):
    q, r, y, _ = _xent_case(6, 40, 32, torch.bfloat16, 41)
    y[:] = torch.arange(6)
    b = torch.zeros(40, device="cuda")
    b[2] = -math.inf  # query 2's target is left out
    loss = px.softmax_cross_entropy(q, r, y, bias=b, reduction="none")
    assert loss[2] == math.inf and loss[[0, 1, 3, 4, 5]].isfinite().all()
    # Nothing left: every target is out, and no probability anywhere.
    b[:] = -math.inf
    q, r = q.requires_grad_(), r.requires_grad_()
    loss = px.softmax_cross_entropy(q, r, y, bias=b, reduction="none")
    assert (loss == math.inf).all()
    loss.sum().backward()
    # Only the targets' own terms remain: G = -1 at the target.
    want = -r.detach().double()[y]
    _within(q.grad, want, want.abs() * 2.0 ** -7, "grad of queries")
    # Only the target left in: certain, loss 0.
    b[:] = -math.inf
    b[3] = 0.25
    loss = px.softmax_cross_entropy(q.detach(), r.detach(), torch.full_like(y, 3), bias=b, reduction="none")
    assert (loss == 0).all()


def test_softmax_targets_out_of_range(px):
    q, r, y, _ = _xent_case(4, 40, 32, torch.bfloat16, 51)
    y[1], y[2] = 40, -7
    q, r = q.requires_grad_(), r.requires_grad_()
    loss = px.softmax_cross_entropy(q, r, y, reduction="none")
    assert loss[[1, 2]].isnan().all() and loss[[0, 3]].isfinite().all()
    loss.sum().backward()
    assert (q.grad[[1, 2]] == 0).all() and r.grad.isfinite().all()
    # All ignored: a mean over nothing, and zero gradients of the sum.
    y[:] = -100
    assert px.softmax_cross_entropy(q.detach(), r.detach(), y).isnan()
    dq, dr = torch.autograd.grad(px.softmax_cross_entropy(q, r, y, reduction="sum"), (q, r))
    assert not dq.any() and not dr.any()
    # An ignore_index that is a row number.
    y[:] = torch.tensor([3, 5, 3, 9])
    loss = px.softmax_cross_entropy(q.detach(), r.detach(), y, ignore_index=3, reduction="none")
    assert (loss[[0, 2]] == 0).all() and (loss[[1, 3]] > 0).all()


def test_softmax_no_queries(px):
    q = torch.zeros(0, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    r = _rand(9, 16, seed=1, dtype=torch.bfloat16).requires_grad_()
    y = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert px.softmax_cross_entropy(q, r, y, reduction="none").shape == (0,)
    assert px.softmax_cross_entropy(q, r, y).isnan()
    loss = px.softmax_cross_entropy(q, r, y, reduction="sum")
    assert loss == 0
    loss.backward()
    assert r.grad.shape == r.shape and not r.grad.any()


def test_softmax_one_gradient_only(px):
    q, r, y, b = _xent_case(130, 300, 72, torch.float16, 61)
    q1, r1 = q.detach().requires_grad_(), r.detach().requires_grad_()
    dq, dr = torch.autograd.grad(px.softmax_cross_entropy(q1, r1, y), (q1, r1))
    assert torch.equal(torch.autograd.grad(px.softmax_cross_entropy(q1, r.detach(), y), q1)[0], dq)
    assert torch.equal(torch.autograd.grad(px.softmax_cross_entropy(q.detach(), r1, y), r1)[0], dr)


def test_softmax_gradient_against_differences(px):
    """The gradient against central differences of the loss in 64 bits along
    random directions, at the operands' values."""
    q, r, y, b = _xent_case(50, 400, 48, torch.bfloat16, 71, bias=True)
    q1, r1 = q.detach().requires_grad_(), r.detach().requires_grad_()
    dq, dr = torch.autograd.grad(px.softmax_cross_entropy(q1, r1, y, scale=1.5, bias=b, reduction="sum"), (q1, r1))

    def loss64(qq, rr):
        z = 1.5 * (qq @ rr.T) + b.double()
        return (torch.logsumexp(z, 1) - z.gather(1, y[:, None])[:, 0]).sum()

    _xent64.dtype = torch.bfloat16
    _, _, _, (_, bq), (_, br) = _xent64(q, r, y, 1.5, b, -100, torch.ones(50, device="cuda"))
    for k in range(4):
        uq, ur = _rand(50, 48, seed=80 + k).double(), _rand(400, 48, seed=90 + k).double()
        e = 1e-5
        num = (loss64(q.double() + e * uq, r.double() + e * ur) - loss64(q.double() - e * uq, r.double() - e * ur)) / (2 * e)
        got = (dq.double() * uq).sum() + (dr.double() * ur).sum()
        bound = (bq * uq.abs()).sum() + (br * ur.abs()).sum() + 1e-5
        assert abs(float(num - got)) <= float(bound)


def test_results_do_not_change_between_runs(px):
    q, r, y, b = _xent_case(500, 20_000, 96, torch.bfloat16, 101, bias=True, ignored=True)
    q, r = q.requires_grad_(), r.requires_grad_()
    first = None
    for _ in range(3):
        loss = px.softmax_cross_entropy(q, r, y, bias=b)
        got = (loss.detach(), *torch.autograd.grad(loss, (q, r)))
        first = first or got
        assert all(torch.equal(x, w) for x, w in zip(got, first))


# ---------------------------------------------------------------- streams, graphs, devices

def test_calls_in_a_row_see_what_the_last_one_wrote(px):
    # The same buffers with other values each time, with no wait between: each
    # kernel starts while the one before it ends.
    n, m, d = 20_000, 64, 128
    bases = [_rand(n, d, seed=80 + i) * 4.0 ** i for i in range(4)]
    q = _rand(m, d, seed=79)
    y = torch.arange(m, device="cuda")

    def step(base):
        codes, scales = px.quantize_rows(base)
        back = px.dequantize_rows(codes, scales)
        qc, qs = px.quantize_rows(q)
        scores = px.int8_scores(qc, qs, codes, scales)
        a, b = q.bfloat16().requires_grad_(), back.bfloat16().requires_grad_()
        loss = px.softmax_cross_entropy(a, b, y, scale=0.01)
        return (back, scores, loss.detach(), *torch.autograd.grad(loss, (a, b)))

    want = []
    for base in bases:
        want.append(step(base))
        torch.cuda.synchronize()
    for i in [1, 0, 3, 2] * 5:
        assert all(torch.equal(x, w) for x, w in zip(step(bases[i]), want[i]))
    # Half a scale, and two roundings (the scale's, the product's) of at most 127 scales.
    _within(want[2][0], bases[2].double(), (0.5 + 2 * 127 * 2 * U) * bases[2].abs().amax(1, keepdim=True).double() / 127)


def test_row_operators_on_other_streams(px):
    """Two streams at once, each with its own inputs, against the default
    stream's results."""
    cases = [_xent_case(200, 3000, 64, torch.bfloat16, 200 + k) for k in range(2)]
    codes = [_scores_case(100, 4000, 128, 300 + k, False)[:4] for k in range(2)]

    def step(k):
        q, r, y, _ = cases[k]
        q, r = q.detach().requires_grad_(), r.detach().requires_grad_()
        loss = px.softmax_cross_entropy(q, r, y)
        return (loss.detach(), *torch.autograd.grad(loss, (q, r)), px.int8_scores(*codes[k]), *px.quantize_rows(cases[k][1]))

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(step(k))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, w) for x, w in zip(a, b))


def test_row_operators_in_graphs(px):
    """Two captured graphs of one step each, replayed in turn on new inputs."""
    graphs = []
    for k in range(2):
        q, r, y, _ = _xent_case(150, 2000, 64, torch.bfloat16, 400 + k)
        q, r = q.detach().clone().requires_grad_(), r.detach().clone().requires_grad_()

        def step(q=q, r=r, y=y):
            loss = px.softmax_cross_entropy(q, r, y, scale=2.0)
            dq, dr = torch.autograd.grad(loss, (q, r))
            qc, qs = px.quantize_rows(q)
            rc, rs = px.quantize_rows(r)
            return loss.detach(), dq, dr, px.int8_scores(qc, qs, rc, rs)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, q, r, step, out))
    for round_ in range(3):
        for k, (graph, q, r, step, out) in enumerate(graphs):
            with torch.no_grad():
                q.copy_(_rand(*q.shape, seed=500 + 10 * round_ + k))
                r.copy_(_rand(*r.shape, seed=600 + 10 * round_ + k))
            graph.replay()
            got = [o.clone() for o in out]
            assert all(torch.equal(g, w) for g, w in zip(got, step()))


def test_first_calls_inside_a_capture():
    """A process whose first use of each operator is a graph capture."""
    code = """
import torch, proxima_b200 as px
q = torch.randn(70, 64, device='cuda').bfloat16().requires_grad_()
r = torch.randn(900, 64, device='cuda').bfloat16().requires_grad_()
y = torch.arange(70, device='cuda')
def step():
    loss = px.softmax_cross_entropy(q, r, y, reduction='sum')
    qc, qs = px.quantize_rows(q); rc, rs = px.quantize_rows(r)
    return (loss.detach(), *torch.autograd.grad(loss, (q, r)), px.int8_scores(qc, qs, rc, rs), px.dequantize_rows(qc, qs))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g.replay()
got = [o.clone() for o in out]
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print('captured')
"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_two_host_threads(px):
    import threading
    cases = [_xent_case(100, 5000, 48, torch.float16, 700 + k) for k in range(2)]

    def step(k):
        q, r, y, _ = cases[k]
        q, r = q.detach().requires_grad_(), r.detach().requires_grad_()
        loss = px.softmax_cross_entropy(q, r, y, reduction="sum")
        qc, qs = px.quantize_rows(q)
        rc, rs = px.quantize_rows(r)
        return [loss.detach(), *torch.autograd.grad(loss, (q, r)), px.int8_scores(qc, qs, rc, rs)]

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    failed = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = step(k)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                    failed.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(100)
    assert not failed and not any(th.is_alive() for th in threads)


def test_rows_of_the_same_tensor(px):
    # The queries are some of the rows themselves.
    x = (_rand(200, 40, seed=5) / 6).to(torch.bfloat16).requires_grad_()
    y = torch.arange(50, device="cuda") + 100
    loss = px.softmax_cross_entropy(x[:50], x, y, scale=2.0, reduction="sum")
    loss.backward()
    q, r = x.detach()[:50].clone().requires_grad_(), x.detach().clone().requires_grad_()
    dq, dr = torch.autograd.grad(px.softmax_cross_entropy(q, r, y, scale=2.0, reduction="sum"), (q, r))
    dr[:50] += dq
    assert torch.equal(x.grad, dr)


def test_rows_status(px):
    px.rows_status()


def test_training_then_scoring(px):
    """The operators as they are used together: a few steps of training over
    a base, then the trained rows cut to 8 bits and scored beside an index."""
    t, v, d = 64, 2000, 64
    rows = (_rand(v, d, seed=1) / 8).to(torch.bfloat16).requires_grad_()
    queries = (_rand(t, d, seed=2) / 8).to(torch.bfloat16).requires_grad_()
    y = torch.arange(t, device="cuda") * 7
    opt = torch.optim.SGD([rows, queries], lr=1.0)
    for _ in range(3):
        opt.zero_grad()
        px.softmax_cross_entropy(queries, rows, y, scale=4.0, reduction="sum").backward()
        assert rows.grad.isfinite().all() and queries.grad.isfinite().all()
        opt.step()
    r32, q32 = rows.detach().float(), queries.detach().float()
    rc, rs = px.quantize_rows(r32)
    qc, qs = px.quantize_rows(q32)
    scores = px.int8_scores(qc, qs, rc, rs)
    want = px.dequantize_rows(qc, qs).double() @ px.dequantize_rows(rc, rs).double().T
    mag = px.dequantize_rows(qc, qs).double().abs() @ px.dequantize_rows(rc, rs).double().abs().T
    _within(scores, want, 6 * U * mag, "scores")
    idx = px.FlatIndex(d, px.Metric.InnerProduct)
    idx.add(r32.cpu().numpy())
    _, best = idx.search_batch(q32.cpu().numpy(), k=1)
    top = scores.max(1).values.double().cpu().numpy()
    # |q.r - qhat.rhat| <= |q - qhat| |r| + |qhat| |r - rhat|.
    qh, rh = px.dequantize_rows(qc, qs), px.dequantize_rows(rc, rs)
    slack = ((q32 - qh).norm(dim=1) * r32.norm(dim=1).max() + qh.norm(dim=1) * (r32 - rh).norm(dim=1).max()).cpu().numpy()
    assert (np.abs(top - best[:, 0]) <= slack * 1.01 + 1e-5).all()
