"""The operators on embedding rows where they can go wrong: gradients that
cancel, gradients and batches that are not ordinary, calls from several
threads. Bounds as in test_rows_gpu.py, evaluated per output.
"""

import math

import pytest
import torch

from test_rows_gpu import (ACC, HALF, TINY, TYPES, U, _check_xent, _codes64, _rand, _scores64, _scores_bound, _scores_case,
                           _within, _xent_case)

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


# ---------------------------------------------------------------- gradients that cancel

def _gradients_of_exact_logits(q, r, y, b, scale):
    """Gradients of the summed loss in 64 bits and bounds on the kernels'
    errors, for operands whose dot products are exact in fp32 in any order, so
    that what is left is the rounding of G (and of the outputs)."""
    dtype = q.dtype
    q, r = q.detach().double(), r.detach().double()
    (t, _), v = q.shape, r.shape[0]
    s = scale * (q @ r.T)
    z = s if b is None else s + b.double()
    lse = torch.logsumexp(z, 1)
    p = torch.exp(z - lse[:, None])
    pick = torch.arange(t, device=q.device)
    G = p.clone()
    G[pick, y] = -torch.where(torch.arange(v, device=q.device) == y[:, None], 0.0, p).sum(1)
    # A logit in log2 units is a fused multiply and add: two roundings in its
    # factor, three in the bias, one of the result; the shift by lse and by the
    # gradient's factor (2^14 at most) has four, the lse itself six of its size:
    # together below 16u of the magnitudes' sum. Then the sum over the rows (a
    # chain of at most v / 64 + 200 additions) and two exponentials of 2^-22.
    size = s.abs().amax() + lse.abs().amax() + 16
    if b is not None:
        size = size + torch.where(b.isinf(), 0.0, b.double()).abs().amax()
    dp = 1.01 * (16 * U * size + 2 * 2.0 ** -22 + (v / 64 + 200) * U)
    # G: an entry above 2^-9 as the sum of two numbers of its type, of which the
    # second rounds what the first left, half a step of at most half a step of the
    # entry; others as one number. fp16 entries have steps of 2^-24 at a lift of
    # 2^14 above the largest gradient, here 1.
    held = torch.where(G.abs() > 1.001 * 2.0 ** -9, HALF[dtype] ** 2, HALF[dtype])
    dG = G.abs() * (1.01 * held + dp + 4 * U) + (2.0 ** -39 if dtype == torch.float16 else 0.0)
    terms = 2 * int((G != 0).sum(1).max()), 2 * int((G != 0).sum(0).max())
    dq, dr = scale * G @ r, scale * G.T @ q
    half = 1.01 * HALF[dtype] + 4 * U
    bq = scale * (dG + ACC * (terms[0] + 2) * G.abs()) @ r.abs() + half * dq.abs() + TINY[dtype]
    br = scale * (dG + ACC * (terms[1] + 2) * G.abs()).T @ q.abs() + half * dr.abs() + TINY[dtype]
    return (dq, bq), (dr, br)


def _check_gradients(px, q, r, y, b, scale):
    q, r = q.detach().requires_grad_(), r.detach().requires_grad_()
    got = torch.autograd.grad(px.softmax_cross_entropy(q, r, y, scale=scale, bias=b, reduction="sum"), (q, r))
    for x, (want, bound), name in zip(got, _gradients_of_exact_logits(q, r, y, b, scale), ("queries", "rows")):
        _within(x, want, bound, "grad of " + name)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,v,d", [(1, 2, 64), (40, 300, 64), (200, 5000, 200), (33, 66, 520), (70, 1000, 19), (300, 260_009, 64)])
@pytest.mark.parametrize("behind", [0.0, 7.0])
def test_softmax_hard_negatives(px, dtype, t, v, d, behind):
    # Each query is its own row, and one other row differs from that in one
    # place by a little: both hold about half of the softmax (or, the target
    # being behind, the other nearly all), and in all other places their parts of
    # dq cancel. The values are whole sixteenths.
    g = torch.Generator(device="cuda").manual_seed(t + v + d)
    r = torch.randint(-16, 17, (v, d), device="cuda", generator=g).double() / 16
    order = torch.randperm(v, device="cuda", generator=g)
    y, near = order[:t], order[t:2 * t]
    r[near] = r[y]
    place = torch.randint(0, d, (t,), device="cuda", generator=g)
    r[near, place] += torch.where(r[y, place] > 0, -1, 1) * torch.randint(1, 5, (t,), device="cuda", generator=g) / 16
    q = r[y]
    scale = 2.0 ** round(math.log2(24 / float(q.square().sum(1).mean())))
    b = torch.full((v,), -24.0, device="cuda")
    b[order[:2 * t]] = 0.0
    b[y] = -behind
    unit = 8 * ((d + 7) // 8)
    qx, rx = (torch.zeros(n, unit, dtype=dtype, device="cuda")[:, :d] for n in (t, v))
    _check_gradients(px, qx.copy_(q), rx.copy_(r), y, b, scale)


@pytest.mark.parametrize("dtype,mine,others", [(torch.bfloat16, 25, 9), (torch.bfloat16, 9, 25), (torch.float16, 32, 6), (torch.float16, 6, 32)])
@pytest.mark.parametrize("v", [2, 700])
def test_softmax_rows_with_many_queries(px, dtype, mine, others, v):
    # All queries alike, of two rows that hold the softmax between them: `mine`
    # queries have the first as their target and `others` the second, in the
    # first's share of the softmax, so both rows' gradients are nearly zero. An
    # entry's rounding is the same for all queries of a kind.
    t, d = mine + others, 40
    q = _rand(1, d, seed=3).mul(4).round().div(4).expand(t, d).to(dtype)
    r = _rand(v, d, seed=4).mul(4).round().div(4).to(dtype)
    r[1] = r[0]
    b = torch.full((v,), -math.inf, device="cuda")
    b[0], b[1] = math.log(mine / others), 0.0
    y = (torch.arange(t, device="cuda") >= mine).long()
    _check_gradients(px, q, r, y, b, 0.5)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,v,d", [(33, 64, 24), (40, 300, 64), (257, 700, 200), (520, 900, 390), (1000, 300, 32), (300, 230_009, 16),
                                   (150_000, 1100, 16)])
def test_softmax_large_entries_anywhere(px, dtype, t, v, d):
    # Queries from certain of their target to far from it, in no order, so that
    # entries of all sizes, and blocks with and without large ones, meet in all
    # slices of the products.
    q, r, y, _ = _xent_case(t, v, d, dtype, t + v)
    g = torch.Generator(device="cuda").manual_seed(t)
    sharp = torch.rand(t, device="cuda", generator=g) < 0.3
    with torch.no_grad():
        q[sharp] = (0.5 * q + 3.0 / d * r[y])[sharp]
    b = torch.where(torch.rand(v, device="cuda", generator=g) < 0.01, 6.0, 0.0)
    _check_xent(px, q, r, y, None, scale=2.0)
    _check_xent(px, q, r, y, b, scale=0.5, weights=torch.linspace(-1, 1, t, device="cuda"))


# ---------------------------------------------------------------- batches and gradients out of the ordinary

@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,v,d", [(4, 40, 32), (300, 2000, 100), (70, 90, 600), (300, 520_009, 16)])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_softmax_all_queries_ignored(px, dtype, t, v, d, reduction):
    # A batch of padding: the mean over nothing is NaN, and nobody's gradient.
    q, r, y, b = _xent_case(t, v, d, dtype, 5, bias=True)
    y.fill_(-100)
    q, r = q.requires_grad_(), r.requires_grad_()
    loss = px.softmax_cross_entropy(q, r, y, bias=b, reduction=reduction)
    assert loss.isnan() if reduction == "mean" else not loss.any()
    for x in torch.autograd.grad(loss.sum(), (q, r)):
        assert torch.equal(x, torch.zeros_like(x))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,v,d", [(1, 40, 32), (70, 300, 64), (300, 5000, 100)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_softmax_gradients_that_are_not_finite(px, dtype, t, v, d, bad):
    # One query's gradient is no number: its row of dq, and all of dr, which it
    # has a part in; the other queries' rows are as without it.
    q, r, y, _ = _xent_case(t, v, d, dtype, 6)
    q, r = q.requires_grad_(), r.requires_grad_()

    def gradients(w, targets=y):
        loss = px.softmax_cross_entropy(q, r, targets, reduction="none")
        return torch.autograd.grad(loss, (q, r), grad_outputs=w)

    w = torch.linspace(0.5, 2, t, device="cuda")
    w[t // 2] = 0.0
    want = gradients(w)
    w[t // 2] = bad
    dq, dr = gradients(w)
    others = torch.arange(t, device="cuda") != t // 2
    assert torch.equal(dq[others], want[0][others])
    assert not dq[t // 2].isfinite().any() and not dr.isfinite().any()
    # An ignored query's counts for nothing, whatever it is.
    targets = y.clone()
    targets[t // 2] = -100
    dq, dr = gradients(w, targets)
    assert torch.equal(dq, want[0]) and torch.equal(dr, want[1])
    # The gradient of a sum, and a batch with no query to count.
    loss = px.softmax_cross_entropy(q, r, y, reduction="sum")
    for x in torch.autograd.grad(loss * bad, (q, r)):
        assert not x.isfinite().any()
    loss = px.softmax_cross_entropy(q, r, torch.full_like(y, -100), reduction="sum")
    for x in torch.autograd.grad(loss, (q, r), grad_outputs=torch.tensor(bad, device="cuda")):
        assert torch.equal(x, torch.zeros_like(x))


# ---------------------------------------------------------------- several threads

def _in_threads(work, count, rounds):
    """work(k) on `count` threads with a stream each, `rounds` times; an
    exception in any of them is raised here."""
    import threading

    done, failed, start = [0] * count, [], threading.Barrier(count)

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(60)
                for _ in range(rounds):
                    work(k)
                    done[k] += 1
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(k,), daemon=True) for k in range(count)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(100)
    if failed:
        raise failed[0]
    assert done == [rounds] * count


def test_threads_with_scores_of_different_shapes(px):
    # Launches of one kernel that ask for different amounts of shared memory,
    # close behind one another: the C ABI's calls alone, their arguments made
    # before.
    import sys

    lib, n = px._lib.load(), 64
    shapes = [(1, 128), (256, 768), (1, 128), (256, 768), (64, 1024), (1, 128)]
    one, calls, outs = torch.ones(256, device="cuda"), [], []
    for m, d in shapes:
        q, x = (torch.full((rows, d), 1, dtype=torch.int8, device="cuda") for rows in (m, n))
        out, stream = torch.zeros(m, n, device="cuda"), torch.cuda.Stream()
        outs.append((out, q, x, stream))
        calls.append((0, q.data_ptr(), d, one.data_ptr(), m, x.data_ptr(), d, one.data_ptr(), n, d, None, 0, out.data_ptr(), n,
                      stream.cuda_stream))
    torch.cuda.synchronize()

    def work(k):
        f, args = lib.px_int8_scores_device, calls[k]
        for _ in range(15_000):
            status = f(*args)
            if status:
                px._lib.check(status)

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    try:
        _in_threads(work, len(shapes), 1)
    finally:
        sys.setswitchinterval(interval)
        torch.cuda.synchronize()
    for (m, d), (out, *_) in zip(shapes, outs):
        assert (out == d).all()


def test_threads_with_steps_of_different_shapes(px):
    # Each thread its own operands, types and pieces; all results as alone.
    shapes = [(100, 5000, 48, torch.float16), (300, 900, 200, torch.bfloat16), (7, 20_000, 16, torch.bfloat16)]
    cases = [_xent_case(t, v, d, dtype, 700 + k) for k, (t, v, d, dtype) in enumerate(shapes)]

    def step(k):
        q, r, y, _ = cases[k]
        q, r = q.detach().requires_grad_(), r.detach().requires_grad_()
        loss = px.softmax_cross_entropy(q, r, y, reduction="sum")
        return [loss.detach(), *torch.autograd.grad(loss, (q, r)), *px.quantize_rows(r.detach())]

    want = [step(k) for k in range(len(shapes))]
    torch.cuda.synchronize()

    def work(k):
        got = step(k)
        torch.cuda.current_stream().synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[k]))

    _in_threads(work, len(shapes), 30)


# ---------------------------------------------------------------- scores

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [256, 301])
@pytest.mark.parametrize("small,large", [(2.0 ** -70, 2.0 ** -65), (2.0 ** -100, 2.0 ** -40), (2.0 ** 80, 2.0 ** -120)])
def test_int8_scores_of_scales_far_from_one(px, dtype, n, small, large):
    # Scores within fp32's range whose two scales' product is below its normal
    # numbers, or whose scales lie far apart.
    q, qs, x, xs, _ = _scores_case(40, n, 500, 3, False)
    for a, b in ((small, large), (large, small)):
        if a * 2 ** 23 > 2.0 ** 127:
            continue
        want = _scores64(q, qs * a, x, xs * b, None)
        _within(px.int8_scores(q, qs * a, x, xs * b, dtype=dtype), want, _scores_bound(want, None, dtype) + TINY[torch.float32])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [256, 301])
def test_int8_scores_of_zero_sums(px, dtype, n):
    # Rows at right angles, and rows of zeros, score 0 whatever their lengths.
    q = torch.zeros(33, 64, dtype=torch.int8, device="cuda")
    x = torch.zeros(n, 64, dtype=torch.int8, device="cuda")
    q[:, 0], x[1:, 1] = 127, 127
    qs, xs = torch.full((33,), 1e25, device="cuda"), torch.full((n,), 1e25, device="cuda")
    b = torch.arange(n, device="cuda") % 100 + 0.5
    assert not px.int8_scores(q, qs, x, xs, dtype=dtype).any()
    assert torch.equal(px.int8_scores(q, qs, x, xs, bias=b, dtype=dtype), b.to(dtype).expand(33, n))


# ---------------------------------------------------------------- derivatives that do not exist

def test_derivatives_do_not_vanish(px):
    """Where an operator has no derivative, asking for one raises; nothing
    comes back as if the derivative were zero."""
    from torch.autograd import forward_ad

    x, codes = _rand(5, 32, seed=1), torch.ones(5, 32, dtype=torch.int8, device="cuda")
    scales, bias = torch.ones(5, device="cuda"), torch.zeros(5, device="cuda")
    q, r, y, _ = _xent_case(4, 9, 32, torch.bfloat16, 2)
    uses = {
        "quantize_rows": [lambda a: px.quantize_rows(a)[1], x],
        "dequantize_rows": [lambda a: px.dequantize_rows(codes, a), scales],
        "int8_scores": [lambda a: px.int8_scores(codes, a, codes, scales), scales],
        "int8_scores rows": [lambda a: px.int8_scores(codes, scales, codes, a), scales],
        "int8_scores bias": [lambda a: px.int8_scores(codes, scales, codes, scales, bias=a), bias],
    }
    for name, (use, a) in uses.items():
        want = use(a)
        got = use(a.clone().requires_grad_())
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match=f"{name.split()[0]} has no derivative"):
            got.sum().backward()
        with torch.no_grad():
            assert not use(a.clone().requires_grad_()).requires_grad
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError):
                use(forward_ad.make_dual(a.clone(), torch.ones_like(a)))
            assert torch.equal(use(a), want)
    out = torch.empty(5, 5, device="cuda")
    with pytest.raises(ValueError, match="out cannot be given"):
        px.int8_scores(codes, scales, codes, scales, bias=bias.clone().requires_grad_(), out=out)
    with torch.no_grad():
        assert px.int8_scores(codes, scales, codes, scales, bias=bias.clone().requires_grad_(), out=out) is out
    # The loss has a backward derivative only.
    loss = px.softmax_cross_entropy(q, r, y)
    with forward_ad.dual_level():
        b = torch.zeros(9, device="cuda")
        for args, kw in (((forward_ad.make_dual(q, q), r, y), {}), ((q, forward_ad.make_dual(r, r), y), {}),
                         ((q, r, y), {"bias": forward_ad.make_dual(b, b)})):
            with pytest.raises(NotImplementedError):
                px.softmax_cross_entropy(*args, **kw)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                px.softmax_cross_entropy(*args, **kw)
        assert torch.equal(px.softmax_cross_entropy(q, r, y), loss)


@pytest.mark.filterwarnings("ignore")
def test_row_operators_in_compiled_functions(px):
    # A compiled function runs the operators between its graphs.
    import torch._dynamo

    q, r, y, b = _xent_case(20, 300, 40, torch.bfloat16, 9, bias=True)

    def step(q, r):
        loss = px.softmax_cross_entropy(q * 0.5, r, y, scale=2.0, bias=b) * 3
        codes, scales = px.quantize_rows(r.detach().float() + 0.0)
        qc, qs = px.quantize_rows(q.detach() * 2)
        return loss, px.int8_scores(qc, qs, codes, scales) + 1, px.dequantize_rows(codes, scales * 2)

    def all_of(f):
        a, c = q.detach().clone().requires_grad_(), r.detach().clone().requires_grad_()
        loss, *rest = f(a, c)
        return [loss.detach(), *torch.autograd.grad(loss, (a, c)), *rest]

    want = all_of(step)
    torch._dynamo.reset()
    got = all_of(torch.compile(step, backend="eager"))
    assert all(torch.equal(x, w) for x, w in zip(got, want))


@pytest.mark.parametrize("scale", [2.0 ** 126, 2.0 ** -140])
def test_softmax_scales_at_the_ends(px, scale):
    q, r, y, _ = _xent_case(3, 20, 16, torch.bfloat16, 3)
    with torch.no_grad():
        q.zero_()  # logits of zero, whatever the scale
    loss = px.softmax_cross_entropy(q, r, y, scale=scale, reduction="none")
    assert ((loss.double() - math.log(20)).abs() <= 1e-5).all()
    for large in (2.0 ** 127, 1e39, 1e300):
        with pytest.raises(ValueError, match="scale must be below"):
            px.softmax_cross_entropy(q, r, y, scale=large)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1025, 2048, 5000])
def test_quantize_long_strided_rows(px, dtype, d):
    # Rows longer than a group's registers hold, with something between them:
    # values on and beside halves of the scale, zeros, infinities, NaN at the end.
    s = torch.tensor([1.0, 0.375, 2.0 ** -12], dtype=torch.float64)
    at = (torch.arange(d, dtype=torch.float64) % 253 - 126.5)
    x = torch.full((9, d + 40), math.nan, dtype=torch.float64)
    x[:3, :d] = s[:, None] * at
    x[3:6, :d] = torch.nextafter((s[:, None] * at).to(dtype), torch.full((3, d), 300.0, dtype=dtype)).double()
    x[:6, d - 1] = torch.cat([s, s]) * 127
    x[6:, :d] = 0.0
    x[7, 3], x[8, 5] = math.inf, 1.0
    x[8, d - 1] = math.nan
    x = x.to(dtype).cuda()[:, :d]
    codes, scales = px.quantize_rows(x)
    assert scales[6] == 0 and scales[7:].isnan().all() and not codes[6:].any()
    want, want_scales = _codes64(x[:6])
    assert torch.equal(scales[:6], want_scales) and torch.equal(codes[:6], want)
