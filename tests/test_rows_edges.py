"""What of the operators on embedding rows can be checked without a GPU
beyond their argument checks."""

import pytest
import torch


@pytest.mark.parametrize("t,v,d", [(1, 10_000_000, 64), (1, 100_000_000, 8), (65, 2_000_000, 64), (1000, 100_000, 384), (5000, 60_000, 128)])
def test_gradient_pieces_keep_their_bound(px, t, v, d):
    # A piece of the gradient's matrix is at most 256 MB or 512 columns, with the
    # queries padded to 64 and both 16-bit parts counted; beside it lie the fp32
    # sums of the queries' gradients (148 tiles of 256 x 256 at most here), a byte
    # per 32 queries and 64 columns, twice, and little else.
    need = px._lib.load().px_softmax_xent_workspace_bytes(0, t, v, d, 1)
    padded = (t + 63) // 64 * 64
    piece = max(256 << 20, 512 * 4 * padded)
    columns = piece // (4 * padded)
    parts = 2 * (columns // 64 + 4) * ((t + 255) // 256 * 8)
    assert 0 < need <= piece + 148 * 256 * 256 * 4 + parts + 4096


def test_operators_without_a_derivative_say_so():
    from torch.autograd import forward_ad

    from proxima_b200 import rows

    x = torch.ones(3, requires_grad=True)

    def call(a, b):
        return torch.ones(3, dtype=torch.int8), torch.ones(3)

    def use(a, b=None):
        return rows._NoDerivative.apply("op", call, a, b) if rows._wanted(a, b) else call(a, b)

    codes, scales = use(x)
    assert scales.requires_grad and not codes.requires_grad
    with pytest.raises(RuntimeError, match="op has no derivative"):
        scales.sum().backward()
    with pytest.raises(RuntimeError, match="op has no derivative"):
        torch.autograd.grad((scales * x).sum(), x)
    # Nothing asked for: the results as they are.
    with torch.no_grad():
        assert not rows._wanted(x) and not use(x)[1].requires_grad
    assert not rows._wanted(x.detach(), None) and not use(x.detach())[1].requires_grad
    with forward_ad.dual_level():
        plain = x.detach()
        dual = forward_ad.make_dual(plain, torch.ones(3))
        assert rows._wanted(None, dual) and not rows._wanted(plain, None)
        with torch.no_grad():
            assert rows._wanted(dual)
        with pytest.raises(NotImplementedError):
            use(dual)
        use(plain)
    assert not rows._wanted(plain)


def test_the_package_needs_no_torch():
    """A star import in a process that has no torch: the searches are there,
    and the operators on tensors say what they miss when they are first used."""
    import os
    import subprocess
    import sys

    code = """
import sys
sys.modules["torch"] = None  # importing it raises
from proxima_b200 import *
import proxima_b200
assert FlatIndex and PqIndex and Metric and PxError and "softmax_cross_entropy" in dir(proxima_b200)
try:
    proxima_b200.quantize_rows
except ImportError:
    print("no torch")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == "no torch", r.stderr[-2000:]


def test_traces_are_refused(px):
    from torch.fx.experimental.proxy_tensor import make_fx

    x, codes, y = torch.ones(3, 8), torch.ones(3, 8, dtype=torch.int8), torch.zeros(3, dtype=torch.int64)
    for name, use in (("quantize_rows", lambda a: px.quantize_rows(a)[1]),
                      ("dequantize_rows", lambda a: px.dequantize_rows(codes, a[:, 0])),
                      ("int8_scores", lambda a: px.int8_scores(codes, a[:, 0], codes, a[:, 0])),
                      ("softmax_cross_entropy", lambda a: px.softmax_cross_entropy(a, a, y))):
        for trace in (lambda: torch.jit.trace(use, x, check_trace=False), lambda: make_fx(use)(x)):
            with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
                trace()


def test_scales_whose_logits_would_not_be_numbers(px):
    import ctypes

    at = ctypes.c_void_p(16)
    for scale in (2.0 ** 127, 3.4e38):
        status = px._lib.load().px_softmax_xent_device(0, at, 8, 4, at, 8, 6, 8, 2, at, -100, scale, None, 0, at, at, at, at,
                                                       None, 0, None)
        assert status == px._lib.PX_EINVAL and "scale must be below 2^127" in px._lib.last_error()
