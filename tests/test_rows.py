"""Argument checks of the operators on embedding rows, without a GPU: the C
ABI's run before any device work, the Python layer's before the library is
called."""

import ctypes
import math

import pytest
import torch

VP = ctypes.c_void_p


@pytest.fixture
def lib(px):
    return px._lib.load()


def _refused(px, status, code, text):
    assert status == code, (status, px._lib.last_error())
    assert text in px._lib.last_error()


def test_quantize_arguments(px, lib):
    L = px._lib
    f = lib.px_quantize_rows_device
    _refused(px, f(0, VP(16), 0, 4, 0, 8, VP(16), 16, VP(16), None), L.PX_EINVAL, "dim must be > 0")
    _refused(px, f(0, VP(16), 0, -1, 8, 8, VP(16), 16, VP(16), None), L.PX_EINVAL, "n must be >= 0")
    _refused(px, f(0, VP(16), 0, 1 << 31, 8, 8, VP(16), 16, VP(16), None), L.PX_EUNSUPPORTED, "2^31")
    _refused(px, f(0, VP(16), 3, 4, 8, 8, VP(16), 16, VP(16), None), L.PX_EINVAL, "type")
    _refused(px, f(0, VP(16), 0, 4, 8, 7, VP(16), 16, VP(16), None), L.PX_EINVAL, "stride")
    _refused(px, f(0, None, 0, 4, 8, 8, VP(16), 16, VP(16), None), L.PX_EINVAL, "null buffer")
    _refused(px, f(0, VP(18), 0, 4, 8, 8, VP(16), 16, VP(16), None), L.PX_EINVAL, "x: misaligned")
    _refused(px, f(0, VP(17), 2, 4, 8, 8, VP(16), 16, VP(16), None), L.PX_EINVAL, "x: misaligned")
    _refused(px, f(0, VP(16), 0, 4, 8, 8, VP(16), 16, VP(18), None), L.PX_EINVAL, "scales: misaligned")
    assert f(0, None, 0, 0, 8, 8, None, 16, None, None) == L.PX_OK
    g = lib.px_dequantize_rows_device
    _refused(px, g(0, VP(16), 16, VP(16), 4, 8, 5, VP(16), 8, None), L.PX_EINVAL, "type")
    _refused(px, g(0, VP(16), 16, VP(16), 4, 8, 0, VP(16), 7, None), L.PX_EINVAL, "stride")
    _refused(px, g(0, VP(16), 16, None, 4, 8, 0, VP(16), 8, None), L.PX_EINVAL, "null buffer")


def test_scores_arguments(px, lib):
    L = px._lib

    def f(q=16, ldq=16, m=4, x=16, ldx=16, n=5, dim=8, type_=0, out=16, ldo=5):
        return lib.px_int8_scores_device(0, VP(q), ldq, VP(16), m, VP(x), ldx, VP(16), n, dim, None, type_, VP(out),
                                         ldo, None)

    _refused(px, f(q=24), L.PX_EINVAL, "queries: rows must start on 16-byte boundaries")
    _refused(px, f(ldx=24), L.PX_EINVAL, "rows: rows must start on 16-byte boundaries")
    _refused(px, f(dim=17), L.PX_EINVAL, "the row stride is less than dim")
    _refused(px, f(dim=131072, ldq=131072, ldx=131072), L.PX_EUNSUPPORTED, "pass 32 bits")
    _refused(px, f(ldo=4), L.PX_EINVAL, "less than n")
    _refused(px, f(out=18), L.PX_EINVAL, "misaligned")
    _refused(px, f(type_=9), L.PX_EINVAL, "type")
    _refused(px, f(m=1 << 30, n=1 << 30, ldo=1 << 30), L.PX_EUNSUPPORTED, "m * n is too large")
    assert f(m=0) == L.PX_OK and f(n=0, ldo=0) == L.PX_OK


def test_softmax_arguments(px, lib):
    L = px._lib

    def f(t=4, v=6, dim=8, q=16, ldq=8, type_=2, scale=1.0, bias=None, reduction=0, total=16, targets=16):
        return lib.px_softmax_xent_device(0, VP(q), ldq, t, VP(16), 8, v, dim, type_, VP(targets), -100, scale,
                                          VP(bias), reduction, VP(16), VP(16), VP(total), VP(16), None, 0, None)

    _refused(px, f(dim=0), L.PX_EINVAL, "dim must be > 0")
    _refused(px, f(v=0), L.PX_EINVAL, "at least one base row")
    _refused(px, f(type_=0), L.PX_EUNSUPPORTED, "PX_F16 or PX_BF16")
    _refused(px, f(type_=7), L.PX_EINVAL, "PX_F16 or PX_BF16")
    for scale in (0.0, -1.0, math.inf, math.nan):
        _refused(px, f(scale=scale), L.PX_EINVAL, "scale must be positive and finite")
    _refused(px, f(q=8), L.PX_EINVAL, "16-byte boundaries")
    _refused(px, f(ldq=12), L.PX_EINVAL, "16-byte boundaries")
    _refused(px, f(targets=None), L.PX_EINVAL, "null buffer")
    _refused(px, f(bias=8), L.PX_EINVAL, "bias must be 16-byte aligned")
    _refused(px, f(reduction=3), L.PX_EINVAL, "reduction")
    _refused(px, f(reduction=2, total=None), L.PX_EINVAL, "null buffer")
    _refused(px, f(targets=20), L.PX_EINVAL, "targets: misaligned")
    _refused(px, f(t=1 << 30, v=1 << 30), L.PX_EUNSUPPORTED, "t * v is too large")
    assert f(t=0) == L.PX_OK

    def g(t=4, stride=0, grad=16, gq=16, ldgq=8):
        return lib.px_softmax_xent_backward_device(0, VP(16), 8, t, VP(16), 8, 6, 8, 2, VP(16), -100, 1.0, None, VP(16),
                                                   VP(16), VP(grad), stride, None, VP(gq), ldgq, None, 8, None, 0, None)

    _refused(px, g(stride=2), L.PX_EINVAL, "grad_stride")
    _refused(px, g(grad=None), L.PX_EINVAL, "null buffer")
    _refused(px, g(ldgq=7), L.PX_EINVAL, "less than dim")
    _refused(px, g(gq=17), L.PX_EINVAL, "misaligned")
    assert g(t=0) == L.PX_OK and g(gq=None) == L.PX_OK


def test_softmax_workspace(px, lib):
    """The workspace never grows as the logits do: at most 256 MB (or 1024
    columns) of the gradient's 16-bit matrix beside fp32 sums of the queries'
    size, 24 bytes per column, and 16 bytes per query and split."""
    f = lib.px_softmax_xent_workspace_bytes
    for t, v, d in ((1, 1, 1), (1, 10_000_000, 768), (1000, 100_000, 384), (8192, 8192, 768), (10_000, 1_000_000, 128),
                    (200_000, 1000, 64)):
        fwd, bwd = f(0, t, v, d, 0), f(0, t, v, d, 1)
        m_tiles, n_tiles = -(-t // 256), -(-d // 256)
        piece = max(2 * 1024 * t, 256 << 20)
        slabs = max(148, m_tiles * n_tiles) * 256 * 256 * 4
        assert 0 < fwd <= t * (16 * 4 * 148 + 4) + 1024
        lists = 24 * max(piece // (2 * t), 1024)
        assert 0 < bwd <= piece + slabs + lists + 4 * t + 4096, (t, v, d, bwd)
    assert f(0, 0, 10, 8, 1) == 0 and f(0, 10, 0, 8, 0) == 0 and f(0, -1, 10, 8, 0) == 0


def test_no_gpu_is_reported(px, lib):
    if lib.px_device_count() > 0:
        pytest.skip("a GPU is present")
    L = px._lib
    st = lib.px_quantize_rows_device(0, VP(16), 0, 4, 8, 8, VP(16), 16, VP(16), None)
    _refused(px, st, L.PX_ECUDA, "no CUDA device")
    _refused(px, lib.px_rows_status_device(0, None), L.PX_ECUDA, "no CUDA device")


def test_python_layer_refuses_cpu_tensors(px):
    x = torch.zeros(4, 8)
    with pytest.raises(TypeError, match="argument 'x': expected a 2-d CUDA tensor of float32, float16, bfloat16"):
        px.quantize_rows(x)
    with pytest.raises(TypeError, match="argument 'codes'"):
        px.dequantize_rows(x.to(torch.int8), x[:, 0])
    with pytest.raises(TypeError, match="argument 'q_codes'"):
        px.int8_scores(x, x[:, 0], x, x[:, 0])
    with pytest.raises(TypeError, match="argument 'queries': expected a 2-d CUDA tensor of float16, bfloat16"):
        px.softmax_cross_entropy(x, x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(AttributeError):
        px.no_such_operator


@pytest.mark.gpu
def test_python_layer_refusals(px):
    def z(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    i8, b16 = torch.int8, torch.bfloat16
    with pytest.raises(TypeError):
        px.quantize_rows(z(4))
    with pytest.raises(TypeError):
        px.quantize_rows(z(4, 8, dtype=torch.float64))
    with pytest.raises(ValueError, match="dim must be > 0"):
        px.quantize_rows(z(4, 0))
    with pytest.raises(ValueError, match="scales length"):
        px.dequantize_rows(z(4, 8, dtype=i8), z(3))
    with pytest.raises(TypeError, match="dtype"):
        px.dequantize_rows(z(4, 8, dtype=i8), z(4), dtype=torch.float64)
    q, x = z(2, 8, dtype=i8), z(4, 8, dtype=i8)
    with pytest.raises(ValueError, match="does not match row dim"):
        px.int8_scores(q, z(2), z(4, 9, dtype=i8), z(4))
    with pytest.raises(ValueError, match="q_scales length"):
        px.int8_scores(q, z(3), x, z(4))
    with pytest.raises(ValueError, match="bias length"):
        px.int8_scores(q, z(2), x, z(4), bias=z(5))
    with pytest.raises(ValueError, match="out has shape"):
        px.int8_scores(q, z(2), x, z(4), out=z(2, 5))
    with pytest.raises(TypeError, match="argument 'out'"):
        px.int8_scores(q, z(2), x, z(4), out=z(2, 4, dtype=b16))
    with pytest.raises(ValueError, match="do not overlap"):
        px.int8_scores(q, z(2), x, z(4), out=z(1, 4).expand(2, 4))
    with pytest.raises(ValueError, match="exceeds 131071"):
        px.int8_scores(z(1, 131072, dtype=i8), z(1), z(1, 131072, dtype=i8), z(1))
    assert px.int8_scores(z(0, 8, dtype=i8), z(0), x, z(4)).shape == (0, 4)
    assert px.int8_scores(q, z(2), z(0, 8, dtype=i8), z(0)).shape == (2, 0)
    c, s = px.quantize_rows(z(0, 8))
    assert c.shape == (0, 8) and s.shape == (0,) and px.dequantize_rows(c, s).shape == (0, 8)
    qq, rr, y = z(2, 8, dtype=b16), z(4, 8, dtype=b16), z(2, dtype=torch.int64)
    with pytest.raises(TypeError, match="argument 'rows'"):
        px.softmax_cross_entropy(qq, z(4, 8, dtype=torch.float16), y)
    with pytest.raises(TypeError, match="argument 'targets'"):
        px.softmax_cross_entropy(qq, rr, y.int())
    with pytest.raises(ValueError, match="targets length"):
        px.softmax_cross_entropy(qq, rr, z(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="at least one base row"):
        px.softmax_cross_entropy(qq, z(0, 8, dtype=b16), y)
    with pytest.raises(ValueError, match="ignore_index"):
        px.softmax_cross_entropy(qq, rr, y, ignore_index=2 ** 64)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            px.softmax_cross_entropy(qq, rr, y, scale=scale)
    with pytest.raises(ValueError, match="reduction"):
        px.softmax_cross_entropy(qq, rr, y, reduction="max")
    with pytest.raises(ValueError, match="bias has no gradient"):
        px.softmax_cross_entropy(qq, rr, y, bias=z(4).requires_grad_())
    with pytest.raises(ValueError, match="bias length"):
        px.softmax_cross_entropy(qq, rr, y, bias=z(5))
