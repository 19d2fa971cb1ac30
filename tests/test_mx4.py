"""4-bit rows and their product on the CPU: the PyTorch form against the
definition in 64 bits, the gradients, the refusals."""

import math

import pytest
import torch

from mgproto_amd import ops
from mx4_oracle import GRID, assert_close, values

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,K', [(1, 1), (3, 32), (5, 33), (4, 128),
                                 (7, 300)])
def test_round_trip_is_the_definition(M, K, dtype):
    x = (torch.randn(M, K) * torch.exp(3 * torch.randn(M, K))).clamp(
        -6e4, 6e4).to(dtype)
    q = ops.mx4_quantize(x)
    assert q.shape == (M, K) and q.dtype == dtype
    codes, scales = q.parts()
    assert codes.shape == (M, -(-K // 32) * 16)
    assert scales.shape == (M, -(-K // 32))
    again = ops.MX4Tensor.from_parts(codes, scales, dtype)
    assert torch.equal(again.codes, q.codes)
    assert torch.equal(again.scales, q.scales)
    # element k is the nibble k & 1 of byte k / 2
    code = codes[M - 1, (K - 1) // 2] >> 4 * ((K - 1) & 1) & 7
    assert float(GRID[code.item()]) * 2.0 ** (int(scales[M - 1, -1]) - 127) \
        == float(q.dequantize()[M - 1, K - 1].abs())
    assert torch.equal(q.dequantize().double(), values(x))
    assert torch.equal(q.dequantize(torch.float32).double(), values(x))


def test_every_value_and_every_tie():
    mid = (GRID[1:] + GRID[:-1]) / 2
    row = torch.cat([GRID, mid, mid * (1 + 2 ** -20), mid * (1 - 2 ** -20),
                     torch.tensor([7.0, 7.9])]).float()
    row = torch.cat([row, -row])
    row = torch.nn.functional.pad(row, (0, -len(row) % 31)).view(-1, 31)
    x = torch.cat([row, torch.full((len(row), 1), 6.0)], dim=1)
    for e in (-100, -1, 0, 1, 100):
        q = ops.mx4_quantize(x * 2.0 ** e)
        assert torch.equal(q.dequantize().double(), values(x * 2.0 ** e))


def test_scales_at_the_ends():
    x = torch.zeros(6, 32)
    x[0, 0] = torch.finfo(torch.float32).max
    x[1, 0] = 2.0 ** -126                    # E would be -128
    x[2, 0] = 2.0 ** -149
    x[3, 0] = 1.0
    x[3, 1] = -0.0
    x[4, 5] = math.nan
    x[5, 5] = -math.inf
    q = ops.mx4_quantize(x)
    codes, scales = q.parts()
    assert scales[:, 0].tolist() == [252, 0, 0, 125, 255, 255]
    assert codes[4:].eq(0).all()
    assert q.scales[..., 1:].eq(0).all()          # behind the row
    v = q.dequantize()
    assert torch.equal(v[:4].double(), values(x)[:4])
    assert v[4:].isnan().all()


def test_leading_axes_strides_and_parts():
    x = torch.randn(2, 3, 64)
    q = ops.mx4_quantize(x)
    assert q.shape == (2, 3, 64) and q.codes.shape == (1, 6, 64)
    t = torch.randn(64, 5).t()               # rows not contiguous
    assert torch.equal(ops.mx4_quantize(t).dequantize(),
                       ops.mx4_quantize(t.contiguous()).dequantize())
    codes, scales = q.parts()
    assert codes.shape == (2, 3, 32) and scales.shape == (2, 3, 2)
    p = ops.MX4Tensor.from_parts(codes, scales, torch.float32)
    assert p.shape == (2, 3, 64)
    assert torch.equal(p.dequantize(), q.dequantize())
    assert ops.mx4_quantize(torch.zeros(0, 32)).dequantize().shape == (0, 32)
    assert ops.mx4_quantize(torch.zeros(4, 0)).dequantize().shape == (4, 0)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,K,N', [(1, 1, 1), (5, 33, 7), (16, 256, 40)])
def test_linear_and_its_gradients(M, K, N, dtype):
    x = torch.randn(M, K).to(dtype).requires_grad_()
    w = (torch.randn(N, K) / K ** 0.5).requires_grad_()
    b = torch.randn(N).requires_grad_()
    g = torch.randn(M, N).to(dtype)
    y = ops.mx4_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    xv, wv, g64 = values(x), values(w), g.double()
    assert_close(y, xv @ wv.t() + b.double(),
                 xv.abs() @ wv.abs().t() + b.double().abs(), K + 1)
    assert_close(dx, g64 @ wv, g64.abs() @ wv.abs(), N)
    assert_close(dw, g64.t() @ xv, g64.abs().t() @ xv.abs(), M)
    assert_close(db, g64.sum(0), g64.abs().sum(0), M)
    # a held weight gives the same result, and a gradient to x and bias
    held = ops.mx4_quantize(w)
    y2 = ops.mx4_linear(x, held, b)
    assert torch.equal(y2, y)
    dx2, db2 = torch.autograd.grad(y2, (x, b), g)
    assert torch.equal(dx2, dx) and torch.equal(db2, db)


def test_gradient_against_differences():
    # between values of the grid, with the block's maximum where it was, the
    # product is linear: the differences are the gradient
    M, K, N = 3, 64, 4
    x = GRID[torch.randint(0, 6, (M, K))].float()
    x[:, ::32] = 6.0
    w = GRID[torch.randint(0, 6, (N, K))].float()
    w[:, ::32] = -6.0
    g = torch.randn(M, N)
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(ops.mx4_linear(x, w), (x, w), g)
    loss = lambda a, b: float((ops.mx4_linear(a, b).double() * g).sum())  # noqa: E731
    with torch.no_grad():
        for m, k in [(0, 1), (1, 33), (2, 63)]:
            x2 = x.clone()
            x2[m, k] = 4.0 if x[m, k] < 2 else 0.5
            d = (loss(x2, w) - loss(x, w)) / float(x2[m, k] - x[m, k])
            assert d == pytest.approx(float(dx[m, k]), abs=1e-3)
        for n, k in [(0, 2), (3, 40)]:
            w2 = w.clone()
            w2[n, k] = 4.0 if w[n, k] < 2 else 0.5
            d = (loss(x, w2) - loss(x, w)) / float(w2[n, k] - w[n, k])
            assert d == pytest.approx(float(dw[n, k]), abs=1e-3)


def test_empty_sizes():
    for M, K, N in [(0, 32, 4), (3, 0, 4), (3, 32, 0)]:
        x = torch.randn(M, K, requires_grad=True)
        w = torch.randn(N, K, requires_grad=True)
        b = torch.randn(N, requires_grad=True)
        y = ops.mx4_linear(x, w, b)
        assert y.shape == (M, N)
        if K == 0:
            assert torch.equal(y, b.expand(M, N))
        grads = torch.autograd.grad(y.sum(), (x, w, b))
        assert [t.shape for t in grads] == [x.shape, w.shape, b.shape]


def test_refusals():
    x, w = torch.randn(4, 64), torch.randn(8, 64)
    q = ops.mx4_quantize(w)
    with pytest.raises(TypeError, match='float64'):
        ops.mx4_quantize(x.double())
    with pytest.raises(TypeError):
        ops.mx4_quantize(x.int())
    with pytest.raises(ValueError, match='number'):
        ops.mx4_quantize(torch.tensor(1.0))
    with pytest.raises(ValueError, match='do not match'):
        ops.mx4_linear(x[:, :32], q)
    with pytest.raises(ValueError, match='do not match'):
        ops.mx4_linear(x, w[0])
    with pytest.raises(ValueError, match='bias'):
        ops.mx4_linear(x, q, torch.zeros(7))
    with pytest.raises(TypeError, match='weight'):
        ops.mx4_linear(x, w.double())
    with pytest.raises(ValueError, match='weight on meta'):
        ops.mx4_linear(x, w.to('meta'))
    with pytest.raises(ValueError, match='8 rows of 129'):
        ops.MX4Tensor(q.codes, q.scales, (8, 129))
    with pytest.raises(ValueError, match='7 rows of 64'):
        ops.MX4Tensor(q.codes, q.scales, (7, 64))
    with pytest.raises(TypeError):
        ops.MX4Tensor(q.codes.int(), q.scales, (8, 64))
    with pytest.raises(ValueError, match='blocks of 32'):
        ops.MX4Tensor.from_parts(*(t[:, :1] for t in q.parts()))
    with pytest.raises(TypeError, match='float64'):
        q.dequantize(torch.float64)
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(ops.mx4_linear(xg, q).sum(), xg,
                                create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), xg)
