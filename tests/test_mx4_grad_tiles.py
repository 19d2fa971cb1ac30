"""Every tile of the input's gradient, and blocks that walk over several tiles,
with whole numbers: every sum is exact in fp32."""

import math

import pytest
import torch

from mgproto_amd import ops
from mx4_oracle import GRID, values

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
TILES = [2, 3, 4, 5]        # forms: 256 x 256, 256 x 128, 128 x 128, 256 x 64


def _grid(*shape):
    return (GRID.cuda()[torch.randint(0, 8, shape, device='cuda')]
            * (torch.randint(0, 2, shape, device='cuda') * 2 - 1)).float()


@pytest.mark.parametrize('tile', TILES)
@pytest.mark.parametrize('M,K,N', [
    (1, 1, 1), (17, 129, 65), (130, 257, 131), (300, 200, 1000),
    (1100, 64, 1001), (513, 640, 384), (255, 70, 2048), (257, 65, 32),
    (70, 520, 5000)])
def test_every_tile_at_every_size(M, K, N, tile):
    ext = ops._native_or_die()
    w = _grid(N, K)
    g = torch.randint(-4, 5, (M, N), device='cuda')
    wq = ops.mx4_quantize(w)
    want = (g.double().cpu() @ values(w))
    for code, dtype in enumerate(DTYPES):
        base = torch.full((M * N + 3,), math.nan, dtype=dtype, device='cuda')
        for lo in (0, 3):                  # on 16 bytes, and not
            gd = base[lo:lo + M * N].view(M, N)
            gd.copy_(g)
            to = (code + lo) % 3
            dx, _, _ = ext.mx4_linear_backward(
                gd, wq.codes, wq.scales, None, None, K, to, -1, -1, tile)
            assert torch.equal(dx.cpu(), want.to(DTYPES[to])), (dtype, lo)
            base.fill_(math.nan)


# sums of 1, 2, 3 and 5 steps of 32 a part, whole and not; 1, 2 and 3 parts; more
# tiles than the 256 or 512 blocks that there are at most
@pytest.mark.parametrize('tile', TILES)
@pytest.mark.parametrize('N', [32, 64, 96, 160, 7, 33, 90, 155])
@pytest.mark.parametrize('dtype', DTYPES)
def test_more_tiles_than_blocks(tile, N, dtype):
    M, K = 66001, 261
    ext = ops._native_or_die()
    w = _grid(N, K)
    g = torch.randint(-4, 5, (M, N), device='cuda').to(dtype)
    wq = ops.mx4_quantize(w)
    want = g.float() @ wq.dequantize(torch.float32)
    for _ in range(3):
        dx, _, _ = ext.mx4_linear_backward(g, wq.codes, wq.scales, None, None,
                                           K, 0, -1, -1, tile)
        assert torch.equal(dx, want)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,K,N', [(15680, 2048, 96), (250883, 64, 64),
                                   (70001, 500, 40)])
def test_large_sizes_as_they_are_chosen(M, K, N, dtype):
    """Both products of a step whose tiles are more than the blocks."""
    x, w = _grid(M, K), _grid(N, K)
    # sums of up to 250883 products of at most 6 in halves: below 2^24 halves
    g = torch.zeros(M, N, device='cuda')
    g[torch.arange(M, device='cuda'),
      torch.randint(0, N, (M,), device='cuda')] = 1.0
    g[:, 0] = -1.0
    g = g.to(dtype)
    x.requires_grad_()
    w.requires_grad_()
    y = ops.mx4_linear(x.to(dtype), w)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    xv, wv = (ops.mx4_quantize(t.detach()).dequantize(torch.float32)
              for t in (x, w))
    assert torch.equal(y, (xv @ wv.t()).to(dtype))
    assert torch.equal(dx, (g.float() @ wv).to(dtype).float())
    assert torch.equal(dw, g.float().t() @ xv)


def test_forms_that_are_not_there():
    q = ops.mx4_quantize(torch.randn(8, 64, device='cuda'))
    for form in (-2, 6):
        with pytest.raises(ValueError, match='no form'):
            ops._native_or_die().mx4_linear_backward(
                torch.randn(4, 8, device='cuda'), q.codes, q.scales, None,
                None, 64, 0, -1, -1, form)
