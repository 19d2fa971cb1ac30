"""4-bit rows and their product on the GPU against the definition in 64 bits."""

import math

import pytest
import torch

from mgproto_amd import ops
from mx4_oracle import GRID, assert_close, values

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _same(q, ref):
    assert torch.equal(q.codes.cpu(), ref.codes)
    assert torch.equal(q.scales.cpu(), ref.scales)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,K', [(1, 1), (3, 32), (5, 33), (64, 127),
                                 (4, 128), (7, 300), (1000, 1024),
                                 (333, 1003)])
def test_quantize(M, K, dtype):
    x = (torch.randn(M, K) * torch.exp(3 * torch.randn(M, K))).clamp(
        -6e4, 6e4).to(dtype)
    x[M // 2, K // 2] = math.inf
    x[M - 1, 0] = math.nan
    q = ops.mx4_quantize(x.cuda())
    _same(q, ops.mx4_quantize(x))
    for t in DTYPES:
        want = ops.mx4_quantize(x).dequantize(t)
        got = q.dequantize(t).cpu()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    ok = ~want.isnan()
    assert torch.equal(q.dequantize(torch.float32).cpu().double()[ok],
                       values(x)[ok])


def test_quantize_every_value_at_every_scale():
    mid = (GRID[1:] + GRID[:-1]) / 2
    row = torch.cat([GRID, mid, mid * (1 + 2 ** -20), mid * (1 - 2 ** -20)])
    row = torch.cat([row, -row])
    row = torch.nn.functional.pad(row, (0, -len(row) % 31)).view(-1, 31)
    x = torch.cat([row, torch.full((len(row), 1), 6.0)], dim=1).double()
    for e in (-149, -140, -130, -127, -126, -125, -60, 0, 60, 124, 125):
        xe = (x * 2.0 ** e).float()
        _same(ops.mx4_quantize(xe.cuda()), ops.mx4_quantize(xe))
        xe = xe.bfloat16()
        _same(ops.mx4_quantize(xe.cuda()), ops.mx4_quantize(xe))
    for e in (-24, -14, 0, 13):
        xe = (x * 2.0 ** e).half()
        _same(ops.mx4_quantize(xe.cuda()), ops.mx4_quantize(xe))


@pytest.mark.parametrize('dtype', DTYPES)
def test_every_tail_of_a_row(dtype):
    """Rows that end anywhere in a piece of 8, from any place; NaN around."""
    for K in range(1, 41):
        big = torch.full((6, K + 9), math.nan, dtype=dtype, device='cuda')
        x = torch.randn(6, K).to(dtype)
        w = ops.mx4_quantize(torch.randn(5, K))
        wd = w.to('cuda')
        xv, wv = values(x), values(w.dequantize(torch.float32))
        for at in (0, 1, 5):
            big.fill_(math.nan)
            big[:, at:at + K] = x.cuda()
            rows = big[:, at:at + K]
            _same(ops.mx4_quantize(rows), ops.mx4_quantize(x))
            for form in (0, 1, 2):
                y = ops._native_or_die().mx4_linear(rows, wd.codes, wd.scales,
                                                    K, None, form)
                assert_close(y, xv @ wv.t(), xv.abs() @ wv.abs().t(), K)
        g = torch.randn(6, K).to(dtype)          # K columns of a gradient
        v = ops.mx4_quantize(torch.randn(K, 32))
        vd, vv = v.to('cuda'), values(v.dequantize(torch.float32))
        dx, _, db = ops._native_or_die().mx4_linear_backward(
            g.cuda(), vd.codes, vd.scales, None, None, 32, 0, -1, 0, 1)
        g64 = g.double()
        assert_close(dx, g64 @ vv, g64.abs() @ vv.abs(), K)
        assert_close(db, g64.sum(0), g64.abs().sum(0), 6)


@pytest.mark.parametrize('dtype', DTYPES)
def test_quantize_strides_and_alignments(dtype):
    base = torch.randn(40, 300).to(dtype)
    for view in (lambda t: t[:, :256], lambda t: t[:, 1:257],
                 lambda t: t[:, 8:200], lambda t: t[::3, 3:100],
                 lambda t: t.t(), lambda t: t[:1].expand(5, 300)):
        _same(ops.mx4_quantize(view(base.cuda())),
              ops.mx4_quantize(view(base)))


SIZES = [(1, 1, 1), (1, 32, 16), (2, 33, 5), (16, 128, 64), (17, 129, 65),
         (33, 96, 40), (64, 2048, 256), (130, 257, 131), (300, 200, 1000),
         (1100, 64, 1001), (8, 4096, 512), (513, 640, 384)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,K,N', SIZES)
def test_linear_and_its_gradients(M, K, N, dtype):
    x = torch.randn(M, K).to(dtype)
    w = torch.randn(N, K) / K ** 0.5
    b = torch.randn(N)
    g = torch.randn(M, N).to(dtype)
    xd, wd, bd = (t.cuda().requires_grad_() for t in (x, w, b))
    y = ops.mx4_linear(xd, wd, bd)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), g.cuda())
    assert y.dtype == dtype and dx.dtype == dtype
    assert dw.dtype == db.dtype == torch.float32
    xv, wv, g64 = values(x), values(w), g.double()
    want = xv @ wv.t() + b.double()
    mass = xv.abs() @ wv.abs().t() + b.double().abs()
    assert_close(y, want, mass, K + 1)
    assert_close(dx, g64 @ wv, g64.abs() @ wv.abs(), 3 * N)
    assert_close(dw, g64.t() @ xv, g64.abs().t() @ xv.abs(), 3 * M)
    assert_close(db, g64.sum(0), g64.abs().sum(0), M)
    # a held weight takes the form that rounds x on the way
    held = ops.mx4_quantize(wd)
    assert_close(ops.mx4_linear(xd, held, bd), want, mass, K + 1)
    with torch.no_grad():
        assert_close(ops.mx4_linear(xd, wd, bd), want, mass, K + 1)


@pytest.mark.parametrize('M,K,N', SIZES + [(2000, 512, 300)])
def test_whole_numbers_are_exact(M, K, N):
    # every sum is a whole number of quarters below 2^22: fp32 holds it
    x = GRID[torch.randint(0, 8, (M, K))] * (torch.randint(0, 2, (M, K)) * 2 - 1)
    w = GRID[torch.randint(0, 8, (N, K))] * (torch.randint(0, 2, (N, K)) * 2 - 1)
    g = torch.randint(-4, 5, (M, N)).double()
    xv, wv = values(x.float()), values(w.float())
    x, w = (t.float().cuda().requires_grad_() for t in (x, w))
    y = ops.mx4_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), g.float().cuda())
    assert torch.equal(y.double().cpu(), xv @ wv.t())
    assert torch.equal(dx.double().cpu(), g @ wv)
    assert torch.equal(dw.double().cpu(), g.t() @ xv)
    held = ops.mx4_quantize(w)
    for dtype in DTYPES:
        y = ops.mx4_linear(x.detach().to(dtype), held)
        assert torch.equal(y.cpu(), (xv @ wv.t()).to(dtype))
    # a gradient in bf16 and fp16 holds these numbers too
    for dtype in (torch.bfloat16, torch.float16):
        xt = x.detach().to(dtype).requires_grad_()
        y = ops.mx4_linear(xt, w)
        dx, dw = torch.autograd.grad(y, (xt, w), g.to(dtype).cuda())
        assert torch.equal(dx.cpu(), (g @ wv).to(dtype))
        assert torch.equal(dw.double().cpu(), g.t() @ xv)


@pytest.mark.parametrize('form', range(7))
@pytest.mark.parametrize('M,K,N', SIZES + [(260, 1, 260), (129, 384, 70),
                                           (700, 1000, 520)])
def test_every_form_at_every_size(M, K, N, form):
    ext = ops._native_or_die()
    x = GRID[torch.randint(0, 8, (M, K))] * (torch.randint(0, 2, (M, K)) * 2 - 1)
    w = GRID[torch.randint(0, 8, (N, K))] * (torch.randint(0, 2, (N, K)) * 2 - 1)
    b = torch.randint(-8, 9, (N,)).float()
    want = values(x.float()) @ values(w.float()).t() + b
    wq = ops.mx4_quantize(w.float().cuda())
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 1),
                        (torch.float16, 2)):
        base = torch.full((M, K + 9), math.nan, dtype=dtype, device='cuda')
        for lo in (0, 1, 8):
            xd = base[:, lo:lo + K]
            xd.copy_(x)
            y = ext.mx4_linear(xd, wq.codes, wq.scales, K, b.cuda(), form)
            assert torch.equal(y.cpu(), want.to(dtype))
            base.fill_(math.nan)
        q = ops.mx4_quantize(x.to(dtype).cuda())
        y = ext.mx4_linear_q(q.codes, q.scales, K, wq.codes, wq.scales,
                             b.to(dtype).cuda(), code, form)
        assert torch.equal(y.cpu(), want.to(dtype))


@pytest.mark.parametrize('form', [0, 1])
@pytest.mark.parametrize('M,K,N', SIZES + [
    (260, 1, 260), (129, 384, 70), (700, 1000, 520), (2500, 300, 260),
    (5000, 64, 64), (3001, 128, 128), (4099, 30, 300), (1500, 513, 24),
    (40, 600, 2000)])
def test_every_gradient_form_at_every_size(M, K, N, form):
    # whole numbers: sums of up to 5000 products of at most 4 x 6 are exact
    ext = ops._native_or_die()
    x = GRID[torch.randint(0, 8, (M, K))] * (torch.randint(0, 2, (M, K)) * 2 - 1)
    w = GRID[torch.randint(0, 8, (N, K))] * (torch.randint(0, 2, (N, K)) * 2 - 1)
    g = torch.randint(-4, 5, (M, N)).double()
    xv, wv = values(x.float()), values(w.float())
    dx, dw, db = g @ wv, g.t() @ xv, g.sum(0)
    xq, wq = (ops.mx4_quantize(t.float().cuda()) for t in (x, w))
    for code, dtype in enumerate(DTYPES):
        base = torch.full((M * N + 3,), math.nan, dtype=dtype, device='cuda')
        for lo in (0, 3):                  # on 16 bytes, and not
            gd = base[lo:lo + M * N].view(M, N)
            gd.copy_(g)
            got = ext.mx4_linear_backward(
                gd, wq.codes, wq.scales, xq.codes, xq.scales, K, code,
                (code + 1) % 3, (code + 2) % 3, form)
            for t, want, c in zip(got, (dx, dw, db),
                                  (code, (code + 1) % 3, (code + 2) % 3)):
                assert torch.equal(t.cpu(), want.to(DTYPES[c])), (dtype, lo, c)
            base.fill_(math.nan)


@pytest.mark.parametrize('form', [0, 1])
def test_gradients_at_the_ends_of_the_scales(form):
    # each value has to come out of bf16 as it is, subnormal ones too
    ext = ops._native_or_die()
    e = torch.arange(-127, 126, 4).double()
    x = GRID.repeat(4)[None, :] * torch.exp2(e)[:, None]        # rows of 32
    x[:, 0] = 6.0 * torch.exp2(e)
    q = ops.mx4_quantize(x.float().cuda())
    eye = torch.eye(len(e))
    for g, want in ((eye, values(x.float())),):
        _, dw, _ = ext.mx4_linear_backward(
            g.cuda(), None, None, q.codes, q.scales, 32, -1, 0, -1, form)
        assert torch.equal(dw.double().cpu(), want)
        dx, _, _ = ext.mx4_linear_backward(
            g.cuda(), q.codes, q.scales, None, None, 32, 0, -1, -1, form)
        assert torch.equal(dx.double().cpu(), want)


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16])
@pytest.mark.parametrize('M,K,N', [(300, 200, 136), (130, 257, 131),
                                   (2000, 70, 1000), (3001, 128, 33),
                                   (2101, 333, 235)])
def test_every_part_of_a_wide_output_gradient(M, K, N, dtype):
    """Alone and together, where both products read the same parts: each has
    its bits of the sum."""
    ext = ops._native_or_die()
    x, w, g = torch.randn(M, K), torch.randn(N, K), torch.randn(M, N).to(dtype)
    xv, wv, g64 = values(x), values(w), g.double()
    xq, wq = ops.mx4_quantize(x.cuda()), ops.mx4_quantize(w.cuda())
    for want_x, want_w in ((0, -1), (-1, 0), (0, 0)):
        dx, dw, _ = ext.mx4_linear_backward(
            g.cuda(), wq.codes, wq.scales, xq.codes, xq.scales, K, want_x,
            want_w, -1, 1)
        # three parts for each term of a sum
        if want_x == 0:
            assert_close(dx, g64 @ wv, g64.abs() @ wv.abs(), 3 * N)
        if want_w == 0:
            assert_close(dw, g64.t() @ xv, g64.abs().t() @ xv.abs(), 3 * M)
    # one term whose last bit only the last part holds
    g = torch.zeros(M, N, dtype=dtype)
    g[5, 7] = 1 + torch.finfo(dtype).eps
    wq, xq = (ops.mx4_quantize(torch.ones(n, K).cuda()) for n in (N, M))
    for want_x, want_w in ((0, -1), (-1, 0), (0, 0)):
        dx, dw, _ = ext.mx4_linear_backward(
            g.cuda(), wq.codes, wq.scales, xq.codes, xq.scales, K, want_x,
            want_w, -1, 1)
        if want_x == 0:
            assert torch.equal(dx.cpu(), g.float().sum(1, True).expand(M, K))
        if want_w == 0:
            assert torch.equal(dw.cpu(), g.float().sum(0)[:, None].expand(N, K))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,K,N', [(70, 130, 40), (3000, 200, 300)])
def test_infinities_in_the_output_gradient(M, K, N, dtype):
    # they reach the rows and columns that the formula gives them, as they are
    x = GRID[torch.randint(1, 8, (M, K))].float().cuda()
    w = GRID[torch.randint(1, 8, (N, K))].float().cuda()
    g = torch.zeros(M, N)
    g[M - 1, 5], g[2, N - 1], g[7, 7] = math.inf, -math.inf, math.nan
    xd, wd = x.to(dtype).requires_grad_(), w.requires_grad_()
    y = ops.mx4_linear(xd, wd)
    dx, dw = torch.autograd.grad(y, (xd, wd), g.to(dtype).cuda())
    want = torch.zeros(M, K)
    want[M - 1], want[2], want[7] = math.inf, -math.inf, math.nan
    assert torch.equal(dx.float().cpu().nan_to_num(1, 2, 3),
                       want.nan_to_num(1, 2, 3))
    want = torch.zeros(N, K)
    want[5], want[N - 1], want[7] = math.inf, -math.inf, math.nan
    assert torch.equal(dw.cpu().nan_to_num(1, 2, 3), want.nan_to_num(1, 2, 3))


@pytest.mark.parametrize('form', [2, 5, 6])
@pytest.mark.parametrize('K', [32, 200, 330, 520])
def test_more_tiles_than_blocks(K, form):
    # every block walks over several tiles, of 1, 2, 3 and 5 steps
    M, N = 66000, 530
    ext = ops._native_or_die()
    x = GRID[torch.randint(0, 8, (M, K))].float().cuda()
    w = GRID[torch.randint(0, 8, (N, K))].float().cuda()
    x[torch.rand(M, K, device='cuda') < 0.3] *= -4
    w[::3] *= -0.5
    want = (ops.mx4_quantize(x).dequantize()
            @ ops.mx4_quantize(w).dequantize().t())      # exact in fp32, too
    wq = ops.mx4_quantize(w)
    for _ in range(3):
        y = ext.mx4_linear(x, wq.codes, wq.scales, K, None, form)
        assert torch.equal(y, want)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M', [1, 40, 3000])
def test_strides_and_alignments_of_rows(dtype, M):
    base = torch.randn(M, 300).to(dtype).cuda()
    w = ops.mx4_quantize(torch.randn(96, 256).cuda())
    for lo in (0, 1, 8, 44):
        x = base[:, lo:lo + 256]
        assert torch.equal(ops.mx4_linear(x, w),
                           ops.mx4_linear(x.contiguous(), w))
    x = torch.randn(256, M).to(dtype).cuda().t()
    assert torch.equal(ops.mx4_linear(x, w),
                       ops.mx4_linear(x.contiguous(), w))
    # an expanded output gradient
    x = base[:, :256].detach().requires_grad_()
    y = ops.mx4_linear(x, w)
    (d1,) = torch.autograd.grad(y.sum(), x, retain_graph=True)
    (d2,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(d1, d2)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M', [4, 100, 2000])
def test_nan_and_infinity_stay_in_their_rows(dtype, M):
    K, N = 160, 200
    x, w = torch.randn(M, K).to(dtype), torch.randn(N, K)
    x[1, 40], x[3, 159], w[7, 0] = math.nan, -math.inf, math.inf
    g = torch.randn(M, N).to(dtype)
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = ops.mx4_linear(xd, wd)
    dx, dw = torch.autograd.grad(y, (xd, wd), g.cuda())
    bad = torch.zeros(M, N, dtype=torch.bool)
    bad[1], bad[3], bad[:, 7] = True, True, True
    assert torch.equal(y.cpu().isnan(), bad)
    assert torch.equal(ops.mx4_linear(xd, ops.mx4_quantize(wd)).cpu().isnan(),
                       bad)
    # a block reads as NaN in the gradients, too
    badx = torch.zeros(M, K, dtype=torch.bool)
    badx[:, :32] = True
    assert torch.equal(dx.cpu().isnan(), badx)
    badw = torch.zeros(N, K, dtype=torch.bool)
    badw[:, 32:64], badw[:, 128:160] = True, True
    assert torch.equal(dw.cpu().isnan(), badw)


def test_scales_far_apart():
    x = torch.randn(50, 256) * torch.exp2(
        torch.randint(-60, 60, (50, 8)).float()).repeat_interleave(32, 1)
    w = torch.randn(70, 256) * torch.exp2(
        torch.randint(-60, 60, (70, 8)).float()).repeat_interleave(32, 1)
    y = ops.mx4_linear(x.cuda(), w.cuda())
    xv, wv = values(x), values(w)
    assert_close(y, xv @ wv.t(), xv.abs() @ wv.abs().t(), 256)


def test_empty_sizes():
    for M, K, N in [(0, 32, 4), (3, 0, 4), (3, 32, 0)]:
        x = torch.randn(M, K, device='cuda', requires_grad=True)
        w = torch.randn(N, K, device='cuda', requires_grad=True)
        b = torch.randn(N, device='cuda', requires_grad=True)
        y = ops.mx4_linear(x, w, b)
        assert y.shape == (M, N)
        if K == 0:
            assert torch.equal(y, b.expand(M, N))
        for t, d in zip((x, w, b), torch.autograd.grad(y.sum(), (x, w, b))):
            assert d.shape == t.shape
            if M * K * N == 0 and t is not b:
                assert not d.any()


@pytest.mark.parametrize('M', [1, 300])
def test_other_stream_and_graph(M):
    K, N = 320, 130
    w = torch.randn(N, K, device='cuda', requires_grad=True)
    held = ops.mx4_quantize(w)
    x = torch.zeros(M, K, device='cuda', dtype=torch.bfloat16,
                    requires_grad=True)
    g = torch.randn(M, N, device='cuda').bfloat16()
    ins = [torch.randn(M, K, device='cuda').bfloat16() for _ in range(3)]

    def step():
        y = ops.mx4_linear(x, w)
        return (y.detach(), ops.mx4_linear(x.detach(), held),
                *torch.autograd.grad(y, (x, w), g))

    want = []
    for t in ins:
        with torch.no_grad():
            x.copy_(t)
        want.append([r.clone() for r in step()])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(again, want[-1]):
        assert torch.equal(a, b)
    del again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for t, ws in zip(ins * 2, want * 2):
        with torch.no_grad():
            x.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, ws):
            assert torch.equal(a, b)
        torch.randn(1000, device='cuda').sum().item()


def test_results_do_not_change_from_run_to_run():
    x = torch.randn(3000, 512, device='cuda').bfloat16().requires_grad_()
    w = torch.randn(256, 512, device='cuda', requires_grad=True)
    g = torch.randn(3000, 256, device='cuda').bfloat16()
    runs = []
    for _ in range(3):
        y = ops.mx4_linear(x, w)
        runs.append((y, *torch.autograd.grad(y, (x, w), g)))
    for r in runs[1:]:
        for a, b in zip(runs[0], r):
            assert torch.equal(a, b)


def test_refusals():
    q = ops.mx4_quantize(torch.randn(8, 64))
    with pytest.raises(ValueError, match='weight on cpu'):
        ops.mx4_linear(torch.randn(4, 64, device='cuda'), q)
    ext = ops._native_or_die()
    qd = q.to('cuda')
    x = torch.randn(4, 64, device='cuda')
    with pytest.raises(ValueError, match='input on cuda'):
        ops.mx4_linear(x, q)
    w = torch.randn(8, 64, device='cuda')
    with pytest.raises(ValueError, match='do not match'):
        ops.mx4_linear(x[:, :63], w)
    with pytest.raises(ValueError, match='do not match'):
        ops.mx4_linear(x, w[0])
    with pytest.raises(TypeError, match='weight'):
        ops.mx4_linear(x, w.double())
    with pytest.raises(TypeError, match='weight'):
        ops.mx4_linear(x, [w])
    with pytest.raises(ValueError, match='weight on cpu'):
        ops.mx4_linear(x, w.cpu())
    with pytest.raises(ValueError, match='bias'):
        ops.mx4_linear(x, w, torch.zeros(7, device='cuda'))
    with pytest.raises(TypeError, match='bias'):
        ops.mx4_linear(x, w, torch.zeros(8, device='cuda').double())
    with pytest.raises(ValueError, match='do not match'):
        ops.mx4_linear(x[:, :63], qd)
    with pytest.raises(TypeError, match='Double'):
        ops.mx4_linear(x.double(), qd)
    with pytest.raises(ValueError, match='bias'):
        ops.mx4_linear(x, qd, torch.zeros(7, device='cuda'))
    with pytest.raises(ValueError, match='bias on cpu'):
        ops.mx4_linear(x, qd, torch.zeros(8))
    with pytest.raises(ValueError, match='do not match'):
        ops.mx4_linear(x, ops.mx4_quantize(torch.zeros(2, 8, 64)).to('cuda'))
    with pytest.raises(RuntimeError, match='do not hold rows'):
        ext.mx4_linear(x, qd.codes[:, :, :32].contiguous(), qd.scales, 64,
                       None)
    with pytest.raises(RuntimeError, match='contiguous'):
        ext.mx4_linear(x, qd.codes[:, :, ::2], qd.scales, 64, None)
    with pytest.raises(ValueError, match='no form'):
        ext.mx4_linear(x, qd.codes, qd.scales, 64, None, 7)
    with pytest.raises(TypeError, match='Double'):
        ops.mx4_quantize(x.double())
    with pytest.raises(ValueError, match='not a number'):
        ops.mx4_quantize(x[0, 0])
    with pytest.raises(TypeError, match='a tensor, not list'):
        ops.mx4_quantize([x])
    with pytest.raises(ValueError, match='2\\^29 rows'):
        ops.mx4_quantize(x[:1, :1].expand(2 ** 29, 1))
    with pytest.raises(ValueError, match='2\\^22 elements'):
        ops.mx4_linear(x[:1, :1].expand(1, 2 ** 22), qd)
    neg = torch.complex(x, x).conj().imag
    assert neg.is_neg()
    with pytest.raises(TypeError, match='resolve_neg'):
        ops.mx4_linear(neg, qd)
    assert torch.equal(ops.mx4_linear(neg.resolve_neg(), qd),
                       ops.mx4_linear(-x, qd))
    with pytest.raises(TypeError, match='resolve_neg'):
        ops.grad_norm([neg])
    with pytest.raises(ValueError, match='no weight'):
        ext.mx4_linear_backward(x, None, None, None, None, 64, 0, -1, -1)
    with pytest.raises(ValueError, match='no rows'):
        ext.mx4_linear_backward(x, None, None, None, None, 64, -1, 0, -1)
    with pytest.raises(ValueError, match='does not match'):
        ext.mx4_linear_backward(torch.randn(4, 7, device='cuda'), qd.codes,
                                qd.scales, None, None, 64, 0, -1, -1)


@pytest.mark.parametrize('held', [False, True])
@pytest.mark.parametrize('wants', ['x', 'b', 'xb', 'w', 'xw', 'wb', 'xwb'])
def test_each_set_of_leaves_has_its_gradients(held, wants):
    if held and 'w' in wants:
        pytest.skip('held weights have no gradient')
    M, K, N = 70, 136, 40
    x, b = torch.randn(2, M // 2, K), torch.randn(N)
    w, g = torch.randn(N, K), torch.randn(2, M // 2, N)
    every = {'x': x.cuda(), 'w': w.cuda(), 'b': b.cuda().bfloat16()}
    leaves = [every[c].requires_grad_() for c in wants]
    weight = ops.mx4_quantize(every['w']) if held else every['w']
    y = ops.mx4_linear(every['x'], weight, every['b'])
    assert torch.equal(
        y, ops.mx4_linear(every['x'].detach(),
                          weight if held else weight.detach(),
                          every['b'].detach()))
    got = dict(zip(wants, torch.autograd.grad(y, leaves, g.cuda())))
    g64 = g.reshape(M, N).double()
    xv, wv = values(x.reshape(M, K)), values(w)
    want = {'x': (g64 @ wv, g64.abs() @ wv.abs(), N),
            'w': (g64.t() @ xv, g64.abs().t() @ xv.abs(), M),
            'b': (g64.sum(0), g64.abs().sum(0), M)}
    for c in wants:
        assert got[c].dtype == every[c].dtype and got[c].shape == every[c].shape
        v, mass, n = want[c]
        assert_close(got[c].reshape(v.shape), v, mass, n)
    with pytest.raises(RuntimeError):       # its tensors are freed
        torch.autograd.grad(y, leaves, g.cuda())


def test_second_derivatives_are_refused():
    x = torch.randn(4, 64, device='cuda', requires_grad=True)
    w = torch.randn(8, 64, device='cuda', requires_grad=True)
    g = torch.randn(4, 8, device='cuda', requires_grad=True)
    dx, dw = torch.autograd.grad(ops.mx4_linear(x, w), (x, w), g,
                                 create_graph=True)
    for d in (dx, dw):
        with pytest.raises(RuntimeError, match='once'):
            d.sum().backward(retain_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(d.sum(), g, retain_graph=True)


def test_checkpointing_and_saved_tensor_hooks():
    from torch.utils.checkpoint import checkpoint
    x = torch.randn(96, 128, device='cuda', requires_grad=True)
    w = torch.randn(64, 128, device='cuda', requires_grad=True)
    want = torch.autograd.grad(ops.mx4_linear(x, w).square().sum(), (x, w))
    y = checkpoint(lambda a, b: ops.mx4_linear(a, b).square(), x, w,
                   use_reentrant=False)
    for a, b in zip(torch.autograd.grad(y.sum(), (x, w)), want):
        assert torch.equal(a, b)
    with torch.autograd.graph.save_on_cpu():
        y = ops.mx4_linear(x, w).square()
    for a, b in zip(torch.autograd.grad(y.sum(), (x, w)), want):
        assert torch.equal(a, b)
