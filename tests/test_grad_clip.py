"""Global gradient norm and clipping against 64-bit arithmetic; the refusals."""

import math

import pytest
import torch

from mgproto_amd import ops

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def _norm(ts, p):
    a = torch.cat([t.double().cpu().abs().flatten() for t in ts])
    if p == math.inf:
        return float(a.max()) if len(a) else 0.0
    return float((a ** p).sum()) ** (1 / p)


def _list(sizes, dtype, device, scale=1.0):
    return [(torch.randn(s) * scale).to(dtype).to(device) for s in sizes]


def _check(got, src, norm, max_norm):
    f = min(1.0, max_norm / (norm + 1e-6))
    for g, t in zip(got, src):
        want = t.double().cpu() * f
        h = torch.finfo(g.dtype).eps / 2
        # the factor and its product are fp32 at least: two roundings more
        tol = want.abs() * (h + 2 * 2.0 ** -24) * (1 + h) \
            + torch.finfo(g.dtype).tiny * torch.finfo(g.dtype).eps
        assert ((g.double().cpu() - want).abs() <= tol).all()


SIZES = [[1], [5, 1, 0, 17], [(3, 4, 5), (1000,), (64, 64, 3, 3)],
         [8192, 8193, 16383, 100000], list(range(1, 260))]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('p', [1.0, 2.0, math.inf])
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('sizes', SIZES, ids=len)
def test_norm_and_clip(sizes, dtype, p, device):
    src = _list(sizes, dtype, device)
    norm = _norm(src, p)
    assert float(ops.grad_norm(src, p)) == pytest.approx(norm, rel=2.0 ** -23)
    for max_norm in (0.5 * norm, 2 * norm, 0.0):
        ts = [t.clone() for t in src]
        out = ops.clip_grads_(ts, max_norm, p)
        assert out.dtype == torch.float32 and out.dim() == 0
        assert float(out) == pytest.approx(norm, rel=2.0 ** -23)
        _check(ts, src, norm, max_norm)
        if max_norm > norm:
            assert all(torch.equal(a, b) for a, b in zip(ts, src))


@pytest.mark.parametrize('device', DEVICES)
def test_into_other_buffers(device):
    src = (_list([5, (7, 9)], torch.bfloat16, device)
           + _list([33], torch.float16, device)
           + _list([(4, 1, 3)], torch.float32, device))
    keep = [t.clone() for t in src]
    flat = torch.full((5 + 63 + 33 + 12 + 4,), 7.0, device=device)
    views, at = [], 1                       # on odd places
    for t in src:
        views.append(flat[at:at + t.numel()].view(t.shape))
        at += t.numel()
    norm = _norm(src, 2.0)
    ops.clip_grads_(src, 1.0, out=views)
    assert all(torch.equal(a, b) for a, b in zip(src, keep))
    _check(views, src, norm, 1.0)
    assert flat[0] == 7 and (flat[at:] == 7).all()
    outs = [torch.empty_like(t, dtype=torch.float16) for t in src]
    ops.clip_grads_(src, 1e6, out=outs)
    assert all(torch.equal(o, t.half()) for o, t in zip(outs, src))


@pytest.mark.parametrize('device', DEVICES)
def test_layouts(device):
    a = torch.randn(4, 6, 5, 5).contiguous(
        memory_format=torch.channels_last).to(device)
    b = torch.randn(6, 10, device=device).t()
    c = torch.randn(20, 20, device=device)[::2, 1:7]      # with gaps
    e = torch.randn(3, 1, device=device).expand(3, 4)
    norm = _norm([a, b, c, e], 2.0)
    assert float(ops.grad_norm([a, b, c, e])) == pytest.approx(
        norm, rel=2.0 ** -23)
    outs = [torch.empty(t.shape, device=device) for t in (a, b, c, e)]
    ops.clip_grads_([a, b, c, e], 0.5, out=outs)
    _check(outs, [a, b, c, e], norm, 0.5)
    keep = [a.clone(), b.clone()]
    norm = _norm(keep, 2.0)
    ops.clip_grads_([a, b], 0.5)
    _check([a, b], keep, norm, 0.5)
    assert a.is_contiguous(memory_format=torch.channels_last)


@pytest.mark.parametrize('device', DEVICES)
def test_large_small_and_not_finite(device):
    for dtype, scale in ((torch.float32, 1e30), (torch.float32, 1e-30),
                         (torch.bfloat16, 1e30)):
        ts = _list([1000, 3], dtype, device, scale)
        keep = [t.clone() for t in ts]
        norm = _norm(ts, 2.0)
        assert float(ops.grad_norm(ts)) == pytest.approx(norm, rel=2.0 ** -23)
        ops.clip_grads_(ts, 1.0)
        _check(ts, keep, norm, 1.0)
    for p in (1.0, 2.0, math.inf):
        ts = _list([100, 40], torch.float32, device)
        ts[1][7] = math.nan
        assert math.isnan(float(ops.clip_grads_(ts, 1.0, p)))
        assert all(t.isnan().all() for t in ts)
        ts = _list([100, 40], torch.float32, device)
        ts[1][7] = -math.inf
        assert float(ops.clip_grads_(ts, 1.0, p)) == math.inf
        assert ts[1][7].isnan() and not ts[0].any()
        assert int(ts[1].isnan().sum()) == 1
        zero = [torch.zeros(5, device=device)]
        assert float(ops.clip_grads_(zero, 1.0, p)) == 0.0


@pytest.mark.parametrize('device', DEVICES)
def test_empty_lists(device):
    assert float(ops.grad_norm([])) == 0.0
    assert float(ops.clip_grads_([], 1.0)) == 0.0
    e = [torch.zeros(0, 3, device=device), torch.zeros(0, device=device)]
    assert float(ops.grad_norm(e)) == 0.0
    assert float(ops.clip_grads_(e, 1.0)) == 0.0
    one = torch.randn(7, device=device)
    assert float(ops.grad_norm(one)) == pytest.approx(_norm([one], 2.0),
                                                      rel=2.0 ** -23)


@pytest.mark.parametrize('device', DEVICES)
def test_refusals(device):
    t = torch.randn(10, device=device)
    with pytest.raises(ValueError, match='norm_type'):
        ops.grad_norm([t], 3.0)
    with pytest.raises(ValueError, match='norm_type'):
        ops.clip_grads_([t], 1.0, -math.inf)
    with pytest.raises(ValueError, match='max_norm'):
        ops.clip_grads_([t], -1.0)
    with pytest.raises(ValueError, match='max_norm'):
        ops.clip_grads_([t], math.nan)
    with pytest.raises(TypeError, match='float64|Double'):
        ops.grad_norm([t.double()])
    with pytest.raises(TypeError, match='[sS]parse'):
        ops.grad_norm([t, torch.eye(3, device=device).to_sparse()])
    with pytest.raises(TypeError):
        ops.grad_norm([t, None])
    with pytest.raises(ValueError, match='meta'):
        ops.grad_norm([t, t.to('meta')])
    with pytest.raises(ValueError, match='outputs'):
        ops.clip_grads_([t], 1.0, out=[])
    with pytest.raises(ValueError, match='out'):
        ops.clip_grads_([t], 1.0, out=[t[:5]])
    keep = t.clone()
    for bad in ([t, t], [t[:6], t[5:]]):
        with pytest.raises(RuntimeError, match='shares'):
            ops.clip_grads_(bad, 1.0)
    with pytest.raises(RuntimeError, match='shares'):
        ops.clip_grads_([t[:5], t[5:]], 1.0, out=[t[1:6], t[6:].new_empty(5)])
    with pytest.raises(RuntimeError, match='gaps or shares'):
        ops.clip_grads_([t[::2]], 1.0)
    with pytest.raises(RuntimeError, match='gaps or shares'):
        ops.clip_grads_([t[:1].expand(4)], 1.0)
    assert torch.equal(t, keep)
    # the same gradient twice is counted twice where nothing overlaps
    outs = [torch.empty_like(t) for _ in range(2)]
    norm = ops.clip_grads_([t, t], 0.1, out=outs)
    assert float(norm) == pytest.approx(_norm([t, t], 2.0), rel=2.0 ** -23)
    assert torch.equal(outs[0], outs[1])


@pytest.mark.gpu
def test_stream_and_graph():
    src = _list([5000, 77, 30000], torch.float32, 'cuda')
    ts = [torch.zeros_like(t) for t in src]
    for t in ts:
        ops.clip_grads_([t], 1.0)

    def fill(k):
        for t, s in zip(ts, src):
            t.copy_(s * k)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fill(1.0)
        ops.clip_grads_(ts, 3.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grads_(ts, 3.0)
        small = ops.grad_norm(ts, math.inf)
    for k in (1.0, 1e-4, 5.0, 0.5):
        fill(k)
        want = [t.clone() for t in ts]
        n = ops.clip_grads_(want, 3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert float(norm) == float(n)
        assert all(torch.equal(a, b) for a, b in zip(ts, want))
        assert float(small) == _norm(ts, math.inf)


def test_version_counter():
    t = torch.randn(4)
    v = t._version
    ops.clip_grads_([t], 0.1)
    assert t._version > v


@pytest.mark.gpu
@pytest.mark.parametrize('sizes', [
    [4095, 4096, 4097, 12288] * 3,             # pieces that end on a border
    [9000001, 5, 3000000, 1],                  # more pieces than blocks
    [30000 + i % 5 for i in range(560)],       # several launches, many sums
], ids=['borders', 'long', 'many'])
def test_long_lists_of_every_type(sizes):
    src = [torch.randn(n, device='cuda').to(DTYPES[i % 3])
           for i, n in enumerate(sizes)]
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in src))
    flat = torch.full((sum(sizes) + 2,), 7.0, device='cuda',
                      dtype=torch.bfloat16)
    outs = list(flat[1:-1].split(sizes))
    assert float(ops.clip_grads_(src, 0.5 * norm, out=outs)) == pytest.approx(
        norm, rel=2.0 ** -23)
    # the factor, the product in fp32, the rounding
    near = lambda o, t, h: ((o.double() - t.double() / 2).abs() <= (  # noqa: E731
        h + 2.0 ** -22) * t.double().abs() / 2 + torch.finfo(
            o.dtype).smallest_normal * 2 * h).all()
    assert all(near(o, t, 2.0 ** -8) for o, t in zip(outs, src))
    assert flat[0] == 7 and flat[-1] == 7
    again = [t.clone() for t in src]
    ops.clip_grads_(again, 0.5 * norm)
    assert all(near(o, t, torch.finfo(t.dtype).eps / 2)
               for o, t in zip(again, src))
    assert torch.equal(ops.grad_norm(src),
                       ops.clip_grads_(src, 2 * norm, out=outs))
