"""Calls of the 4-bit layers and of gradient clipping that once went wrong."""

import math

import pytest
import torch

from mgproto_amd import ops
from mgproto_amd.models import use_mx4
from mgproto_amd.models.conv1x1 import GemmConv2d
from mx4_oracle import assert_close, values

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def _check_layer(conv, x):
    """The layer's output is the convolution of the rounded values."""
    with torch.no_grad():
        y = conv(x)
    rows = x.permute(0, 2, 3, 1)
    a = values(rows.reshape(-1, rows.shape[-1]))
    w = values(conv.weight.reshape(conv.out_channels, -1))
    b = conv.bias.detach().double().cpu()
    assert_close(y.permute(0, 2, 3, 1).reshape(len(a), -1), a @ w.t() + b,
                 a.abs() @ w.abs().t() + b.abs(), conv.in_channels + 1)


@pytest.mark.parametrize('device', DEVICES)
def test_held_codes_follow_weights_made_in_inference_mode(device):
    with torch.inference_mode():
        conv = GemmConv2d(32, 8, 1).to(device)
    assert conv.weight.is_inference()
    use_mx4(conv)
    x = torch.randn(2, 32, 3, 3, device=device)
    _check_layer(conv, x)
    other = GemmConv2d(32, 8, 1).to(device)
    with torch.inference_mode():
        conv.load_state_dict(other.state_dict())
    _check_layer(conv, x)
    with torch.inference_mode():
        conv.weight.mul_(-3)
    _check_layer(conv, x)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('which', ['x', 'w', 'b'])
@pytest.mark.parametrize('held', [False, True])
@pytest.mark.parametrize('leaf', [False, True])
def test_forward_mode_derivatives_are_refused(which, held, leaf, device):
    if held and which == 'w':
        return                           # held weights have no derivative
    from torch.autograd import forward_ad
    every = {'x': torch.randn(4, 64, device=device),
             'w': torch.randn(8, 64, device=device),
             'b': torch.randn(8, device=device)}
    weight = ops.mx4_quantize(every['w']) if held else None
    with forward_ad.dual_level():
        t = every[which].requires_grad_(leaf)
        every[which] = forward_ad.make_dual(t, torch.ones_like(t))
        with pytest.raises(NotImplementedError):
            ops.mx4_linear(every['x'], weight or every['w'], every['b'])
        with torch.no_grad(), pytest.raises(NotImplementedError):
            ops.mx4_linear(every['x'], weight or every['w'], every['b'])
        # an ordinary call within the level is none of its business
        ops.mx4_linear(torch.randn(2, 64, device=device),
                       ops.mx4_quantize(torch.randn(3, 64, device=device)))


@pytest.mark.parametrize('device', DEVICES)
def test_clipping_refuses_forward_mode_derivatives(device):
    from torch.autograd import forward_ad
    t, out = torch.randn(9, device=device), torch.zeros(9, device=device)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.grad_norm([t, d]),
                     lambda: ops.clip_grads_([d], 0.1),
                     lambda: ops.clip_grads_([d], 0.1, out=[out])):
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call()
    assert not out.any()


@pytest.mark.gpu
def test_more_blocks_than_one_axis_of_a_launch():
    """2^28 rows of 129: 2^24 blocks of 256 threads, rounded alone and beside
    a weight, and read back."""
    R, K = 2 ** 28 + 5, 129
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 200 * 2 ** 30:
        pytest.skip('needs 200 GiB')
    x = torch.empty(R, K, device='cuda', dtype=torch.bfloat16).normal_()
    # ends, and around the rows of block 2^23, where a second axis begins
    parts = [slice(0, 40), slice(2 ** 27 - 40, 2 ** 27 + 40),
             slice(R - 40, R)]
    small = [ops.mx4_quantize(x[p].clone()) for p in parts]
    q = ops.mx4_quantize(x)
    for p, s in zip(parts, small):
        assert torch.equal(q.codes[:, p], s.codes)
        assert torch.equal(q.scales[:, p], s.scales)
    v = q.dequantize()
    for p, s in zip(parts, small):
        assert torch.equal(v[p], s.dequantize())
    del v, q
    w = torch.randn(1, K, device='cuda', requires_grad=True)
    y = ops.mx4_linear(x, w)
    for p in parts:
        a, b = values(x[p]), values(w)
        assert_close(y[p], a @ b.t(), a.abs() @ b.abs().t(), K)
    del x, y, small
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize('call', ['quantize', 'dequantize', 'held', 'few',
                                  'train', 'backward', 'norm', 'clip'])
def test_errors_of_launches_are_reported(call):
    """Every entry point asks for the runtime's last error after its launches;
    here it is one that a host call left."""
    import ctypes
    hip = ctypes.CDLL('libamdhip64.so')
    ext = ops._native_or_die()
    x, w = (torch.randn(40, 64, device='cuda') for _ in range(2))
    q = ops.mx4_quantize(w)
    y = torch.empty(40, 40, device='cuda')
    ws = w.clone().requires_grad_()
    calls = {
        'quantize': lambda: ops.mx4_quantize(x),
        'dequantize': lambda: q.dequantize(),
        'held': lambda: ops.mx4_linear(x, q),
        'few': lambda: ext.mx4_linear_q(q.codes, q.scales, 64, q.codes,
                                        q.scales, None, 0),
        'train': lambda: ops.mx4_linear(x, ws),
        'backward': lambda: ext.mx4_linear_backward(
            y, q.codes, q.scales, q.codes, q.scales, 64, 0, 0, 0),
        'norm': lambda: ops.grad_norm([x, w]),
        'clip': lambda: ops.clip_grads_([x, w], 1.0)}
    for c in calls.values():
        c()
    torch.cuda.synchronize()
    assert hip.hipGetDeviceCount(None) != 0       # no place for the result
    with pytest.raises(RuntimeError, match='invalid argument'):
        calls[call]()
    calls[call]()                                 # it is reported once
    torch.cuda.synchronize()


def _captured(net):
    from mgproto_amd.engine.graphstep import GraphedStep
    gs = GraphedStep(net, None, {}, torch.device('cpu'), 2, 8,
                     channels_last=False)
    opt = torch.optim.SGD(net.parameters(), lr=0.1)
    x = torch.zeros(2, 3, 8, 8)

    def kept():
        before = gs.graph = object()              # as if it were captured
        assert gs.matches(x, opt, True, False)
        return gs.graph is before

    kept()
    assert kept()
    return gs, kept


def test_a_captured_step_knows_its_clipping_and_its_layers():
    from mgproto_amd.models import no_mx4
    net = torch.nn.Sequential(GemmConv2d(3, 4, 1), torch.nn.ReLU(),
                              GemmConv2d(4, 4, 1))
    gs, kept = _captured(net)
    gs.clip_grad_norm = 1.0
    assert not kept() and kept()
    gs.clip_grad_norm = 0.5
    assert not kept() and kept()
    use_mx4(net, train=True)
    assert not kept() and kept()
    use_mx4(net[2], train=True)                   # as it was
    assert kept()
    no_mx4(net[0])
    assert not kept() and kept()
    use_mx4(net[2])
    assert not kept() and kept()


@pytest.mark.parametrize('here,there', [(1.0, None), (None, 1.0), (1.0, 2.0)])
def test_a_captured_step_clips_as_the_trainer(here, there):
    from mgproto_amd.engine import trainer
    net = torch.nn.Sequential(GemmConv2d(3, 4, 1))
    gs, _ = _captured(net)
    gs.clip_grad_norm = there
    with pytest.raises(ValueError, match='clip_grad_norm'):
        trainer._training(net, [], device=torch.device('cpu'), graph_step=gs,
                          clip_grad_norm=here)


def test_a_captured_step_follows_the_learning_rate():
    from mgproto_amd.engine.graphstep import GraphedStep
    net = torch.nn.Linear(4, 4)
    gs = GraphedStep(net, None, {'aux': 0.5, 'crs_ent': 1.0},
                     torch.device('cpu'), 2, 8, channels_last=False)
    opt = torch.optim.Adam([{'params': [net.weight], 'lr': 0.1},
                            {'params': [net.bias]}])
    decay = torch.optim.lr_scheduler.StepLR(opt, 1, 0.4)
    x = torch.zeros(2, 3, 8, 8)

    def kept():
        before = gs.graph = object()
        assert gs.matches(x, opt, True, False)
        return gs.graph is before

    kept()
    assert kept()
    opt.step()
    decay.step()
    assert not kept() and kept()
    opt.param_groups[1]['weight_decay'] = 1e-4
    assert not kept() and kept()
    gs.coefs['aux'] = 0.25
    assert not kept() and kept()
    opt.param_groups[0]['lr'] = torch.tensor(0.1)     # read by the step
    kept()
    opt.param_groups[0]['lr'].mul_(0.5)
    assert kept()


def _nearest(v, dtype):
    """float64 -> the nearest value of a 16-bit type, ties to even, with no
    type in between; normal numbers."""
    bits = 8 if dtype == torch.bfloat16 else 11
    m, e = torch.frexp(v)
    return torch.ldexp(torch.round(m * 2.0 ** bits), e - bits)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_wide_gradients_are_rounded_once(dtype, device):
    half = torch.finfo(dtype).eps / 2
    # alone, the element becomes max_norm (1 - 1e-6 / v): a billionth below the
    # middle of two values, which 32 bits cannot tell from it
    for sign in (1, -1):
        for middle, want in ((1 + 3 * half, 1 + 2 * half), (1 + half, 1.0)):
            g = torch.zeros(5000, device=device)
            g[4321] = sign * 2.0 ** 20
            out = torch.empty(5000, device=device, dtype=dtype)
            ops.clip_grads_([g], middle, out=[out])
            assert float(out[4321]) == sign * want
            assert int((out != 0).sum()) == 1
    g = torch.randn(300, 41, device=device)
    out = torch.empty_like(g, dtype=dtype)
    norm = float(g.double().norm())
    ops.clip_grads_([g], 100 * norm / 3e2, out=[out])
    v = g.double().cpu() * (100 * norm / 3e2 / (
        float(g.cpu().double().square().sum()) ** 0.5 + 1e-6))
    # where the factor's last bits decide, either neighbour
    lo, hi = (_nearest(v * (1 + s * 2.0 ** -50), dtype) for s in (-1, 1))
    got = out.double().cpu()
    tiny = v.abs() < torch.finfo(dtype).tiny
    assert ((got == lo) | (got == hi) | tiny).all()
    # infinities and numbers past the type
    g = torch.tensor([3e38, -3e38, 1.0], device=device)
    out = torch.empty(3, device=device, dtype=dtype)
    ops.clip_grads_([g], math.inf, out=[out])
    assert torch.equal(out.cpu(), torch.tensor([3e38, -3e38, 1.0]).to(dtype))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('to', [torch.bfloat16, torch.float16, torch.float32])
def test_norms_past_the_range_of_32_bits(to, device):
    """The factor is below the smallest fp32 number, what it gives is not."""
    n, m = 4096, 4096 * 5 + 3
    g = [torch.full((n,), 2.0 ** 127, device=device, dtype=torch.bfloat16),
         torch.randn(m, device=device).mul(1e37).bfloat16()]
    norm = math.sqrt(sum(float((t.double().cpu() * 2.0 ** -127).square().sum())
                         for t in g)) * 2.0 ** 127
    assert norm > 2.0 ** 132
    for max_norm in (1.0, 2.0 ** -20):
        outs = [torch.empty_like(t, dtype=to) for t in g]
        assert float(ops.clip_grads_(g, max_norm, out=outs)) == math.inf
        f = max_norm / (norm + 1e-6)
        h = torch.finfo(to).eps / 2
        for o, t in zip(outs, g):
            want = t.double().cpu() * f
            # the factor and its product, both in 32 bits; the rounding, or
            # half of the smallest step
            tol = want.abs() * (h + 2.0 ** -23) * (1 + h) + \
                torch.finfo(to).tiny * h
            assert ((o.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize('device', DEVICES)
def test_gradients_of_other_strides_are_checked_for_overlap(device):
    """Before they are copied: both forms refuse what both promise to."""
    keep = torch.randn(60, device=device)
    rows = lambda t, lo: t[lo:lo + 20].view(4, 5)  # noqa: E731
    calls = [
        # a transposed gradient that another output is written over
        lambda t: ([rows(t, 0).t(), rows(t, 20).t()],
                   [rows(t, 40).view(5, 4), rows(t, 10).view(5, 4)]),
        # one with gaps, from its own output's place into another's
        lambda t: ([t[40:50], t[:20:2]], [t[10:20], t[:10]]),
        lambda t: ([t[:20:2], t[40:50]], [t[:10], t[10:20]]),
        # its own output, but not from the same place on
        lambda t: ([rows(t, 2).t()], [rows(t, 0).view(5, 4)])]
    for call in calls:
        t = keep.clone()
        grads, outs = call(t)
        with pytest.raises(RuntimeError, match='shares'):
            ops.clip_grads_(grads, 0.1, out=outs)
        assert torch.equal(t, keep)
    # a turned view of itself is its own source
    t = keep.clone()
    grads, outs = [t[:25].view(5, 5).t()], [t[:25].view(5, 5)]
    want = keep[:25].view(5, 5).t()
    norm = float(want.double().norm())
    ops.clip_grads_(grads, 2 * norm, out=outs)
    assert torch.equal(t[:25].view(5, 5), want)
    assert torch.equal(t[25:], keep[25:])


@pytest.mark.gpu
def test_codes_made_in_a_capture_are_made_again_outside():
    """A capture records the rounding of a changed weight and does not do it."""
    conv = GemmConv2d(32, 8, 1).cuda()
    use_mx4(conv)
    x = torch.randn(2, 32, 3, 3, device='cuda')
    with torch.no_grad():
        conv(x)
        conv.weight.normal_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = conv(x)
        _check_layer(conv, x)                     # eager, before any replay
        for _ in range(3):
            conv.weight.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, conv(x))
            _check_layer(conv, x)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('stride', [1, 2])
def test_single_images(stride, device):
    """Convolutions take an image without a batch axis, 4-bit ones too."""
    conv = GemmConv2d(40, 24, 1, stride=stride).to(device)
    x = torch.randn(1, 40, 7, 5, device=device)
    shape = conv(x[0]).shape
    for train in (False, True):
        use_mx4(conv, train=train)
        with torch.no_grad():
            assert conv(x[0]).shape == shape
            assert torch.equal(conv(x[0]), conv(x)[0])
        for bad in (x[0, 0], x[None]):
            with pytest.raises(ValueError, match='an image'):
                conv(bad)


def test_no_mx4_leaves_nothing_behind():
    from mgproto_amd.models import no_mx4
    conv = GemmConv2d(32, 8, 1)
    before = set(vars(conv)), list(conv.buffers())
    for modes in ((False,), (True,), (False, True), (True, False),
                  (False, True, False)):
        for train in modes:
            use_mx4(conv, train=train)
        no_mx4(conv)
        assert not list(conv.buffers())
        assert set(vars(conv)) - before[0] <= {'mx4'} and conv.mx4 is None


def test_serving_says_what_it_serves():
    from mgproto_amd.model import construct_MGProto
    from mgproto_amd.serving import InferenceEngine

    def engine(arch, weights, mx4=False):
        m = construct_MGProto(arch, pretrained=False, img_size=64,
                              prototype_shape=(20, 16, 1, 1), num_classes=5,
                              add_on_layers_type='regular', sz_embedding=8,
                              mem_capacity=8, mine_K=3)
        if mx4:
            use_mx4(m.features, train=True)
        return InferenceEngine(m, torch.device('cpu'), weights=weights)

    assert engine('resnet50', 'float').weights == 'float'
    assert engine('resnet50', 'mx4').weights == 'mx4'
    assert engine('resnet50', 'float', mx4=True).weights == 'mx4'
    assert engine('vgg11', 'float').weights == 'float'
    with pytest.raises(ValueError, match='no 1x1'):
        engine('vgg11', 'mx4')


@pytest.mark.parametrize('device', DEVICES)
def test_values_past_the_range_are_refused(device):
    """2^128 and more: no product or gradient of them could be right."""
    grid = torch.tensor([0., .5, 1., 1.5, 2., 3., 4., 6.])
    for scale in (252, 253, 254, 255):
        for code in range(8):
            codes = torch.zeros(3, 64 // 2, dtype=torch.uint8)
            codes[1, 20] = code << 4 | 8              # and a negative zero
            scales = torch.full((3, 2), 127, dtype=torch.uint8)
            scales[1, 1] = scale
            parts = codes.to(device), scales.to(device)
            value = float(grid[code]) * 2.0 ** (scale - 127)
            if scale < 255 and value >= 2.0 ** 128:
                with pytest.raises(ValueError, match='2\\^128'):
                    ops.MX4Tensor.from_parts(*parts)
                continue
            q = ops.MX4Tensor.from_parts(*parts)
            for dtype in (torch.float32, torch.bfloat16):
                got = float(q.dequantize(dtype)[1, 41])
                assert got == value or scale == 255 and math.isnan(got)
    empty = torch.zeros(0, 16, dtype=torch.uint8)
    assert ops.MX4Tensor.from_parts(empty, empty[:, :1]).shape == (0, 32)
    with pytest.raises(TypeError):
        ops.MX4Tensor.from_parts(torch.zeros(2, 16), torch.zeros(2, 1))


def test_no_eager_graph_lives_when_a_step_is_captured():
    """A small batch runs eagerly, the next one may be captured: nothing of
    the first one's autograd graph is left then."""
    import gc
    import types
    import weakref
    from mgproto_amd.engine import trainer
    alive = []

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.lin = torch.nn.Linear(3, 4)
            self.iteration_counter = torch.zeros(1)
            self.queue = types.SimpleNamespace(mem_len=torch.zeros(4))
            self.capacity_pc = torch.ones(4)
            self.update_interval = 1

        def forward(self, x, gt):
            y = self.lin(x)
            mark = y.grad_fn.metadata['mark'] = type('Mark', (), {})()
            alive.append(weakref.ref(mark))       # as long as the node
            return y[:, :, None].expand(-1, -1, 3) * 1.0, y * 2.0

    class Step:
        clip_grad_norm = None
        seen = 0

        def matches(self, image, *_):
            return len(image) == 4

        def step(self, *_, **__):
            gc.collect()
            assert alive and all(r() is None for r in alive)
            self.seen += 1
            z = torch.zeros(())
            return dict.fromkeys(('loss', 'ce', 'mine', 'aux', 'n_correct',
                                  'grad_norm'), z)

    net, step = Net(), Step()
    opt = torch.optim.SGD(net.parameters(), lr=0.1)
    batches = [(torch.randn(n, 3), torch.randint(0, 4, (n,)))
               for n in (2, 4, 3, 4)]
    trainer._training(net, batches, optimizer=opt, use_mine=True,
                      aux_criterion=lambda x, t: x.square().mean(),
                      coefs={'crs_ent': 1.0, 'mine': 0.2, 'aux': 0.5},
                      device=torch.device('cpu'), amp_dtype=None,
                      graph_step=step, log=lambda *_: None, print_every=1)
    assert step.seen == 2 and len(alive) == 2


def test_living_graphs_are_seen():
    from mgproto_amd.utils.graphs import eager_graph_of
    if not ops.native_available():
        pytest.skip('needs the extension')
    a, b = (torch.randn(3, requires_grad=True) for _ in range(2))
    c = torch.randn(3)
    assert not eager_graph_of([a, b, c])
    y = (a * 2).sum()
    assert eager_graph_of([b, a]) and not eager_graph_of([b, c])
    y.backward()
    assert eager_graph_of([a])                # freed tensors, living nodes
    y = y.detach()
    assert not eager_graph_of([a])
    kept = [(b + 1)]
    kept.append(kept)
    del kept
    assert not eager_graph_of([b])            # a cycle is collected


@pytest.mark.parametrize('device', DEVICES)
def test_an_output_gradient_that_stands_for_its_negative(device):
    x = torch.randn(5, 40, device=device, requires_grad=True)
    w = torch.randn(7, 40, device=device, requires_grad=True)
    g = torch.randn(5, 7, device=device)
    neg = torch.complex(g, g).conj().imag
    assert neg.is_neg()
    got = torch.autograd.grad(ops.mx4_linear(x, w), (x, w), neg)
    want = torch.autograd.grad(ops.mx4_linear(x, w), (x, w), -g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
