"""4-bit 1x1 convolutions and gradient clipping where the framework uses them:
layers, trainer, serving."""

import copy
import io
import json
import os
import subprocess
import sys

import pytest
import torch
import torch.nn.functional as F

from mgproto_amd import ops
from mgproto_amd.engine.trainer import clip_optimizer_grads
from mgproto_amd.model import construct_MGProto
from mgproto_amd.models import no_mx4, use_mx4
from mgproto_amd.models.conv1x1 import GemmConv2d
from mgproto_amd.serving import InferenceEngine
from mx4_oracle import assert_close, values

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _model(arch='resnet50', size=64):
    torch.manual_seed(0)
    return construct_MGProto(arch, pretrained=False, img_size=size,
                             prototype_shape=(20, 16, 1, 1), num_classes=5,
                             add_on_layers_type='regular', sz_embedding=8,
                             mem_capacity=8, mine_K=3)


def _want(conv, x):
    """The convolution of the rounded values, 64 bits."""
    sh, sw = conv.stride
    rows = x[:, :, ::sh, ::sw].permute(0, 2, 3, 1)
    shape = rows.shape
    a = values(rows.reshape(-1, shape[-1]))
    w = values(conv.weight.reshape(conv.out_channels, -1))
    y, mass = a @ w.t(), a.abs() @ w.abs().t()
    if conv.bias is not None:
        b = conv.bias.detach().double().cpu()
        y, mass = y + b, mass + b.abs()
    return (t.view(*shape[:-1], -1).permute(0, 3, 1, 2) for t in (y, mass))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('train', [False, True])
@pytest.mark.parametrize('stride,bias', [(1, True), (2, False)])
def test_convolution(stride, bias, train, device):
    conv = GemmConv2d(40, 24, 1, stride=stride, bias=bias).to(device)
    assert use_mx4(conv, train=train) == 1
    x = torch.randn(2, 40, 7, 5, device=device)
    for t in (x, x.contiguous(memory_format=torch.channels_last),
              x.bfloat16()):
        with torch.no_grad():
            y = conv(t)
        want, mass = _want(conv, t)
        assert y.shape == want.shape and y.dtype == t.dtype
        assert y.is_contiguous(memory_format=torch.channels_last)
        assert_close(y, want, mass, 41)
    no_mx4(conv)
    with torch.no_grad():
        assert torch.equal(conv(x), F.conv2d(x, conv.weight, conv.bias,
                                             stride))
    assert list(conv.state_dict()) == (['weight', 'bias'] if bias
                                       else ['weight'])
    assert not list(conv.buffers())


def test_only_plain_1x1_convolutions():
    m = torch.nn.Sequential(GemmConv2d(8, 8, 3, padding=1),
                            GemmConv2d(8, 8, 1, groups=2),
                            GemmConv2d(8, 8, 1, padding=1),
                            torch.nn.Conv2d(8, 8, 1), GemmConv2d(8, 4, 1))
    assert use_mx4(m) == 1 and m[4].mx4 == 'held'


def test_held_weights_follow_the_float_ones():
    conv = GemmConv2d(32, 8, 1)
    use_mx4(conv)
    x = torch.randn(1, 32, 2, 2)
    other = GemmConv2d(32, 8, 1)
    with torch.no_grad():
        before = conv(x)
        conv.load_state_dict(other.state_dict())
        use_mx4(other)
        assert torch.equal(conv(x), other(x))
        assert not torch.equal(conv(x), before)
        conv.weight.mul_(2)
        want, mass = _want(conv, x)
        assert_close(conv(x), want, mass, 33)
    again = copy.deepcopy(conv)
    with torch.no_grad():
        assert torch.equal(again(x), conv(x))
    conv.train()
    with pytest.raises(RuntimeError, match='cannot train'):
        conv(x)
    conv.eval()
    xg = x.clone().requires_grad_()
    conv(xg).sum().backward()               # the input's gradient is there
    assert xg.grad.abs().sum() > 0 and conv.weight.grad is None


@pytest.mark.parametrize('device', DEVICES)
def test_no_stale_codes(device):
    """Other parameters of the same version, copies and files of a layer whose
    weight changed after its codes were made."""
    conv = GemmConv2d(32, 8, 1).to(device)
    use_mx4(conv)
    x = torch.randn(1, 32, 2, 2, device=device)

    def check(c):
        with torch.no_grad():
            want, mass = _want(c, x)
            assert_close(c(x), want, mass, 33)

    other = GemmConv2d(32, 8, 1).to(device)
    assert other.weight._version == conv.weight._version
    conv.load_state_dict(other.state_dict(), assign=True)
    check(conv)
    conv.weight = torch.nn.Parameter(torch.randn_like(conv.weight))
    check(conv)
    with torch.no_grad():
        conv.weight.mul_(-3)
    again = copy.deepcopy(conv)
    check(again)
    f = io.BytesIO()
    torch.save(conv, f)
    f.seek(0)
    check(torch.load(f, weights_only=False))
    conv.to(torch.bfloat16)
    x = x.bfloat16()
    check(conv)
    with torch.inference_mode():
        conv.weight.mul_(2)
        conv(x)
    check(conv)
    with torch.inference_mode():
        late = GemmConv2d(32, 8, 1).to(device).bfloat16()
        use_mx4(late)
    assert not late._mx4_codes.is_inference()


@pytest.mark.gpu
def test_a_captured_layer_takes_new_codes():
    conv = GemmConv2d(32, 8, 1).cuda()
    use_mx4(conv)
    x = torch.randn(2, 32, 3, 3, device='cuda')
    with torch.no_grad():
        conv(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = conv(x)
        for k in range(3):
            conv.weight.normal_()
            use_mx4(conv)
            graph.replay()
            assert torch.equal(y, conv(x))


@pytest.mark.parametrize('device', DEVICES)
def test_training_gradients(device):
    conv = GemmConv2d(64, 16, 1).to(device)
    use_mx4(conv, train=True)
    x = torch.randn(3, 64, 4, 4, device=device)
    x = x.contiguous(memory_format=torch.channels_last).requires_grad_()
    g = torch.randn(3, 16, 4, 4, device=device)
    conv(x).backward(g)
    rows = lambda t: t.detach().double().cpu().permute(0, 2, 3, 1).reshape(  # noqa: E731
        -1, t.shape[1])
    a, w, g64 = values(rows(x)), values(conv.weight.view(16, 64)), rows(g)
    assert_close(conv.weight.grad.view(16, 64), g64.t() @ a,
                 g64.abs().t() @ a.abs(), 3 * 48)
    assert_close(rows(x.grad).float(), g64 @ w, g64.abs() @ w.abs(), 3 * 16)
    assert_close(conv.bias.grad, g64.sum(0), g64.abs().sum(0), 48)
    assert conv.weight.grad.shape == conv.weight.shape


@pytest.mark.parametrize('device', DEVICES)
def test_backbone_keeps_its_state_dict(device):
    m = _model().to(device).eval()
    keys = list(m.state_dict())
    n = use_mx4(m.features)
    assert n == sum(isinstance(c, GemmConv2d) for c in m.features.modules())
    assert n > 30 and all(c.mx4 is None for c in m.add_on_layers.modules()
                          if isinstance(c, GemmConv2d))
    assert list(m.state_dict()) == keys
    m.load_state_dict(copy.deepcopy(m.state_dict()))
    with torch.no_grad():
        out, _ = m(torch.randn(2, 3, 64, 64, device=device), None)
    assert torch.isfinite(out).all()


def test_clip_optimizer_grads():
    a, b, c = (torch.nn.Parameter(torch.randn(n)) for n in (5, 7, 3))
    opt = torch.optim.Adam([{'params': [a, c]}, {'params': [b], 'lr': 0.1}])
    a.grad, b.grad = torch.randn(5), torch.randn(7)
    keep = torch.cat([a.grad, b.grad]).double()
    norm = clip_optimizer_grads(opt, 0.1)
    assert float(norm) == pytest.approx(float(keep.norm()), rel=2.0 ** -23)
    got = torch.cat([a.grad, b.grad]).double()
    assert float(got.norm()) == pytest.approx(0.1, rel=1e-4)
    assert c.grad is None


def _step(m, opt, x, t, clip):
    out, _ = m(x, t)
    F.cross_entropy(out.float()[:, :, 0], t).backward()
    return clip_optimizer_grads(opt, clip)


@pytest.mark.parametrize('device', DEVICES)
def test_training_step_with_4_bits_and_clipping(device):
    """The operators in a row, as the trainer runs them."""
    m = _model('resnet50').to(device).train()
    use_mx4(m.features, train=True)
    ps = [p for p in m.features.parameters()]
    opt = torch.optim.SGD(ps, lr=0.1)
    x = torch.randn(4, 3, 64, 64, device=device)
    t = torch.arange(4, device=device)
    norm = _step(m, opt, x, t, 1e-3)
    assert torch.isfinite(norm) and float(norm) > 1e-3
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in ps)
    after = float(ops.grad_norm([p.grad for p in ps]))
    assert after == pytest.approx(1e-3, rel=1e-2)
    before = [p.detach().clone() for p in ps]
    opt.step()
    moved = ops.grad_norm([p.detach() - q for p, q in zip(ps, before)])
    assert float(moved) <= 0.1 * 1.02e-3


def test_serving_in_4_bits():
    x = torch.randn(2, 3, 64, 64)
    m = _model()
    eng = InferenceEngine(m, torch.device('cpu'), amp=False, weights='mx4')
    res = eng.predict(x)
    with torch.no_grad():
        want = F.softmax(m(x, None)[0][:, :, 0], dim=1)
    for b in range(2):
        assert res[b]['top_classes'][0]['prob'] == pytest.approx(
            float(want[b].max()), abs=1e-4)
    with pytest.raises(ValueError, match='mx8'):
        InferenceEngine(m, torch.device('cpu'), weights='mx8')


def test_train_driver_takes_both(tmp_path):
    env = dict(os.environ, MGPROTO_TINY_TEST='1')
    cmd = [sys.executable, os.path.join(ROOT, 'train.py'), '-arch',
           'resnet50', '-mem_sz', '8', '-mine_level', '3', '-aux_emb_sz', '8',
           '--epochs', '1', '--out', str(tmp_path / 'run'), '--mx4',
           '--clip-grad-norm', '0.5']
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=900,
                       env=env, cwd=ROOT)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    with open(tmp_path / 'run' / 'metrics.jsonl') as f:
        norms = [json.loads(line).get('train/grad_norm') for line in f]
    assert any(n is not None and n > 0 for n in norms)
    r = subprocess.run(cmd[:-1] + ['-1'], capture_output=True, text=True,
                       timeout=300, env=env, cwd=ROOT)
    assert r.returncode != 0 and 'positive' in r.stderr


@pytest.mark.gpu
def test_captured_serving_in_4_bits():
    # the library's convolutions between the 4-bit ones need not repeat
    # themselves bit for bit, and rounding to 4 bits makes a small difference
    # a large one: the layers themselves are compared below
    dev = torch.device('cuda', 0)
    m = _model().to(dev)
    m.features = m.features.to(memory_format=torch.channels_last)
    eng = InferenceEngine(m, dev, weights='mx4').capture(2)
    for _ in range(3):
        res = eng.predict(torch.randn(2, 3, 64, 64, device=dev))
        for r in res:
            assert sum(t['prob'] for t in r['top_classes']) == pytest.approx(
                1.0, abs=1e-4)
            assert r['density_pX'] > 0


@pytest.mark.gpu
def test_captured_held_layers_repeat_the_eager_ones():
    dev = torch.device('cuda', 0)
    torch.manual_seed(0)
    net = torch.nn.Sequential(GemmConv2d(64, 256, 1), torch.nn.ReLU(),
                              GemmConv2d(256, 512, 1, stride=2),
                              GemmConv2d(512, 40, 1)).to(dev).eval()
    use_mx4(net)
    ins = [torch.randn(6, 64, 56, 56, device=dev).bfloat16() for _ in range(3)]
    x = torch.zeros_like(ins[0])
    with torch.no_grad():
        want = [net(t) for t in ins]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = net(x)
    for t, w in zip(ins * 2, want * 2):
        x.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w)
        torch.randn(1000, device=dev).sum().item()


@pytest.mark.gpu
def test_captured_layers_and_clipping_repeat_the_eager_step():
    """Forward, gradients and clipping of a stack of 4-bit layers in a graph:
    every kernel in it has a fixed order, so that replays are the eager step
    bit for bit."""
    dev = torch.device('cuda', 0)
    torch.manual_seed(0)
    net = torch.nn.Sequential(GemmConv2d(64, 96, 1), torch.nn.ReLU(),
                              GemmConv2d(96, 40, 1, stride=2)).to(dev)
    use_mx4(net, train=True)
    ps = list(net.parameters())
    x = torch.zeros(4, 64, 12, 12, device=dev)
    g = torch.randn(4, 40, 6, 6, device=dev)

    def step():
        with torch.autocast('cuda', torch.bfloat16):
            y = net(x)
        grads = list(torch.autograd.grad(y, ps, g.to(y.dtype)))
        return [y.detach(), ops.clip_grads_(grads, 2.0), *grads]

    ins = [torch.randn_like(x) for _ in range(3)]
    want = []
    for t in ins:
        x.copy_(t)
        want.append([r.clone() for r in step()])
    assert all(float(w[1]) > 2.0 for w in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for t, w in zip(ins * 2, want * 2):
        x.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, w):
            assert torch.equal(a, b)
        torch.randn(1000, device=dev).sum().item()


@pytest.mark.gpu
def test_captured_training_step_with_both():
    """The trainer's captured step with 4-bit layers and clipping: plain SGD
    moves the weights by lr times the clipped gradient, in the eager steps and
    in the replays alike. (Only the 4-bit layers and the normalisations learn
    here: the library's weight gradients of small convolutions, replayed with
    other work between, hold garbage now and then.)"""
    from mgproto_amd.engine.graphstep import GraphedStep
    from mgproto_amd.losses import build_aux_loss
    dev = torch.device('cuda', 0)
    coefs = {'crs_ent': 1.0, 'mine': 0.2, 'aux': 0.5}
    m = _model('resnet50').to(dev).train()
    m.features = m.features.to(memory_format=torch.channels_last)
    use_mx4(m.features, train=True)
    for c in m.modules():
        if isinstance(c, torch.nn.Conv2d) and not getattr(c, 'mx4', None):
            c.requires_grad_(False)
    aux = build_aux_loss('Proxy_Anchor', nb_classes=5, sz_embed=8).to(dev)
    ps = [p for p in (*m.features.parameters(), *aux.parameters())
          if p.requires_grad]
    assert len(ps) > 100
    lr, clip = 0.125, 0.25
    opt = torch.optim.SGD(ps, lr=lr)
    gs = GraphedStep(m, aux, coefs, dev, 4, 64, warmup_steps=2,
                     clip_grad_norm=clip)
    for i in range(6):
        x = torch.randn(4, 3, 64, 64, device=dev)
        t = torch.randint(0, 5, (4,), device=dev)
        before = [p.detach().clone() for p in ps]
        assert gs.matches(x, opt, True, False)
        norm = float(gs.step(x, t, opt, use_mine=True)['grad_norm'])
        torch.cuda.synchronize()
        assert not gs.broken and (gs.graph is not None) == (i >= 2)
        moved = [p.detach() - q for p, q in zip(ps, before)]
        # the weights round what they are moved by, to half a step of each
        slack = 2.0 ** -24 * float(ops.grad_norm(before))
        assert float(ops.grad_norm(moved)) == pytest.approx(
            lr * min(norm, clip), rel=1e-4, abs=2 * slack)
        assert norm > 0
