"""Captured library work replays as it ran: memset nodes are fill kernels."""

import ctypes

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip('needs a GPU', allow_module_level=True)

from mgproto_amd.utils.graphs import capture_graph  # noqa: E402


def _other_work():
    """Eager work of other sizes, and a synchronization."""
    junk = [torch.full((k * 1000 + 7,), 1e3, device='cuda')
            for k in range(1, 40)]
    return sum(float(j.sum()) for j in junk)


def _node_types(graph):
    hip = ctypes.CDLL('libamdhip64.so')
    raw, n = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert hip.hipGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    types = []
    for x in nodes:
        t = ctypes.c_int(-1)
        assert hip.hipGraphNodeGetType(ctypes.c_void_p(x),
                                       ctypes.byref(t)) == 0
        types.append(t.value)
    return types


MEMSET = 2                                        # hipGraphNodeTypeMemset


def test_memsets_of_every_kind():
    """Bytes, halves, words and rows from odd places on, in an order that only
    the edges keep: filled, then read, then filled again."""
    hip = ctypes.CDLL('libamdhip64.so')
    buf = torch.zeros(65536, dtype=torch.uint8, device='cuda')
    seen = torch.zeros_like(buf)
    at, size = buf.data_ptr(), ctypes.c_size_t
    host = torch.zeros(65536, dtype=torch.uint8)

    def byte(lo, v, n):
        host[lo:lo + n] = v
        return lambda s: hip.hipMemsetAsync(ctypes.c_void_p(at + lo), v,
                                            size(n), s)

    def d16(lo, v, n):
        host[lo:lo + 2 * n] = torch.tensor([v & 255, v >> 8],
                                           dtype=torch.uint8).repeat(n)
        return lambda s: hip.hipMemsetD16Async(
            ctypes.c_void_p(at + lo), ctypes.c_ushort(v), size(n), s)

    def d32(lo, v, n):
        host[lo:lo + 4 * n] = torch.tensor(
            [v >> 8 * i & 255 for i in range(4)], dtype=torch.uint8).repeat(n)
        return lambda s: hip.hipMemsetD32Async(
            ctypes.c_void_p(at + lo), v, size(n), s)

    def rows(lo, pitch, v, w, h):
        for r in range(h):
            host[lo + r * pitch:lo + r * pitch + w] = v
        return lambda s: hip.hipMemset2DAsync(
            ctypes.c_void_p(at + lo), size(pitch), v, size(w), size(h), s)

    calls = [byte(1, 7, 1), byte(3, 9, 30), byte(48, 5, 16), byte(100, 3, 4099),
             d16(8002, 0x1234, 777), d16(10000, 0x4321, 3),
             d32(12004, 0x01020304, 1001), d32(16388, 0x7f010203, 1),
             rows(20001, 131, 77, 100, 9), rows(24000, 64, 66, 64, 5)]
    first = host.clone()
    host[100:4199] = 200

    def fn():
        s = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        for c in calls:
            assert c(s) == 0
        seen.copy_(buf)                 # after the first, before the second
        assert hip.hipMemsetAsync(ctypes.c_void_p(at + 100), 200, size(4099),
                                  s) == 0

    graph, _ = capture_graph(fn)
    assert MEMSET not in _node_types(graph)
    written = first != 0
    for k in range(4):
        buf.fill_(0x50 + k)
        graph.replay()
        torch.cuda.synchronize()
        want = torch.where(written, first, torch.tensor(0x50 + k).byte())
        assert torch.equal(seen.cpu(), want)
        want[100:4199] = 200
        assert torch.equal(buf.cpu(), want)
        _other_work()


@pytest.mark.parametrize('n', [1000, 2 ** 22 + 3, 2 ** 24])
def test_reductions(n):
    """torch's sums over many blocks clear their counters."""
    x = torch.zeros(n, device='cuda')
    graph, s = capture_graph(lambda: (x.sum(), x.amax(), (x * 2).sum()))
    assert MEMSET not in _node_types(graph)
    for k in range(1, 6):
        x.fill_(0)
        x[::7] = k
        graph.replay()
        torch.cuda.synchronize()
        m = -(-n // 7)
        assert [float(t) for t in s] == [k * m, k, 2 * k * m]
        _other_work()


@pytest.mark.parametrize('cin,cout,k,size', [
    (512, 512, 3, 5), (256, 256, 3, 8), (64, 64, 3, 6), (3, 64, 7, 16),
    (512, 2048, 1, 4), (1024, 256, 1, 8)])
def test_library_convolutions(cin, cout, k, size):
    """Forward and both gradients of a library convolution, bf16. Whole
    numbers of at most 4 * size^2 terms of size 1 for the weight, at most 256
    in all: exact in bf16, whatever the order of the additions."""
    n = 4
    conv = torch.nn.Conv2d(cin, cout, k, padding=k // 2, bias=False).cuda()
    conv = conv.to(torch.bfloat16).to(memory_format=torch.channels_last)
    with torch.no_grad():
        conv.weight.copy_(torch.randint(-1, 2, conv.weight.shape)
                          * (torch.rand(conv.weight.shape) < 32 / cin / k / k))
    cl = lambda t: t.cuda().bfloat16().contiguous(  # noqa: E731
        memory_format=torch.channels_last)
    ins = [(torch.randint(-1, 2, (n, cin, size, size)),
            torch.randint(-1, 2, (n, cout, size, size))
            * (torch.rand(n, cout, 1, 1) < 32 / cout)) for _ in range(3)]
    x, g = (cl(t).requires_grad_(i == 0) for i, t in enumerate(ins[0]))

    def fn():
        y = conv(x)
        return (y.detach(), *torch.autograd.grad(y, (conv.weight, x), g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    graph, outs = capture_graph(fn)
    assert MEMSET not in _node_types(graph)
    w = conv.weight.detach().float().cpu()
    for a, b in ins * 3:
        with torch.no_grad():
            x.copy_(a)
            g.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        x64 = a.float().requires_grad_()
        w64 = w.clone().requires_grad_()
        y = F.conv2d(x64, w64, padding=k // 2)
        want = (y.detach(), *torch.autograd.grad(y, (w64, x64), b.float()))
        for got, t in zip(outs, want):
            assert float(t.abs().max()) <= 256
            assert torch.equal(got.float().cpu(), t)
        _other_work()


@pytest.mark.parametrize('mx4', [False, True])
def test_captured_training_step_of_all_convolutions(mx4):
    """The trainer's captured step with every convolution of the backbone
    learning and the gradients clipped: each replay moves the weights by what
    the gradients of the same batch at the same weights say."""
    from mgproto_amd import ops
    from mgproto_amd.engine.graphstep import GraphedStep
    from mgproto_amd.losses import build_aux_loss
    from mgproto_amd.model import construct_MGProto
    from mgproto_amd.models import use_mx4
    dev = torch.device('cuda', 0)
    torch.manual_seed(0)
    m = construct_MGProto('resnet50', pretrained=False, img_size=64,
                          prototype_shape=(20, 16, 1, 1), num_classes=5,
                          add_on_layers_type='regular', sz_embedding=8,
                          mem_capacity=8, mine_K=3).to(dev).train()
    m.features = m.features.to(memory_format=torch.channels_last)
    if mx4:
        use_mx4(m.features, train=True)
    aux = build_aux_loss('Proxy_Anchor', nb_classes=5, sz_embed=8).to(dev)
    ps = [*m.features.parameters(), *aux.parameters()]
    lr, clip = 0.125, 0.25
    opt = torch.optim.SGD(ps, lr=lr)
    gs = GraphedStep(m, aux, {'crs_ent': 1.0, 'mine': 0.2, 'aux': 0.5}, dev, 4,
                     64, warmup_steps=2, clip_grad_norm=clip)
    for i in range(9):
        x = torch.randn(4, 3, 64, 64, device=dev)
        t = torch.randint(0, 5, (4,), device=dev)
        before = [p.detach().clone() for p in ps]
        assert gs.matches(x, opt, True, False)
        norm = float(gs.step(x, t, opt, use_mine=True)['grad_norm'])
        torch.cuda.synchronize()
        assert not gs.broken and (gs.graph is not None) == (i >= 2)
        assert all(torch.isfinite(p.grad).all() for p in ps)
        # an untrained network of this size has a gradient of a few hundred
        # at most; wrongly cleared buffers hold 1e12 and more
        assert 0 < norm < 1e6
        moved = [p.detach() - q for p, q in zip(ps, before)]
        # the weights round what they are moved by, to half a step of each
        slack = 2.0 ** -24 * float(ops.grad_norm(before))
        assert float(ops.grad_norm(moved)) == pytest.approx(
            lr * min(norm, clip), rel=1e-4, abs=2 * slack)
        _other_work()


def test_no_capture_while_an_eager_graph_lives(capsys):
    """Steps stay eager, and train, until the last output of an eager forward
    is dropped."""
    from mgproto_amd.engine.graphstep import GraphedStep

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.conv = torch.nn.Conv2d(3, 5, 8)

        def forward(self, x, gt):
            y = self.conv(x).flatten(1)
            return y[:, :, None], y

    net = Net().cuda()
    opt = torch.optim.SGD(net.parameters(), lr=1e-3)
    gs = GraphedStep(net, None, {'crs_ent': 1.0, 'mine': 0.0, 'aux': 0.0},
                     torch.device('cuda', 0), 4, 8, amp_dtype=None,
                     warmup_steps=1)
    x = torch.randn(4, 3, 8, 8, device='cuda')
    t = torch.randint(0, 5, (4,), device='cuda')
    kept = [net(x, t)[0]]
    kept.append(kept)                         # a cycle
    losses = []

    def step():
        assert gs.matches(x, opt, False, False)
        losses.append(float(gs.step(x, t, opt)['ce']))

    for _ in range(3):
        step()
        assert gs.graph is None and not gs.broken
    assert capsys.readouterr().out.count('capture waits') == 1
    del kept
    for _ in range(3):
        step()
        assert gs.graph is not None
    assert losses == sorted(losses, reverse=True) and len(set(losses)) == 6
