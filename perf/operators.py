"""What is measured of the 4-bit product and the gradient clipping.

Four kinds of case, one for each way a user reaches the operators:

* ``quantize``: rows rounded to MX blocks (32 elements of the last axis share a
  power-of-two scale, elements are e2m1) and read back as values;
* ``linear``: ``y = Q(x) Q(w)^T + b`` with weights that are kept in 4 bits
  (serving);
* ``train``: the same product with float weights, rounded in the call, and its
  straight-through gradients (fine-tuning for 4 bits);
* ``clip``: the global norm of a list of gradients, and the gradients scaled to
  at most ``max_norm``, written into the optimiser's buffers.
"""

import math

import torch

own = False

_DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16,
           'fp16': torch.float16}
_SIZE = {'fp32': 4, 'bf16': 2, 'fp16': 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # an odd calibration batch in full precision: neither size is a
        # multiple of the block
        dict(name='quantize_odd_fp32', kind='quantize', M=777, K=333,
             dtype='fp32'),
        # the activations in front of a third-stage 1x1 convolution, 28x28
        # pixels of 80 images
        dict(name='quantize_stage3_bf16', kind='quantize', M=62720, K=1024,
             dtype='bf16'),
        # one row through a large layer: the smallest call, weights bound
        dict(name='linear_row_bf16', kind='linear', M=1, K=4096, N=4096,
             dtype='bf16', bias=True),
        # one image at the last stage (14x14 pixels, 2048 -> 512): latency of
        # a single request
        dict(name='linear_image_bf16', kind='linear', M=196, K=2048, N=512,
             dtype='bf16', bias=False),
        # ragged in every size, another type
        dict(name='linear_odd_fp16', kind='linear', M=777, K=333, N=1001,
             dtype='fp16', bias=True),
        # a batch of 80 images at the third stage (28x28, 1024 -> 256)
        dict(name='linear_stage3_bf16', kind='linear', M=62720, K=1024,
             N=256, dtype='bf16', bias=False),
        # the largest product: many rows through a wide layer, bound by the
        # matrix cores
        dict(name='linear_wide_bf16', kind='linear', M=8192, K=4096, N=16384,
             dtype='bf16', bias=True),
        # a small head fine-tuned in full precision, odd sizes
        dict(name='train_head_fp32', kind='train', M=83, K=200, N=65,
             dtype='fp32', bias=True),
        # a training step of a last-stage 1x1 convolution, batch 80
        # (14x14, 512 -> 2048)
        dict(name='train_stage4_bf16', kind='train', M=15680, K=512, N=2048,
             dtype='bf16', bias=False),
        # the warm phase: add-on layers and the proxies only
        dict(name='clip_head_fp32', kind='clip', layout='head', dtype='fp32',
             max_norm=1.0),
        # the joint phase of a ResNet-50 trunk: many tensors, most of them
        # short
        dict(name='clip_trunk_fp32', kind='clip', layout='trunk',
             dtype='fp32', max_norm=0.5),
        # a large model's bf16 gradients
        dict(name='clip_large_bf16', kind='clip', layout='large',
             dtype='bf16', max_norm=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['quantize', 'linear', 'linear', 'train', 'clip'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    if kind == 'quantize':
        while True:
            M, K = _log(rng, 1, 65536), _log(rng, 1, 8192)
            if M * K <= 62720 * 1024:
                return dict(kind=kind, M=M, K=K, dtype=dtype)
    if kind == 'linear':
        while True:
            M, K, N = _log(rng, 1, 65536), _log(rng, 1, 8192), \
                _log(rng, 1, 16384)
            if M * K * N <= 8192 * 4096 * 16384 and M * max(K, N) <= 2 ** 27:
                return dict(kind=kind, M=M, K=K, N=N, dtype=dtype,
                            bias=rng.random() < 0.5)
    if kind == 'train':
        while True:
            M, K, N = _log(rng, 1, 65536), _log(rng, 8, 4096), \
                _log(rng, 8, 4096)
            if M * K * N <= 15680 * 512 * 2048:
                return dict(kind=kind, M=M, K=K, N=N, dtype=dtype,
                            bias=rng.random() < 0.5)
    sizes = [_log(rng, 1, 2 ** 23) for _ in range(_log(rng, 1, 300))]
    while sum(sizes) > 2 ** 28:
        sizes.pop()
    return dict(kind=kind, layout='sizes',
                sizes=' '.join(str(s) for s in sizes), dtype=dtype,
                max_norm=rng.choice([0.1, 1.0, 1e6]))


def _trunk_shapes(layers=(3, 4, 6, 4)):
    """Parameters of a bottleneck ResNet with its add-on layers."""
    shapes = [(64, 3, 7, 7), (64,), (64,)]
    cin = 64
    for stage, blocks in enumerate(layers):
        mid = 64 << stage
        for b in range(blocks):
            shapes += [(mid, cin, 1, 1), (mid,), (mid,),
                       (mid, mid, 3, 3), (mid,), (mid,),
                       (4 * mid, mid, 1, 1), (4 * mid,), (4 * mid,)]
            if b == 0:
                shapes += [(4 * mid, cin, 1, 1), (4 * mid,), (4 * mid,)]
            cin = 4 * mid
    return shapes + _head_shapes(cin)


def _head_shapes(cin=2048):
    return [(64, cin, 1, 1), (64,), (64, 64, 1, 1), (64,), (200, 32)]


def _shapes(case):
    if case['layout'] == 'head':
        return _head_shapes()
    if case['layout'] == 'trunk':
        return _trunk_shapes()
    if case['layout'] == 'large':
        return [s for _ in range(16) for s in
                [(4096, 4096), (4096,), (16384, 4096), (4096,)]]
    return [(int(s),) for s in case['sizes'].split()]


def work(case):
    s = _SIZE[case['dtype']]
    if case['kind'] == 'clip':
        n = sum(math.prod(sh) for sh in _shapes(case))
        return {'bytes': 2 * s * n + 4, 'flops': 3 * n}
    M, K = case['M'], case['K']
    if case['kind'] == 'quantize':
        return {'bytes': 2 * s * M * K, 'flops': 2 * M * K}
    N = case['N']
    b = 4 * N if case['bias'] else 0
    if case['kind'] == 'linear':
        blocks = -(-K // 32)
        return {'bytes': s * M * K + N * blocks * 17 + s * M * N + b,
                'flops': 2 * M * N * K}
    return {'bytes': 2 * s * M * K + 2 * s * M * N + 8 * N * K + 2 * b,
            'flops': 6 * M * N * K}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _activations(M, K, dtype, g):
    """What follows a rectified, normalised layer: half of it zero, a few
    channels much larger than the rest."""
    x = torch.randn(M, K, device='cuda', generator=g)
    x = torch.relu_(x)
    gain = torch.exp(torch.randn(K, device='cuda', generator=g))
    return x.mul_(gain).to(dtype)


def _inputs(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dtype = _DTYPES[case['dtype']]
    state = {'kind': case['kind']}
    if case['kind'] == 'clip':
        state['grads'] = [
            torch.randn(sh, device='cuda', generator=g).mul_(0.02).to(dtype)
            for sh in _shapes(case)]
        state['max_norm'] = case['max_norm']
        return state
    M, K = case['M'], case['K']
    state['x'] = _activations(M, K, dtype, g)
    if case['kind'] == 'quantize':
        return state
    N = case['N']
    state['w'] = torch.randn(N, K, device='cuda',
                             generator=g).mul_(K ** -0.5)
    state['b'] = (torch.randn(N, device='cuda', generator=g).mul_(0.1)
                  if case['bias'] else None)
    if case['kind'] == 'train':
        state['g'] = torch.randn(M, N, device='cuda', generator=g).mul_(
            1.0 / M).to(dtype)
    return state


def _flat(like, dtype=None):
    """One zeroed buffer, and a view of it for each tensor, from multiples of
    64 elements on."""
    step = [-(-t.numel() // 64) * 64 for t in like]
    flat = torch.zeros(sum(step), device='cuda', dtype=dtype or like[0].dtype)
    views = [part[:t.numel()].view(t.shape)
             for part, t in zip(flat.split(step), like)]
    return flat, views


def prepare(case, seed):
    state = _inputs(case, seed)
    if case['kind'] == 'clip':
        # an optimiser that keeps one flat buffer, a view for each parameter
        state['flat'], state['out'] = _flat(state['grads'])
    if case['kind'] == 'linear':    # weights are kept rounded
        if own:
            from mgproto_amd import ops
            state['w'] = ops.mx4_quantize(state['w'])
        else:
            state['w'] = _rounded(state['w'])
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _rounded(x):
    """Values that MX blocks of the last axis stand for, in 32 bits."""
    M, K = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -K % 32)).view(M, -1, 32)
    amax = v.abs().amax(dim=2, keepdim=True)
    # amax = m * 2^e with m in [.5, 1), so floor(log2 amax) = e - 1
    e = torch.frexp(amax).exponent.clamp(-124, 130) - 3
    e = torch.where(amax > 0, e, -127).to(torch.int32)
    # 2^e by its bits; 2^-127 lies below the normal numbers
    up = torch.where(e > -127, (e + 127) << 23, 1 << 22).to(
        torch.int32).view(torch.float32)
    a = (v / up).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    q = torch.copysign(q, v) * up
    q = torch.where(torch.isfinite(amax), q, torch.nan)
    return q.view(M, -1)[:, :K]


def _plain(state):
    kind = state['kind']
    if kind == 'clip':
        total = torch.zeros((), dtype=torch.float64, device='cuda')
        for t in state['grads']:
            total += torch.sum(t.float().square(), dtype=torch.float64)
        norm = total.sqrt()
        coef = (state['max_norm'] / (norm + 1e-6)).clamp(max=1.0).float()
        for t, o in zip(state['grads'], state['out']):
            o.copy_(t.float() * coef)
        return {'norm': norm.float(), 'grads': state['flat']}
    x = state['x']
    xq = _rounded(x)
    if kind == 'quantize':
        return xq.to(x.dtype)
    b = state['b']
    if kind == 'linear':
        y = xq @ state['w'].t()
        return (y if b is None else y + b).to(x.dtype)
    wq = _rounded(state['w'])
    y = xq @ wq.t()
    g = state['g'].float()
    out = {'y': (y if b is None else y + b).to(x.dtype),
           'dx': (g @ wq).to(x.dtype), 'dw': g.t() @ xq}
    if b is not None:
        out['db'] = g.sum(0, dtype=torch.float64).float()
    return out


def _framework(state):
    from mgproto_amd import ops
    kind = state['kind']
    if kind == 'clip':
        norm = ops.clip_grads_(state['grads'], state['max_norm'],
                               out=state['out'])
        return {'norm': norm, 'grads': state['flat']}
    if kind == 'quantize':
        return ops.mx4_quantize(state['x']).dequantize()
    if kind == 'linear':
        return ops.mx4_linear(state['x'], state['w'], state['b'])
    x = state['x'].detach().requires_grad_()
    w = state['w'].detach().requires_grad_()
    leaves = [x, w]
    b = state['b']
    if b is not None:
        b = b.detach().requires_grad_()
        leaves.append(b)
    y = ops.mx4_linear(x, w, b)
    grads = torch.autograd.grad(y, leaves, state['g'])
    return dict(zip(('y', 'dx', 'dw', 'db'), (y.detach(), *grads)))


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------

def _block_values(x):
    """The same rounding from its definition: the nearest of the sixteen
    values, found among the midpoints between them."""
    x = x.double()
    out = torch.empty_like(x)
    grid = torch.tensor([0., .5, 1., 1.5, 2., 3., 4., 6.],
                        dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    for at in range(0, x.shape[1], 32):
        blk = x[:, at:at + 32]
        a = blk.abs().max(dim=1).values
        # the exponent field of a double is floor(log2 a) + 1023
        ex = ((a.view(torch.int64) >> 52) - 1023 - 2).clamp(-127, 127)
        unit = ((ex + 1023) << 52).view(torch.float64).unsqueeze(1)
        r = blk.abs() / unit
        low = torch.bucketize(r, mid, right=False)    # a tie goes down
        high = torch.bucketize(r, mid, right=True)    # a tie goes up
        code = torch.where(low % 2 == 0, low, high)   # ... to the even code
        val = torch.sign(blk) * grid[code] * unit
        val[~torch.isfinite(a)] = math.nan
        out[:, at:at + 32] = val
    return out


def exact(case, seed):
    kind = case['kind']
    state = _inputs(case, seed)
    if kind == 'clip':
        total = sum(float((t.double() ** 2).sum()) for t in state['grads'])
        norm = math.sqrt(total)
        coef = min(1.0, case['max_norm'] / (norm + 1e-6))
        flat, views = _flat(state['grads'], torch.float64)
        for t, v in zip(state['grads'], views):
            torch.mul(t.double(), coef, out=v)
        return {'norm': torch.tensor(norm, dtype=torch.float64),
                'grads': flat}
    xq = _block_values(state['x'])
    if kind == 'quantize':
        return xq
    wq = _block_values(state['w'])
    y = xq @ wq.t()
    if state['b'] is not None:
        y += state['b'].double()
    if kind == 'linear':
        return y
    g = state['g'].double()
    out = {'y': y, 'dx': g @ wq, 'dw': g.t() @ xq}
    if state['b'] is not None:
        out['db'] = g.sum(0)
    return out
