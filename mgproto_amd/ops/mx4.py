"""4-bit rows (MX e2m1 with a power-of-two scale for 32 elements) and their
product, on the matrix cores that take them directly.

* ``mx4_quantize(x)`` rounds the last axis to blocks -> ``MX4Tensor``;
* ``MX4Tensor.dequantize()`` reads it back (bf16 and fp32 hold every value
  below 2^128, and so all that ``mx4_quantize`` makes);
* ``mx4_linear(x, weight, bias)`` is ``Q(x) Q(weight)^T + bias`` with fp32
  sums. A held ``MX4Tensor`` weight serves; a float weight is rounded in the
  call and trains: the gradients are straight-through,
  ``dx = g Q(w)``, ``dw = g^T Q(x)``, ``db = sum g``.

Format (OCP Microscaling Formats v1.0, MXFP4): a block of 32 has the scale
``2^E``, ``E = clamp(floor(log2 max|x|) - 2, -127, 127)``, and each element is
the nearest of ``{0, .5, 1, 1.5, 2, 3, 4, 6} * 2^E`` with its sign, ties to the
even code, 6 at most. A block that holds a NaN or an infinity reads as NaN.

CPU tensors take the PyTorch form (ops/reference.py), GPU tensors the HIP
kernels (ops/hip/mx4_*.hip).
"""

import math
from typing import Optional, Union

import torch

from . import _native_or_die, reference

_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check_float(t: torch.Tensor, what: str):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{what}: a tensor, not {type(t).__name__}')
    if t.dtype not in _CODE:
        raise TypeError(f'{what}: float32, bfloat16 or float16, not {t.dtype}')


def _ext(t: torch.Tensor):
    """The extension for GPU tensors, None for the PyTorch form."""
    return _native_or_die() if t.is_cuda else None


class MX4Tensor:
    """Rows held in 4 bits, laid out for the matrix cores.

    For ``rows`` = R rows of K elements, ``codes`` is uint8 [ceil(K/128), R,
    64]: the 64 bytes of 128 elements (low nibble first) of all rows, then the
    next 128; ``scales`` is uint8 [ceil(K/512), R, 16], where the byte
    ``4*g + s`` belongs to block ``g`` of the ``s``-th 128 (2^(byte-127), 255 =
    NaN). Codes and scales behind K are 0. ``parts`` and ``from_parts`` give
    and take the plain order. ``dtype`` is the type that ``dequantize`` gives
    where none is asked."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape,
                 dtype: torch.dtype = torch.bfloat16):
        shape = torch.Size(shape)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError('MX4Tensor: codes and scales are uint8')
        if len(shape) < 1 or min(shape) < 0:
            raise ValueError(f'MX4Tensor: no rows of shape {tuple(shape)}')
        R, K = math.prod(shape[:-1]), shape[-1]
        if (codes.shape != (-(-K // 128), R, 64)
                or scales.shape != (-(-K // 512), R, 16)):
            raise ValueError(
                f'MX4Tensor: codes {tuple(codes.shape)} and scales '
                f'{tuple(scales.shape)} do not hold {R} rows of {K}')
        if codes.device != scales.device:
            raise ValueError('MX4Tensor: codes and scales on one device')
        if dtype not in _CODE:
            raise TypeError(f'MX4Tensor: no values of type {dtype}')
        self.codes, self.scales = codes.contiguous(), scales.contiguous()
        self.shape, self.dtype = shape, dtype

    @classmethod
    def _of(cls, codes, scales, shape, dtype) -> 'MX4Tensor':
        """From what the kernels made."""
        q = object.__new__(cls)
        q.codes, q.scales, q.shape, q.dtype = codes, scales, shape, dtype
        return q

    @classmethod
    def from_parts(cls, codes: torch.Tensor, scales: torch.Tensor,
                   dtype: torch.dtype = torch.bfloat16) -> 'MX4Tensor':
        """From codes [..., K/2] and scales [..., K/32] in plain order, K a
        multiple of 32, as other programs store them. Values of 2^128 and more
        (scales 2^126 and 2^127 can make them, ``mx4_quantize`` does not) are
        refused: neither bf16 nor fp32 holds them. Waits for the GPU."""
        K = codes.shape[-1] * 2
        if K % 32 or scales.shape != (*codes.shape[:-1], K // 32):
            raise ValueError(
                f'MX4Tensor: codes {tuple(codes.shape)} and scales '
                f'{tuple(scales.shape)} are not blocks of 32')
        shape = (*codes.shape[:-1], K)
        R = math.prod(shape[:-1])
        q = cls(*reference.mx4_arrange(codes.reshape(R, K // 2),
                                       scales.reshape(R, K // 32)),
                shape, dtype)
        # the largest code of a block: 6 stands for 4, 4 for 2
        top = torch.maximum(codes & 7, codes >> 4 & 7).reshape(R, K // 32, 16)
        if R * K:
            top, of = top.amax(2), scales.reshape(R, K // 32)
            if ((of == 253) & (top >= 6) | (of == 254) & (top >= 4)).any():
                raise ValueError('MX4Tensor: a value of 2^128 or more')
        return q

    def parts(self):
        """(codes [..., K/2], scales [..., K/32]) in plain order, K rounded up
        to a multiple of 32."""
        nb, lead = -(-self.K // 32), self.shape[:-1]
        codes, scales = reference.mx4_plain(self.codes, self.scales, self.K)
        return codes.view(*lead, nb * 16), scales.view(*lead, nb)

    @property
    def K(self) -> int:
        return self.shape[-1]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def to(self, device) -> 'MX4Tensor':
        return MX4Tensor(self.codes.to(device), self.scales.to(device),
                         self.shape, self.dtype)

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return mx4_dequantize(self, dtype)

    def __repr__(self):
        return (f'MX4Tensor(shape={tuple(self.shape)}, '
                f'device={self.device}, dtype={self.dtype})')


def _matrix(x: torch.Tensor) -> torch.Tensor:
    """[..., K] -> [M, K]."""
    return x.reshape(math.prod(x.shape[:-1]), x.shape[-1])


def mx4_quantize(x: torch.Tensor) -> MX4Tensor:
    """[..., K] float32, bfloat16 or float16 -> 4-bit rows. No gradient."""
    if isinstance(x, torch.Tensor) and x.is_cuda:
        ext = _ext(x)                  # refuses what the checks below refuse
        if ext is not None:
            return MX4Tensor._of(*ext.mx4_quantize(x), x.shape, x.dtype)
    _check_float(x, 'mx4_quantize')
    if x.dim() < 1:
        raise ValueError('mx4_quantize: a tensor of rows, not a number')
    codes, scales = reference.mx4_quantize(_matrix(x.detach()))
    return MX4Tensor._of(codes, scales, x.shape, x.dtype)


def mx4_dequantize(q: MX4Tensor,
                   dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values that 4-bit rows stand for. bf16 and fp32 hold all that
    ``mx4_quantize`` and ``from_parts`` give; fp16 rounds, and overflows, where a
    scale leaves its range."""
    dtype = dtype or q.dtype
    if dtype not in _CODE:
        raise TypeError(f'mx4_dequantize: no values of type {dtype}')
    ext = _ext(q.codes)
    if ext is not None:
        out = ext.mx4_dequantize(q.codes, q.scales, q.shape[-1], _CODE[dtype])
    else:
        out = reference.mx4_dequantize(q.codes, q.scales, q.K, dtype)
    return out if len(q.shape) == 2 else out.view(q.shape)


class _MX4Linear(torch.autograd.Function):
    """The PyTorch form; that of GPU tensors is native. weight: a float [N, K]
    matrix, or None with (wc, ws) held in 4 bits."""

    @staticmethod
    def forward(ctx, x, weight, wc, ws, bias):
        K = x.shape[-1]
        need_x, need_w = ctx.needs_input_grad[:2]
        xc, xs = reference.mx4_quantize(_matrix(x))
        if weight is not None:
            wc, ws = reference.mx4_quantize(weight)
        with torch.autocast(x.device.type, enabled=False):
            y = reference.mx4_product(xc, xs, wc, ws, K, bias, x.dtype)
        ctx.save_for_backward(*((wc, ws) if need_x else (None, None)),
                              *((xc, xs) if need_w else (None, None)))
        ctx.K = K
        ctx.types = tuple(
            _CODE[t.dtype] if need else -1 for t, need in
            zip((x, weight, bias), (need_x, need_w, ctx.needs_input_grad[4])))
        return y.view(*x.shape[:-1], wc.shape[1])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        with torch.autocast(g.device.type, enabled=False):
            dx, dw, db = reference.mx4_backward(g, *ctx.saved_tensors, ctx.K,
                                                *ctx.types)
        return dx, dw, None, None, db


def mx4_linear(x: torch.Tensor, weight: Union[MX4Tensor, torch.Tensor],
               bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``Q(x) Q(weight)^T + bias``: x [..., K], weight [N, K], bias [N]; the
    result [..., N] has x's type. Sums are fp32, rounded once.

    A NaN or an infinity in a block of x makes its row NaN, one in a block of
    the weight its column. Differentiable once, in x, a float weight and bias.
    """
    held = type(weight) is MX4Tensor
    if isinstance(x, torch.Tensor) and x.is_cuda:
        ext = _ext(x)                  # refuses what the checks below refuse
        if ext is not None and held and len(weight.shape) == 2:
            return ext.mx4_linear(x, weight.codes, weight.scales,
                                  weight.shape[1], bias)
        if ext is not None and isinstance(weight, torch.Tensor):
            return ext.mx4_linear_float(x, weight, bias)
    _check_float(x, 'mx4_linear: input')
    if not held:
        _check_float(weight, 'mx4_linear: weight')
    if x.dim() < 1:
        raise ValueError('mx4_linear: input: rows, not a number')
    if len(weight.shape) != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f'mx4_linear: input {tuple(x.shape)} and weight '
                         f'{tuple(weight.shape)} do not match')
    if weight.device != x.device:
        raise ValueError(f'mx4_linear: input on {x.device}, weight on '
                         f'{weight.device}')
    if bias is not None:
        _check_float(bias, 'mx4_linear: bias')
        if bias.shape != (weight.shape[0],):
            raise ValueError(f'mx4_linear: bias {tuple(bias.shape)} for '
                             f'{weight.shape[0]} columns')
        if bias.device != x.device:
            raise ValueError(f'mx4_linear: input on {x.device}, bias on '
                             f'{bias.device}')
    wc, ws = (weight.codes, weight.scales) if held else (None, None)
    return _MX4Linear.apply(x, None if held else weight, wc, ws, bias)
