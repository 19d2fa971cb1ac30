"""Global gradient norm and clipping of a list of tensors, on the device.

``grad_norm`` and ``clip_grads_`` never wait for the GPU and upload nothing,
so that they work inside a captured step; sums are held in 64 bits and have a
fixed order, so that every rank and every run gets the same factor from the
same gradients.
"""

from typing import Iterable, List, Optional, Sequence, Union

import torch
from torch.autograd import forward_ad

from . import _native_or_die, reference

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _tensors(ts: List[torch.Tensor], what: str):
    for t in ts:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f'{what}: tensors, not {type(t).__name__}')
        if t.layout != torch.strided:
            raise TypeError(f'{what}: dense tensors, not {t.layout}')
        if t.dtype not in _TYPES:
            raise TypeError(f'{what}: float32, bfloat16 or float16, not '
                            f'{t.dtype}')
        if t.device != ts[0].device:
            raise ValueError(f'{what}: tensors on {ts[0].device} and '
                             f'{t.device}')
        if (forward_ad._current_level >= 0
                and forward_ad.unpack_dual(t).tangent is not None):
            raise NotImplementedError(f'{what}: no forward-mode derivative')


def _check_p(norm_type: float, what: str) -> float:
    p = float(norm_type)
    if p not in (1.0, 2.0, float('inf')):
        raise ValueError(f'{what}: norm_type 1, 2 or inf, not {norm_type}')
    return p


def _list(ts) -> List[torch.Tensor]:
    return [ts] if isinstance(ts, torch.Tensor) else list(ts)


def _ext(ts):
    """The extension for GPU tensors, which makes the checks below itself."""
    if not (ts and isinstance(ts[0], torch.Tensor) and ts[0].is_cuda):
        return None
    return _native_or_die()


def grad_norm(grads: Union[torch.Tensor, Iterable[torch.Tensor]],
              norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of the list together, a float32 number on
    their device. An empty list has the norm 0 (on the CPU)."""
    ts = _list(grads)
    ext = _ext(ts)
    if ext is not None:
        return ext.grad_norm(ts, norm_type)
    _tensors(ts, 'grad_norm')
    p = _check_p(norm_type, 'grad_norm')
    if not ts:
        return torch.zeros(())
    with torch.no_grad():
        return reference.grad_norm(ts, p).float()


def clip_grads_(grads: Union[torch.Tensor, Iterable[torch.Tensor]],
                max_norm: float, norm_type: float = 2.0,
                out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the list by ``min(1, max_norm / (norm + 1e-6))`` and returns the
    norm before that, a float32 number on the device.

    In place, or into ``out``: tensors of the same shapes, of any of the three
    types (a flat fp32 buffer's views, say); ``grads`` then stay as they were.
    What is written has to be dense and apart from everything else in the
    call. A norm that is NaN makes every element NaN; an infinite one makes
    the finite elements 0 and the infinite ones NaN (all of them NaN where
    ``max_norm`` is infinite too)."""
    ts = _list(grads)
    outs = ts if out is None else _list(out)
    ext = _ext(ts)
    if ext is not None:
        return ext.clip_grads(ts, outs, max_norm, norm_type)
    _tensors(ts, 'clip_grads_')
    _tensors(outs, 'clip_grads_: out')
    p = _check_p(norm_type, 'clip_grads_')
    if not max_norm >= 0:
        raise ValueError(f'clip_grads_: max_norm {max_norm}')
    if len(outs) != len(ts):
        raise ValueError(f'clip_grads_: {len(ts)} gradients, {len(outs)} '
                         'outputs')
    for g, o in zip(ts, outs):
        if g.shape != o.shape:
            raise ValueError(f'clip_grads_: out {tuple(o.shape)} for a '
                             f'gradient {tuple(g.shape)}')
    if ts and outs[0].device != ts[0].device:
        raise ValueError(f'clip_grads_: gradients on {ts[0].device}, out on '
                         f'{outs[0].device}')
    if not ts:
        return torch.zeros(())
    with torch.no_grad():
        return reference.clip_grads(ts, outs, float(max_norm), p)
