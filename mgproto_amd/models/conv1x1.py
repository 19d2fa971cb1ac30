"""1x1 convolutions as hipBLASLt GEMMs.

A stride-1 1x1 conv on an NHWC tensor IS the GEMM ``[N*H*W, Cin] x
[Cin, Cout]``. MIOpen routes these through CK batched-GEMM kernels that
measure ~45 TF effective on the flagship step (profiles/ — ~11 ms/step);
``torch.matmul`` on the same shapes hits hipBLASLt's tuned bf16 GEMMs.
Per the MI355X design rules, plain library GEMMs belong to
hipBLASLt/rocBLAS — hand-written MFMA kernels are reserved for fused ops.

``conv1x1`` falls back to F.conv2d off the fast path (CPU, fp32,
non-channels-last, strided, or grouped), which is numerically the
reference behavior.
"""

import os
import weakref

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops


def _usable(x: torch.Tensor, conv: nn.Conv2d) -> bool:
    # Measured on the flagship step: plain hipBLASLt matmul on these
    # skinny-K shapes is ~35% SLOWER than MIOpen's CK batched-GEMM picks
    # (1236 vs 1666 img/s, profiles/bench_history_r01.md). Round 2 closed
    # the question: TunableOp-tuned hipBLASLt still loses end-to-end
    # (1646.9 vs 1994.2 img/s) and per shape CK wins 12 of 14 — a hybrid
    # would save 0.04 ms of 4.32 (profiles/bench_r02/conv1x1_per_shape.log).
    # The GEMM path stays opt-in for A/B only.
    if os.environ.get('MGPROTO_GEMM_CONV1X1') != '1':
        return False
    return (x.is_cuda and x.dim() == 4
            and x.dtype in (torch.bfloat16, torch.float16)
            and conv.kernel_size == (1, 1)
            and conv.stride == (1, 1)
            and conv.padding == (0, 0)
            and conv.groups == 1
            and x.is_contiguous(memory_format=torch.channels_last))


def conv1x1(x: torch.Tensor, conv: nn.Conv2d) -> torch.Tensor:
    """Apply a 1x1 nn.Conv2d, as a GEMM when the layout allows."""
    if not _usable(x, conv):
        return F.conv2d(x, conv.weight, conv.bias, conv.stride,
                        conv.padding, conv.dilation, conv.groups)
    N, C, H, W = x.shape
    Co = conv.out_channels
    x2 = x.permute(0, 2, 3, 1).reshape(-1, C)          # free view (NHWC)
    w = conv.weight.view(Co, C)
    if conv.bias is not None:
        y2 = torch.addmm(conv.bias.to(x2.dtype), x2, w.t().to(x2.dtype))
    else:
        y2 = x2 @ w.t().to(x2.dtype)
    return y2.view(N, H, W, Co).permute(0, 3, 1, 2)    # channels_last NCHW


class GemmConv2d(nn.Conv2d):
    """Drop-in nn.Conv2d that takes the hipBLASLt GEMM path for stride-1
    1x1 convs on channels-last bf16 inputs (state dict unchanged), or the
    4-bit product where ``use_mx4`` asked for it."""

    mx4 = None          # None, 'train' or 'held'

    def forward(self, x):
        if self.mx4 is not None:
            return self._mx4_forward(x)
        return conv1x1(x, self)

    # ------------------------------------------------------------ 4-bit form
    def _mx4_pack(self):
        # tensors of the ordinary kind whatever mode the caller is in
        with torch.inference_mode(False), torch.no_grad():
            q = ops.mx4_quantize(self.weight.reshape(self.out_channels, -1))
            old = getattr(self, '_mx4_codes', None)
            if (old is not None and old.shape == q.codes.shape
                    and old.device == q.device):
                # in place: a captured graph reads them where they are
                old.copy_(q.codes)
                self._mx4_scales.copy_(q.scales)
            else:
                # not in the state dict: made from the weight again
                self.register_buffer('_mx4_codes', q.codes, persistent=False)
                self.register_buffer('_mx4_scales', q.scales, persistent=False)
        if self.weight.is_cuda and torch.cuda.is_current_stream_capturing():
            # recorded, not done: the next forward makes them in earnest
            self._mx4_of = _nothing, None
        else:
            self._mx4_of = weakref.ref(self.weight), _state(self.weight)

    def _mx4_weight(self):
        if self.mx4 == 'train':
            return self.weight.view(self.out_channels, -1)
        if (self.training and torch.is_grad_enabled()
                and self.weight.requires_grad):
            raise RuntimeError(
                'this 1x1 convolution holds its weight in 4 bits and cannot '
                'train it: use_mx4(model, train=True), or freeze the weight')
        made_of, state = self._mx4_of
        if (state is None or made_of() is not self.weight
                or state != _state(self.weight)):
            self._mx4_pack()
        return ops.MX4Tensor(self._mx4_codes, self._mx4_scales,
                             (self.out_channels, self.in_channels))

    def __getstate__(self):
        # copies and files: rounded again from the weight that they hold
        state = self.__dict__.copy()
        if '_mx4_of' in state:
            state['_mx4_of'] = _nothing, None
        return state

    def _mx4_forward(self, x):
        if x.dim() not in (3, 4):
            raise ValueError(f'an image [C, H, W] or a batch [N, C, H, W], '
                             f'not {tuple(x.shape)}')
        kind = x.device.type
        if torch.is_autocast_enabled(kind):
            x = x.to(torch.get_autocast_dtype(kind))
        sh, sw = self.stride
        # NHWC rows: a view of a channels-last tensor, strided ones copied
        rows = x[..., ::sh, ::sw].movedim(-3, -1)
        y = ops.mx4_linear(rows, self._mx4_weight(), self.bias)
        return y.movedim(-1, -3)                       # channels_last NCHW


def _state(w: torch.Tensor):
    """What changes with an update; None where updates leave no trace: codes
    of a parameter made in inference mode are made in every forward."""
    return None if w.is_inference() else (w.dtype, w._version)


def _nothing():
    """In the place of a reference to a weight."""


def use_mx4(module: nn.Module, train: bool = False) -> int:
    """Turns the 1x1 convolutions of ``module`` to 4-bit products
    (``ops.mx4_linear``: weights and inputs rounded to MX blocks along the
    channels, fp32 sums). Returns how many there are.

    ``train=False`` rounds the weights now and holds them in 4 bits, for
    inference. The forward that follows an update of a weight (an optimizer's,
    ``load_state_dict``'s, another parameter in its place) rounds it again.
    Updates that leave no trace, through ``.data`` or by a replayed training
    step, are not seen, and the replay of a captured forward sees none, until
    ``use_mx4`` is called again, which writes the new codes in the place of the
    old ones.
    ``train=True`` rounds them in every forward, with straight-through
    gradients to the float weights: fine-tuning for the former. The state dict
    stays what it was either way. ``use_mx4(model.features)`` leaves the
    add-on layers, which the densities read, in full precision."""
    n = 0
    for m in module.modules():
        if not isinstance(m, GemmConv2d) or not _plain_1x1(m):
            continue
        m.mx4 = 'train' if train else 'held'
        if not train:
            m._mx4_pack()
        n += 1
    return n


def no_mx4(module: nn.Module):
    """The reverse of ``use_mx4``."""
    for m in module.modules():
        if isinstance(m, GemmConv2d) and m.mx4 is not None:
            if hasattr(m, '_mx4_codes'):    # held now, or before training
                del m._mx4_codes, m._mx4_scales, m._mx4_of
            m.mx4 = None


def _plain_1x1(conv: nn.Conv2d) -> bool:
    return (conv.kernel_size == (1, 1) and conv.padding == (0, 0)
            and conv.groups == 1)
