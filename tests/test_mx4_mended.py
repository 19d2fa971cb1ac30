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
