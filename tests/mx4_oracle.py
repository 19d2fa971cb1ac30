"""MX4 rounding and its product from the definition, in 64 bits, apart from
the framework's own forms."""

import math

import torch

GRID = torch.tensor([0., .5, 1., 1.5, 2., 3., 4., 6.], dtype=torch.float64)


def values(x: torch.Tensor) -> torch.Tensor:
    """[M, K] -> the values of its blocks, float64 on the CPU."""
    x = x.detach().double().cpu()
    out = torch.zeros_like(x)
    mid = (GRID[1:] + GRID[:-1]) / 2
    for at in range(0, x.shape[1], 32):
        blk = x[:, at:at + 32]
        a = blk.abs().amax(dim=1)
        e = torch.tensor([max(-127, min(127, math.frexp(v)[1] - 3))
                          if v > 0 and math.isfinite(v) else -127
                          for v in a.tolist()], dtype=torch.float64)
        unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), e)[:, None]
        r = blk.abs() / unit
        low = torch.bucketize(r, mid, right=False)
        high = torch.bucketize(r, mid, right=True)
        code = torch.where(low % 2 == 0, low, high)
        v = torch.copysign(GRID[code] * unit, blk)
        v[~torch.isfinite(a)] = math.nan
        out[:, at:at + 32] = v
    return out


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def assert_close(got: torch.Tensor, want: torch.Tensor, mass: torch.Tensor,
                 terms: int):
    """got is want (64 bits) summed in fp32 and rounded once. A sum of n terms
    in any order, each addition off by at most one step 2^-23 of what it has
    so far, is off by at most n 2^-23 mass, where mass is the sum of the
    terms' absolute values; the rounding adds half a step of the result, or of
    the smallest normal number."""
    h = half_step(got.dtype)
    slack = terms * 2.0 ** -23 * mass
    tol = slack + h * (want.abs() + slack) \
        + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    diff = (got.detach().double().cpu() - want).abs()
    bad = ~(diff <= tol)
    assert not bad.any(), (
        f'{int(bad.sum())} of {bad.numel()} off, worst '
        f'{float((diff / tol.clamp(min=1e-300)).max()):.3g} x the bound at '
        f'{bad.nonzero()[0].tolist()}')
