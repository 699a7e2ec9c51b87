"""GELU of ops.linear_act over its whole range: every 16-bit value between -13 and 13 through a 1 x 1 identity weight, the
value and the slope relative to themselves, far into the negative tail."""
import math

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # half a step, relative
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}     # half of the smallest step


def _all_values(dtype, lo, hi):
    v = torch.from_numpy(np.arange(-32768, 32768).astype(np.int16)).view(dtype)
    return v[(v.double() >= lo) & (v.double() <= hi)].cuda()


def _phi(x):
    """(Phi(x), phi(x)) in 64 bits, without cancellation on either side"""
    return 0.5 * torch.erfc(x * -math.sqrt(0.5)), torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [0, 1])
def test_every_value(dtype, rows):
    """x as it is (one column), or in rows of 64 through a 64 x 64 identity (a bf16 / fp16 product by 1 and sums with 0 are
    exact).  Off by the rounding (half a step) and a quarter of it for the evaluation."""
    from hypdiff_amd import ops
    x = _all_values(dtype, -13.0, 13.0)
    if rows:
        x = torch.cat([x, x[:-x.numel() % 64]])
    m = x.reshape(-1, 64) if rows else x[:, None]
    w = torch.eye(m.shape[1], device="cuda").to(dtype)
    y = ops.linear_act(m, w, act="gelu").reshape(-1).double()
    z = x.double()
    want = z * _phi(z)[0]
    h = HALF[dtype]
    over = (y - want).abs() - (h * 1.25 * want.abs() + TINY[dtype])
    assert not bool((over > 0).any()), (float(z[over.argmax()]), float(((y - want) / want).abs()[z.abs() > 1e-3].max()))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_slope_of_every_value(dtype):
    """dL/dx for dL/dy = 1: the slope, at values that the kept fp16 pre-activation holds exactly.  Off by the rounding and a
    quarter of it; the error of Phi counts 1 / (x^2 - 1) there, an eighth below -3, and 2e-6 in absolute numbers above (the slope
    has a zero at -0.75)."""
    from hypdiff_amd import ops
    x = _all_values(dtype, -12.0, 12.0)
    x = x[x.half().double() == x.double()]
    leaf = x[:, None].detach().requires_grad_(True)
    dx = torch.autograd.grad(ops.linear_act(leaf, torch.ones(1, 1, device="cuda", dtype=dtype), act="gelu"), [leaf],
                             torch.ones(x.numel(), 1, device="cuda", dtype=dtype))[0].reshape(-1).double()
    z = x.double()
    Phi, phi = _phi(z)
    want = Phi + z * phi
    over = (dx - want).abs() - (HALF[dtype] * 1.25 * want.abs() + TINY[dtype] + 2e-6 * (z > -3).double())
    assert not bool((over > 0).any()), float(z[over.argmax()])
