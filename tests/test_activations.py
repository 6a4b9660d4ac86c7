"""The activations and their slopes, value by value, against float64 over the whole range: the norm layer with
weight 0 is act(bias), and its bias gradient for an upstream gradient of 1 is act'(bias).

Bounds, in units of 2^-24 of the value: 2^x is off by at most 2 units in the last place (4 of 2^-24), a reciprocal by
one (2), each other operation by one. A result in 16 bits adds its own rounding, 2^-8 (bf16) or 2^-11 (f16) of the value."""

import math

import pytest
import torch

from spectral.nn import group_norm_act

UNIT = 2.0 ** -24
ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def sweep(lo, hi, activation, dtype):
    """z, act(z) in dtype, act'(z) in float32 as the backward pass of dtype uses it."""
    z = torch.linspace(lo, hi, 1 << 20, device="cuda")
    x = torch.randn(1, 1, z.numel(), device="cuda").to(dtype)
    bias = z.clone().requires_grad_(True)
    y = group_norm_act(x, 1, torch.zeros_like(z), bias, activation=activation)
    (slope,) = torch.autograd.grad(y, bias, torch.ones_like(y))
    return z.double(), y.detach().reshape(-1).double(), slope.double()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(ROUND))
@pytest.mark.parametrize(("lo", "hi"), [(-87.0, -20.0), (-20.0, 20.0), (-1.5, 1.5)])
def test_silu(lo, hi, dtype):
    z, y, slope = sweep(lo, hi, "silu", dtype)
    s = torch.sigmoid(z)
    # 2^x and the reciprocal, the sum, the product; float32 carries the exponent's rounding, 16 bits do not.
    single = (10.0 if dtype == torch.float32 else 10.0 + z.abs()) * UNIT
    assert ((y - z * s).abs() <= (single + ROUND[dtype]) * (z * s).abs() + LEAST[dtype]).all()
    terms = s + (z * s * (1 - s)).abs()  # the slope may cancel
    assert ((slope - s * (1 + z * (1 - s))).abs() <= (single + 3 * UNIT) * terms + LEAST[torch.float32]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", list(ROUND))
def test_far_from_zero(activation, dtype):
    # Far below zero the values vanish, far above they are z itself; infinities and NaN do not turn into numbers.
    z = torch.tensor([-3e38, -1e30, -1e4, -200.0, 30.0, 200.0, 1e4, 1e30, math.inf, math.nan, -0.0, 0.0], device="cuda")
    y = group_norm_act(torch.randn(1, 1, z.numel(), device="cuda").to(dtype), 1, torch.zeros_like(z), z, activation=activation).reshape(-1)
    assert (y[:4].abs() <= 2.0 ** -126).all() and torch.equal(y[4:9], z[4:9].to(dtype)) and y[9].isnan() and (y[10:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(ROUND))
@pytest.mark.parametrize(("lo", "hi"), [(-12.5, -6.2), (-6.2, 6.2), (-1.5, 1.5), (6.2, 20.0)])
def test_gelu(lo, hi, dtype):
    z, y, slope = sweep(lo, hi, "gelu", dtype)
    phi, tail = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi), 0.5 * torch.special.erfc(-z / math.sqrt(2))
    # 2^x 4 and its exponent's two roundings z^2, the reciprocal and its argument 3, the polynomial 2 and its fit 2, the
    # products 3; in the 16-bit types the fit is off by 2.2e-6, far below zero by 5e-5.
    fit = 2 * UNIT if dtype == torch.float32 else 2.2e-6 if lo >= -6.2 else 5e-5
    single = fit + (14 + z * z) * UNIT
    assert ((y - z * tail).abs() <= (single + ROUND[dtype]) * (z * tail).abs() + LEAST[dtype]).all()
    assert ((slope - (tail + z * phi)).abs() <= (single + 3 * UNIT) * (tail + z.abs() * phi) + LEAST[torch.float32]).all()
