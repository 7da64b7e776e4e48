"""Activations of an epilogue over the whole range of their argument: a product of zero rows leaves the bias as the argument, exactly."""

from __future__ import annotations

import math

import pytest
import torch
from test_gpu_grouped import DEV, grouped_case, offsets_of

from mase_triton_b200.mxfp.layers import MXFPLinearPTQ
from mase_triton_b200.mxfp.meta import MXFP8_E4M3_fn

pytestmark = pytest.mark.gpu


def arguments(dtype):
    z = torch.cat([torch.linspace(-110, 110, 2201), torch.linspace(-89, -87, 257), torch.linspace(-6, 6, 257),
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 300.0, -300.0, 1e4, -1e4, 6e4, -6e4, 1e13, -1e13, 3e38, -3e38, float("inf"), float("nan")])]).double()
    return z.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).where(z.isfinite(), z).to(dtype).to(DEV)


def formula(z, activation):
    """(y, relative error of the value that is rounded).

    With t = exp(-|a|), y = z t / (1 + t) or z / (1 + t): the exponential is within 2 ulp, the division too, sum and product are half
    an ulp each: 5 ulp of 2^-23.  gelu_tanh: a has seven roundings of 2^-24 (square, cube, two constants and their products, one sum), and
    its error counts |a| times in t.  (16-bit types take a fast exponential, off by up to |a| 2^-24: the half step of the result covers it
    unless the value lies that close to a tie, which none of these does.)"""
    w = z.double()
    if activation == "silu":
        return w / (1 + torch.exp(-w)), torch.full_like(w, 5 * 2.0**-23)
    a = 2 * math.sqrt(2 / math.pi) * (w + 0.044715 * w**3)
    return w / (1 + torch.exp(-a)), 5 * 2.0**-23 + 8 * 2.0**-24 * a.abs().clamp(max=200)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M", [3, 200])
def test_whole_range(lib, dtype, activation, M):
    z = arguments(dtype)
    layer = MXFPLinearPTQ(torch.ones(z.numel(), 32, dtype=dtype, device=DEV), z, MXFP8_E4M3_fn, MXFP8_E4M3_fn, None, "XqWqB", "fused")
    got = layer(torch.zeros(M, 32, dtype=dtype, device=DEV), activation=activation)
    y, relative = formula(z, activation)
    # below the normal range of fp32 an ulp of t is 2^-149, times |z| (at most 104 there); the output's own half step, subnormals included
    tol = relative * y.abs() + 2.0**-140
    tol = tol + torch.finfo(dtype).eps / 2 * (y.abs() + tol) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    finite = z.isfinite()
    assert torch.equal(got[0].isnan(), z.isnan()) and bool((got[:, z.isposinf()] == math.inf).all())
    off = ((got.double() - y).abs() - tol)[:, finite]
    worst = off.max(0).values.argmax()
    assert bool((off <= 0).all()), f"{int((off > 0).any(0).sum())} arguments, worst at {z[finite][worst].item()}: {got[0, finite][worst].item()} for {y[finite][worst].item()}"


def test_tail_times_a_large_multiplier(lib):
    """What lies far out in the tail is no zero: the multiplier may bring it back."""
    layer, _, _, x = grouped_case([4], 64, 32, MXFP8_E4M3_fn, MXFP8_E4M3_fn, torch.float32)
    layer.bias.data.fill_(-88.0)
    m = torch.full((4, 64), 2.0**120, device=DEV)
    got = layer(torch.zeros_like(x), offsets_of([4]), activation="silu", multiplier=m)
    want = -88.0 / (1 + math.exp(88.0)) * 2.0**120
    # t = exp(-88) is subnormal: an ulp of 2^-149 beside 6.05e-39, i.e. 2^-21.9 of it, twice; the rest as above
    assert bool(((got.double() - want).abs() <= (2.0**-20 + 5 * 2.0**-23 + 2.0**-24) * abs(want)).all()), got[0, 0].item() / want
