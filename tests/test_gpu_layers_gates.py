"""The gate functions and their derivatives where they are small, number by number against 64 bits.

x picks single weights, so that every projection is exact and what is left is the gate's own error and the result's rounding.

The gate in 32 bits, relative to the value (EPS = 2^-24, half a step):
  exp(x) is 2^(x log2 e) with the product rounded: |x| * EPS, and |x| * EPS / 4 for the constant; the hardware's power of two 2^-22
  1 / x 2^-23; a rounding EPS
  silu       exponent g, then 1 + e, the reciprocal and a product
  gelu_tanh  the same for 2 sqrt(2 / pi) (g + 0.044715 g^3), which takes seven roundings and constants
  gelu       exponent g^2 / 2, which rounds once more; the rest (reciprocal, polynomial of degree 7, its fit) below 2^-19
An exponential or a reciprocal below 2^-126 comes as zero: the gate may be off by |g| * 2^-126."""
import math

import pytest
import torch

from tilebench_b200.benchmarks.layers.ffn_gated import impl_cuda as ffn
from tilebench_b200.benchmarks.layers.ffn_gated_bwd import impl_cuda as bwd
from tilebench_b200.data import tensors
from test_gpu_layers import ACTS, TINY, clean_status, gen, half_step, normal    # noqa: F401

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
FLUSH = 2.0 ** -126
A, B = math.sqrt(2 / math.pi), 0.044715
RANGES = [(-60.0, 60.0), (-14.0, 6.0), (-1.0, 1.0)]


def exp_error(x):
    return x.abs() * 1.25 * EPS + 2.0 ** -22


def value_error(g, act):
    """Relative error of f(g) in 32 bits."""
    if act == "silu":
        return exp_error(g) + 2.0 ** -23 + 3 * EPS
    if act == "gelu":
        return exp_error(g * g / 2) + g * g / 2 * EPS + 2.0 ** -19
    if act == "gelu_tanh":
        y = 2 * A * (g + B * g ** 3)
        return exp_error(y) + y.abs() * 7 * EPS + 2.0 ** -23 + 3 * EPS
    return torch.zeros_like(g)


def slope_error(g, act):
    """Error of f'(g) in 32 bits: of each of its terms, which may cancel, and of 1 - s by 2^-21."""
    e = value_error(g, act) + 2.0 ** -21
    if act == "silu":
        s = torch.sigmoid(g)
        return e * (s + s * g.abs() * (1 - s)) + g.abs() * s * 2.0 ** -21
    if act == "gelu":
        p = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        return e * (p + g.abs() * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        s, steep = torch.sigmoid(2 * A * (g + B * g ** 3)), 2 * A * g.abs() * (1 + 3 * B * g * g)
        return e * (s + s * (1 - s) * steep) + s * steep * 2.0 ** -21
    return torch.zeros_like(g)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [3, 40, 100, 200, 1100])
def test_values_in_the_tails(cuda_device, m, act, dtype):
    k, f = 64, 160
    x = torch.zeros(m, k, dtype=dtype, device="cuda")
    pick = torch.arange(m, device="cuda") % k
    x[torch.arange(m, device="cuda"), pick] = 1
    for low, high in RANGES:
        wg = torch.linspace(low, high, f * k, device="cuda").view(f, k).to(dtype)
        wu = normal(gen(m), f, k, dtype=dtype)
        g, u = wg.double().t()[pick], wu.double().t()[pick]
        want = tensors.gate(g, act)[0] * u
        tol = (value_error(g, act) + EPS) * want.abs() + g.abs() * FLUSH * u.abs()
        tol = tol + half_step(dtype) * (want.abs() + tol) + TINY[dtype]
        for h in (ffn.run(x, wg, wu, act), ffn.run(x, wg, wu, act, checkpoint=True)[0]):
            bad = (h.double() - want).abs() > tol
            assert not bool(bad.any()), (g[bad][:4], u[bad][:4], h[bad][:4], want[bad][:4])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("k,f", [(160, 160), (168, 163)])
def test_gradients_in_the_tails(cuda_device, k, f, act, dtype):
    """One token and weights that pick: dg is a column of dWg, and a row of dx where Wg is the unit matrix; du the same."""
    unit = torch.zeros(f, k, dtype=dtype, device="cuda")
    unit[torch.arange(f), torch.arange(f)] = 1
    zero = torch.zeros_like(unit)
    x = torch.zeros(1, k, dtype=dtype, device="cuda")
    x[0, 2] = 1
    us = torch.ones(1, -(-f // 128), device="cuda")
    uq = torch.ones(1, f, device="cuda").to(torch.float8_e4m3fn)                 # u = 1
    for low, high in RANGES:
        gq, gs = tensors.checkpoint_fp8(torch.linspace(low, high, f, device="cuda")[None])
        g = gq.double() * gs.double().repeat_interleave(128, dim=1)[:, :f]
        dh = (1 + torch.rand(1, f, generator=gen(f), device="cuda")).to(dtype)
        a, da = tensors.gate(g, act)
        # in fp16, dg and du are held times a power of two: see test_gpu_layers_fp16.py
        small = 2.0 ** -29 * float(dh.double().max()) * max(1.0, float(gs.max())) if dtype == torch.float16 else TINY[dtype]
        flush = 16 * (1 + g * g) * FLUSH
        want = (dh.double() * da, dh.double() * a)
        off = (dh.double() * (slope_error(g, act) + flush), dh.double() * (value_error(g, act) * a.abs() + flush))
        for i, weights in enumerate(((unit, zero), (zero, unit))):
            dx, dwg, dwu = bwd.run(dh, *weights, x, None, gq, gs, uq, us, act)
            tol = (1 + 2 * EPS) * off[i] + 2 * EPS * want[i].abs()
            tol = tol + half_step(dtype) * (want[i].abs() + tol) + small
            tol = tol + half_step(dtype) * (want[i].abs() + tol) + TINY[dtype]
            for got in (dx[:, :f], (dwg, dwu)[i][:, 2][None]):
                bad = (got.double() - want[i]).abs() > tol
                assert not bool(bad.any()), (g[bad][:4], got[bad][:4], want[i][bad][:4])
            assert not dx[:, f:].any() and not dwg[:, :2].any() and not dwu[:, 3:].any()
