"""Gradients of the feed-forward block in fp16 of any size: what an fp16 result can hold is not lost in dg and du.

Tolerances.  dg and du are kept as fp16 numbers times one power of two, which brings max|dh| * 512 * max(scale of g or u), a bound of
both, to between 2^13 and 2^15.  The spacing of the subnormal numbers is 2^-24 there, half of it 2^-25: so beside the rounding of
E = 2^-11 of its value each term is off by at most 2^-25 * 2^-13 of the bound = 2^-29 * max|dh| * max(scale).  Sums and gate functions as
in test_gpu_layers.py; the result rounds once more, to half of 2^-24 where it is subnormal."""
import math

import pytest
import torch

from tilebench_b200 import native
from tilebench_b200.benchmarks.layers.ffn_gated_bwd import impl_cuda as bwd
from tilebench_b200.data import tensors

pytestmark = pytest.mark.gpu

E, GATE, TOP = 2.0 ** -11, 2.0 ** -19, 65504.0


@pytest.fixture(autouse=True)
def clean_status():
    yield
    assert native.device_status()[0] == 0


def inputs(m, k, f, dh_size, weight=None, u_size=2.0, seed=0, x_codes=True):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 3 * k + 5 * f)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    x = normal(m, k).half()
    wg, wu = ((normal(f, k) * (k ** -0.5 if weight is None else weight)).half() for _ in range(2))
    dh = (normal(m, f) * dh_size).clamp(-TOP, TOP).half()
    held = [*tensors.checkpoint_fp8(normal(m, f) * 2.0), *tensors.checkpoint_fp8(normal(m, f) * u_size)]
    return dh, wg, wu, *(tensors.checkpoint_fp8(x) if x_codes else (x, None)), *held


def check(got, args, act):
    dh, wg, wu, x, xs, gq, gs, uq, us = args

    def held(q, s):
        return q.double() * s.double().repeat_interleave(128, dim=1)[:, :q.shape[1]]
    x = x.double() if xs is None else held(x, xs)
    g, u = held(gq, gs), held(uq, us)
    a, da = tensors.gate(g, act)
    dh, wg, wu = dh.double(), wg.double(), wu.double()
    dg, du = dh * u * da, dh * a
    spacing = 2.0 ** -29 * float(dh.abs().max()) * float(torch.maximum(gs.abs().max(), us.abs().max()))
    # error of each term of dg: f' may cancel where f is steep, so its error is GATE of |dh u|
    eg, eu = E * dg.abs() + GATE * (dh * u).abs() + spacing, (E + GATE) * du.abs() + spacing
    want = (dg @ wg + du @ wu, dg.t() @ x, du.t() @ x)
    off = (eg @ wg.abs() + eu @ wu.abs(), eg.t() @ x.abs(), eu.t() @ x.abs())
    size = (dg.abs() @ wg.abs() + du.abs() @ wu.abs(), dg.abs().t() @ x.abs(), du.abs().t() @ x.abs())
    for t, w, o, s, n in zip(got, want, off, size, (2 * dh.shape[1], dh.shape[0], dh.shape[0])):
        tol = o + (n / 16 + 16) * 2.0 ** -23 * s
        tol = tol + E * (w.abs() + tol) + 2.0 ** -25
        fits = w.abs() + tol <= TOP                          # beyond, the result itself may round to infinity
        assert t.dtype == torch.float16 and bool(fits.any())
        assert bool(((t.double() - w).abs() <= tol)[fits].all())


@pytest.mark.parametrize("dh_size", [1e-6, 1e-5, 1e-3, 1.0])
@pytest.mark.parametrize("m,k,f", [(1, 64, 130), (48, 136, 200), (129, 264, 333), (700, 136, 256), (3000, 136, 140), (60, 4104, 6500)])
def test_small_gradients_keep_their_bits(cuda_device, m, k, f, dh_size):
    args = inputs(m, k, f, dh_size, x_codes=m % 2 == 0)
    check(bwd.run(*args, "silu"), args, "silu")


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_small_gradients_of_every_gate(cuda_device, act):
    args = inputs(300, 72, 264, 3e-6)
    check(bwd.run(*args, act), args, act)


@pytest.mark.parametrize("m,k,f", [(5, 64, 128), (129, 264, 333), (700, 136, 256)])
def test_large_gradients_stay_finite(cuda_device, m, k, f):
    """dg of some 1e6, beyond fp16, times weights (and inputs) that bring the results back into its range."""
    args = list(inputs(m, k, f, 2e4, weight=2.0 ** -12, u_size=60.0, x_codes=False))
    args[3] = (args[3].float() * 2.0 ** -12).half()
    got = bwd.run(*args, "silu")
    assert all(bool(t.isfinite().all()) for t in got)
    check(got, args, "silu")


def test_infinities_and_nan_stay_in_their_places(cuda_device):
    """They do not enter the power of two: the other rows of dx keep small gradients, the other columns of the weights' too."""
    args = list(inputs(40, 64, 136, 1e-6, x_codes=False))
    clean = bwd.run(*args, "silu")
    dh = args[0].clone()
    dh[7, 3], dh[9, 5] = math.inf, math.nan
    got = bwd.run(dh, *args[1:], "silu")
    rows = torch.ones(40, dtype=torch.bool, device="cuda")
    rows[[7, 9]] = False
    units = torch.ones(136, dtype=torch.bool, device="cuda")
    units[[3, 5]] = False
    assert torch.equal(got[0][rows], clean[0][rows]) and not got[0][~rows].isfinite().any()
    for a, b in zip(got[1:], clean[1:]):
        assert torch.equal(a[units], b[units]) and not a[~units].isfinite().any()


@pytest.mark.parametrize("offset", [1, 3, 8, 15])
@pytest.mark.parametrize("at", [0, 1, -1, None])
def test_the_largest_gradient_anywhere(cuda_device, offset, at):
    """dh at any address; its one large number, first, second or last, sets the power of two, and what lies around dh does not."""
    m, k, f = 3, 64, 331
    args = list(inputs(m, k, f, 1e-4, weight=2.0 ** -12, u_size=60.0, x_codes=False))
    args[3] = (args[3].float() * 2.0 ** -12).half()
    if at is not None:
        args[0].view(-1)[at] = 6e4
    args[7][:, :], args[8][:, :] = torch.tensor(448.0, device="cuda").to(torch.float8_e4m3fn), 1.0            # u = 448
    args[5][:, :], args[6][:, :] = torch.tensor(8.0, device="cuda").to(torch.float8_e4m3fn), 1.0              # f'(8) is near 1
    flat = torch.full((m * f + 64,), 6e4, dtype=torch.float16, device="cuda")                                # not dh's
    flat[offset:offset + m * f] = args[0].view(-1)
    args[0] = flat[offset:offset + m * f].view(m, f)
    got = bwd.run(*args, "silu")
    assert all(bool(t.isfinite().all()) for t in got)
    check(got, args, "silu")


def test_gradients_of_nothing(cuda_device):
    args = list(inputs(20, 64, 130, 1.0))
    args[0].zero_()
    assert all(not t.any() for t in bwd.run(*args, "gelu"))
    args = list(inputs(20, 64, 130, 1e-5))
    for i in (5, 7):
        args[i] = torch.zeros_like(args[i])
    got = bwd.run(*args, "silu")
    assert all(not t.any() for t in got)


def test_tensors_scaled_by_powers_of_two_give_the_same_bits(cuda_device):
    """A power of two in dh goes through to the gradients, as long as these stay normal numbers."""
    args = list(inputs(130, 136, 264, 1.0))
    dh = args[0] = ((args[0] * 8).round() / 8).half()
    want = bwd.run(*args, "silu")
    args[0] = (dh.float() * 2.0 ** -6).half()
    assert bool((args[0].float() * 64 == dh.float()).all())
    for a, b in zip(bwd.run(*args, "silu"), want):
        normal = b.abs() >= 2.0 ** -8
        assert torch.equal(a[normal].float() * 64, b[normal].float())


@pytest.mark.parametrize("m", [1, 40, 300])
def test_captured_behind_copies_fills_and_another_stream(cuda_device, m):
    """The first kernel of a call begins over the end of what comes before it: a copy, a fill, another stream's work, a call of its own kind."""
    k, f = 136, 200
    dh, wg, wu, x, xs, *held = inputs(m, k, f, 1e-5)
    source, weight = dh.clone(), wg.clone()
    into, w, zeros = torch.empty_like(dh), torch.empty_like(wg), torch.ones_like(dh)
    side = torch.cuda.Stream()

    def step():
        into.copy_(source)
        first = bwd.run(into, wg, wu, x, xs, *held, "silu")
        zeros.zero_()
        none = bwd.run(zeros, wg, wu, x, xs, *held, "silu")
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            w.copy_(weight)
            into.mul_(4096.0)
        torch.cuda.current_stream().wait_stream(side)
        return (*first, *none, *bwd.run(into, w, wu, x, xs, *held, "gelu"), *bwd.run(into, wg, w, x, xs, *held, "relu"))

    def expected():
        a, big, b = source.clone(), source * 4096.0, weight.clone()
        torch.cuda.synchronize()
        none = [torch.zeros_like(t) for t in bwd.run(a, wg, wu, x, xs, *held, "silu")]
        return (*bwd.run(a, wg, wu, x, xs, *held, "silu"), *none, *bwd.run(big, b, wu, x, xs, *held, "gelu"), *bwd.run(big, wg, b, x, xs, *held, "relu"))
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    g = torch.Generator(device="cuda").manual_seed(m)
    for turn in range(4):
        source.copy_(torch.randn(m, f, generator=g, device="cuda") * 10.0 ** -(2 + turn))
        weight.copy_(torch.randn(f, k, generator=g, device="cuda") * 0.1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expected()))
        assert all(torch.equal(a, b) for a, b in zip(step(), expected()))
        torch.cuda.synchronize()


def test_calls_of_different_size_on_two_streams_at_once(cuda_device):
    sets = [inputs(64 + 200 * i, 512, 640, 10.0 ** -(1 + 4 * i), seed=i) for i in range(2)]
    want = [bwd.run(*args, "silu") for args in sets]
    for args, grads in zip(sets, want):
        check(grads, args, "silu")
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(bwd.run(*sets[i], "silu"))
    torch.cuda.synchronize()
    for i in range(2):
        for grads in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(grads, want[i]))
