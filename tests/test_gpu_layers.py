"""The layer operators on the GPU against their formulas in 64 bits.

Tolerances.  A rounding is off by half a step at most: E = finfo.eps / 2 of the value (and half the spacing of the
subnormal numbers, TINY).  A product of depth n summed in 32 bits, in steps of 16, is off by at most (n / 16 + 16) * 2^-23 of
the sum of magnitudes (each step may truncate).  Gate functions are evaluated to 2^-19 of the value in 32 bits."""
import subprocess
import sys

import pytest
import torch

from tilebench_b200 import native
from tilebench_b200.benchmarks.layers.act_checkpoint_fp8 import impl_cuda as save
from tilebench_b200.benchmarks.layers.act_restore_fp8 import impl_cuda as restore
from tilebench_b200.benchmarks.layers.ffn_gated import impl_cuda as ffn
from tilebench_b200.benchmarks.layers.ffn_gated_bwd import impl_cuda as bwd
from tilebench_b200.core.engine import run_benchmark_suite
from tilebench_b200.data import tensors
from tilebench_b200.paths import REPO_ROOT

pytestmark = pytest.mark.gpu

ACTS = ("silu", "gelu", "gelu_tanh", "relu")
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
GATE = 2.0 ** -19


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def depth_error(n):
    return (n / 16 + 16) * 2.0 ** -23


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def same_codes(q, want):
    a, b = q.float(), want.float()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.fixture(autouse=True)
def clean_status(request):
    yield
    if torch.cuda.is_available():
        assert native.device_status()[0] == 0


# ---- saving and restoring --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (1, 8, 0), (3, 127, 0), (5, 128, 0), (5, 128, 8), (7, 136, 0), (2, 1023, 3),
                                           (3, 1024, 0), (3, 1025, 7), (9, 4096, 0), (33, 5461, 11), (17, 2056, 8), (300, 40, 0)])
def test_save_and_restore_are_exact(cuda_device, rows, cols, pad, dtype):
    g = gen(rows * 10007 + cols)
    wide = normal(g, rows, cols + pad) * torch.exp(3 * normal(g, rows, 1))
    x = wide.to(dtype)[:, :cols]
    q, s = save.run(x)
    want_q, want_s = tensors.checkpoint_fp8(x)
    assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))
    for out in (torch.float32, torch.float16, torch.bfloat16):
        got = restore.run(q, s, out)
        assert got.dtype == out and torch.equal(got, tensors.restore_fp8(q, s, out))
    if dtype != torch.float16:                               # restoring to 32 bits is exact, and bf16 holds the same numbers
        assert torch.equal(restore.run(q, s, torch.bfloat16).float(), restore.run(q, s, torch.float32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,pad", [(5, 2060, 0), (5, 2060, 4), (40, 1032, 8), (3, 5464, 8), (70, 8, 8), (6, 140, 4), (3, 2049, 1), (900, 130, 3)])
def test_save_and_restore_by_pieces_of_every_width(cuda_device, rows, cols, pad, dtype):
    g = gen(rows + 17 * cols)
    x = (normal(g, rows, cols + pad) * torch.exp(2 * normal(g, rows, 1))).to(dtype)[:, :cols]
    x[0, -1], x[-1, 0] = float("inf"), float("nan")
    q, s = save.run(x)
    want_q, want_s = tensors.checkpoint_fp8(x)
    assert torch.equal(s, want_s) and same_codes(q, want_q)
    assert same_codes(restore.run(q, s, dtype), tensors.restore_fp8(want_q, want_s, dtype))


@pytest.mark.parametrize("offset", [1, 3, 8])
def test_save_and_restore_at_odd_addresses(cuda_device, offset):
    """Views that begin at any element, codes that begin at any byte; what lies around the outputs stays."""
    ext = native.load()
    rows, cols = 6, 260
    x = normal(gen(offset), rows * cols + offset, dtype=torch.bfloat16)[offset:].view(rows, cols)
    codes = torch.full((rows * cols + 64,), 0x55, dtype=torch.uint8, device="cuda")
    q = codes[offset:offset + rows * cols].view(rows, cols).view(torch.float8_e4m3fn)
    scales = torch.full((rows * 3 + 2,), -7.0, device="cuda")
    s = scales[1:-1].view(rows, 3)
    ext.act_checkpoint_fp8(x, q, s)
    want_q, want_s = tensors.checkpoint_fp8(x)
    assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s, want_s)
    assert scales[0] == -7 and scales[-1] == -7
    assert bool((codes[:offset] == 0x55).all()) and bool((codes[offset + rows * cols:] == 0x55).all())
    back = torch.full((rows * cols + 32,), 9.0, dtype=torch.float16, device="cuda")
    out = back[offset:offset + rows * cols].view(rows, cols)
    ext.act_restore_fp8(q, s, out)
    assert torch.equal(out, tensors.restore_fp8(want_q, want_s, torch.float16))
    assert bool((back[:offset] == 9).all()) and bool((back[offset + rows * cols:] == 9).all())


@pytest.mark.parametrize("cols", [128, 200, 331])
def test_save_special_values(cuda_device, cols):
    inf, nan = float("inf"), float("nan")
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        info = torch.finfo(dtype)
        x = torch.zeros(9, cols, dtype=dtype, device="cuda")
        x[1, :3] = torch.tensor([inf, -inf, nan])
        x[2, :4] = torch.tensor([inf, 3.0, nan, -5.0])
        x[3, 0], x[3, 1] = info.max, -info.max
        x[4, 0] = info.smallest_normal
        x[5, 0] = info.smallest_normal * info.eps            # the smallest subnormal number
        x[6, :2] = torch.tensor([448.0, 450.0])
        x[7] = nan
        x[8, -1] = -1.0
        q, s = save.run(x)
        want_q, want_s = tensors.checkpoint_fp8(x)
        assert torch.equal(s, want_s) and same_codes(q, want_q)
        back, want = restore.run(q, s, dtype), tensors.restore_fp8(want_q, want_s, dtype)
        assert same_codes(back, want)
        assert back[3, 0] == info.max and back[3, 1] == -info.max


def test_every_code_is_restored(cuda_device):
    q = torch.arange(256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).repeat(4, 1)
    s = torch.tensor([[1.0, 2.0 ** -126], [2.0 ** 120, 0.25], [2.0 ** -20, 2.0 ** 7], [2.0 ** -140, 3.0]], device="cuda")
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        assert same_codes(restore.run(q, s, dtype), tensors.restore_fp8(q, s, dtype))
        assert same_codes(restore.run(q[:, :250].contiguous(), s, dtype), tensors.restore_fp8(q[:, :250], s, dtype))


@pytest.mark.parametrize("cols", [256, 250, 131, 15])
def test_scales_of_either_sign_and_any_size(cuda_device, cols):
    """Scales need not be act_checkpoint_fp8's own: products beyond the type's range are held to it on either side."""
    g = gen(cols)
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    q = codes[torch.randint(0, 256, (64, cols), generator=g, device="cuda")]
    blocks = (cols + 127) // 128
    s = torch.exp2(torch.randint(-140, 128, (64, blocks), generator=g, device="cuda").float()) * (1 + torch.rand(64, blocks, generator=g, device="cuda"))
    s[::2] *= -1
    s[5, 0], s[6, 0], s[7, -1] = float("inf"), -float("inf"), float("nan")
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        assert same_codes(restore.run(q, s, dtype), tensors.restore_fp8(q, s, dtype))


# ---- forward -----------------------------------------------------------------------------------------

def block_inputs(m, k, f, dtype, seed=0, pad=0):
    g = gen(seed + 7919 * m + 31 * k + f)
    x = normal(g, m, k + pad, dtype=dtype)[:, :k]
    wg, wu = (normal(g, f, k, scale=k ** -0.5, dtype=dtype) for _ in range(2))
    return x, wg, wu


def forward64(x, wg, wu, act):
    """h, g, u in 64 bits, and bounds of what 32-bit sums may be off by in g and u."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    d = depth_error(x.shape[1])
    return tensors.gate(g, act)[0] * u, g, u, d * (x.abs() @ wg.abs().t()), d * (x.abs() @ wu.abs().t())


def check_h(h, x, wg, wu, act):
    want, g, u, eg, eu = forward64(x, wg, wu, act)
    # |f'| <= 1.13 for all four gates, and |f(g)| <= |g|
    tol = 1.13 * eg * (u.abs() + eu) + g.abs() * eu + GATE * want.abs()
    tol = tol + half_step(h.dtype) * (want.abs() + tol) + TINY[h.dtype]
    assert bool(((h.double() - want).abs() <= tol).all())


def check_held(q, s, v, e):
    """Codes and scales of a 64-bit activation v that was computed with an error of at most e."""
    m, f = v.shape
    pad = (0, s.shape[1] * 128 - f)
    size = torch.nn.functional.pad(v.abs(), pad).view(m, -1, 128)
    off = torch.nn.functional.pad(e, pad).view(m, -1, 128)
    low = tensors.checkpoint_fp8((size - off).clamp(min=0).amax(dim=2).float().view(-1, 1))[1].view_as(s)
    high = tensors.checkpoint_fp8((size + off).amax(dim=2).float().view(-1, 1))[1].view_as(s)
    assert bool(((s == low) | (s == high)).all())
    back = q.double() * s.double().repeat_interleave(128, dim=1)[:, :f]
    step = s.double().repeat_interleave(128, dim=1)[:, :f] * 2.0 ** -10
    assert bool(((back - v).abs() <= torch.maximum((v.abs() + e) * 2.0 ** -4, step) + e).all())


SIZES = [(1, 8, 1), (1, 64, 128), (2, 72, 7), (5, 136, 130), (16, 256, 264), (17, 1048, 333), (64, 512, 96), (127, 128, 129), (128, 200, 256),
         (129, 64, 128), (255, 520, 135), (256, 1024, 384), (300, 264, 1001)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,f", SIZES)
def test_forward(cuda_device, m, k, f, dtype):
    x, wg, wu = block_inputs(m, k, f, dtype)
    act = ACTS[(m + k + f) % 4]
    h = ffn.run(x, wg, wu, act)
    check_h(h, x, wg, wu, act)
    h2, gq, gs, uq, us = ffn.run(x, wg, wu, act, checkpoint=True)
    check_h(h2, x, wg, wu, act)
    _, g, u, eg, eu = forward64(x, wg, wu, act)
    check_held(gq, gs, g, eg)
    check_held(uq, us, u, eu)


@pytest.mark.parametrize("m,k,f", [(129, 64, 9), (200, 520, 136), (247, 2048, 1164), (513, 4096, 70), (1000, 1024, 264), (1024, 4104, 131), (1025, 512, 64)])
def test_forward_of_rows_in_blocks(cuda_device, m, k, f):
    """More than 128 rows and few hidden units: blocks of 128 rows on narrow tiles, with and without shares of the contraction."""
    x, wg, wu = block_inputs(m, k, f, torch.bfloat16, pad=8)
    h = torch.full((m + 2, f), 7.0, dtype=torch.bfloat16, device="cuda")
    native.load().ffn_gated(x, wg, wu, h[1:-1], native.activation("silu"), None, None, None, None)
    check_h(h[1:-1], x, wg, wu, "silu")
    assert bool((h[0] == 7).all()) and bool((h[-1] == 7).all())


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [3, 40, 200])
def test_forward_gates_over_their_range(cuda_device, act, m):
    """Projections from -60 to 60: x picks single weights."""
    k, f = 64, 160
    x = torch.zeros(m, k, dtype=torch.float16, device="cuda")
    x[torch.arange(m), torch.arange(m) % k] = 1
    wg = torch.linspace(-60, 60, f * k, device="cuda").view(k, f).t().contiguous().half()
    wu = normal(gen(m), f, k, dtype=torch.float16)
    check_h(ffn.run(x, wg, wu, act), x, wg, wu, act)
    check_h(ffn.run(x, wg, wu, act, checkpoint=True)[0], x, wg, wu, act)


@pytest.mark.parametrize("m", [1, 4, 100, 260])
def test_forward_strided_rows_and_slices_of_a_joint_weight(cuda_device, m):
    x, _, _ = block_inputs(m, 136, 1, torch.bfloat16, pad=24)
    both = normal(gen(m), 2 * 200, 136, scale=0.1, dtype=torch.bfloat16)
    assert m == 1 or x.stride(0) == 160
    check_h(ffn.run(x, both[:200], both[200:], "silu"), x, both[:200], both[200:], "silu")


@pytest.mark.parametrize("m", [1, 9, 130])
def test_not_a_number_stays_in_its_row(cuda_device, m):
    x, wg, wu = block_inputs(m, 128, 140, torch.bfloat16)
    clean = ffn.run(x, wg, wu, "silu")
    x[m // 2, 5] = float("nan")
    h, gq, gs, uq, us = ffn.run(x, wg, wu, "silu", checkpoint=True)
    other = torch.arange(m, device="cuda") != m // 2
    for got in (h, ffn.run(x, wg, wu, "silu")):
        assert bool(got[m // 2].isnan().all()) and torch.equal(got[other], clean[other]) is True
    assert bool(gq[m // 2].float().isnan().all()) and bool((gs[m // 2] == 1).all())


@pytest.mark.parametrize("f", [128, 136, 131])
@pytest.mark.parametrize("m", [1, 12, 129])
def test_forward_writes_its_rows_only(cuda_device, m, f):
    ext = native.load()
    x, wg, wu = block_inputs(m, 64, f, torch.float16)
    h = torch.full((m + 2, f), 7.0, dtype=torch.float16, device="cuda")
    q = torch.full((2, m + 2, f), 0x33, dtype=torch.uint8, device="cuda")
    s = torch.full((2, m + 2, -(-f // 128)), -3.0, device="cuda")
    qs = [q[i, 1:-1].view(torch.float8_e4m3fn) for i in range(2)]
    ext.ffn_gated(x, wg, wu, h[1:-1], 0, qs[0], s[0, 1:-1], qs[1], s[1, 1:-1])
    want = ffn.run(x, wg, wu, "silu", checkpoint=True)
    got = (h[1:-1], qs[0], s[0, 1:-1], qs[1], s[1, 1:-1])
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))
    ext.ffn_gated(x, wg, wu, h[1:-1], 0, None, None, None, None)
    assert torch.equal(h[1:-1], ffn.run(x, wg, wu, "silu"))
    for t, v in ((h, 7), (q[0], 0x33), (q[1], 0x33), (s[0], -3), (s[1], -3)):
        assert bool((t[0] == v).all()) and bool((t[-1] == v).all())


# ---- backward ----------------------------------------------------------------------------------------

def backward_inputs(m, k, f, dtype, x_codes=True):
    x, wg, wu = block_inputs(m, k, f, dtype)
    g = gen(m + 3 * k + 5 * f)
    dh = normal(g, m, f, scale=0.1, dtype=dtype)
    held = [t for _ in range(2) for t in tensors.checkpoint_fp8(normal(g, m, f, scale=2.0))]
    return dh, wg, wu, *(tensors.checkpoint_fp8(x) if x_codes else (x, None)), *held


def backward64(dh, wg, wu, x, xs, gq, gs, uq, us, act):
    def held(q, s):
        return q.double() * s.double().repeat_interleave(128, dim=1)[:, :q.shape[1]]
    x = x.double() if xs is None else held(x, xs)
    g, u = held(gq, gs), held(uq, us)
    a, da = tensors.gate(g, act)
    dg, du = dh.double() * u * da, dh.double() * a
    sums = (dg @ wg.double() + du @ wu.double(), dg.t() @ x, du.t() @ x)
    size = (dg.abs() @ wg.double().abs() + du.abs() @ wu.double().abs(), dg.abs().t() @ x.abs(), du.abs().t() @ x.abs())
    # f' may cancel to zero where f is steep: its own error is 2^-19 of 1, not of f'
    loose = (GATE * ((dh.double() * u).abs() @ wg.double().abs()), GATE * ((dh.double() * u).abs().t() @ x.abs()), 0)
    under = (wg.double().abs().sum(0) + wu.double().abs().sum(0), x.abs().sum(0), x.abs().sum(0))
    return sums, size, loose, under


def check_gradients(got, args, act, dtype):
    """Each output: dg and du were rounded once (E of every term), summed in 32 bits, and the result rounded once."""
    m, f = args[0].shape
    sums, size, loose, under = backward64(*args, act)
    for t, want, mag, more, tiny, n in zip(got, sums, size, loose, under, (2 * f, m, m)):
        tol = (half_step(dtype) + GATE + depth_error(n)) * mag + more + TINY[dtype] * tiny
        tol = tol + half_step(dtype) * (want.abs() + tol) + TINY[dtype]
        err = (t.double() - want).abs()
        assert t.dtype == dtype and bool((err <= tol).all())
        # roundings are spread over half a step either way: 2-norm E / sqrt(3) of dg's terms and as much of the output
        if want.numel() >= 4096:
            assert float(err.norm()) <= 2 * half_step(dtype) * float(want.norm())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,f", SIZES)
def test_backward(cuda_device, m, k, f, dtype):
    act = ACTS[(m + k) % 4]
    args = backward_inputs(m, k, f, dtype, x_codes=(m % 2 == 0))
    check_gradients(bwd.run(*args, act), args, act, dtype)


@pytest.mark.parametrize("act", ACTS)
def test_backward_gates(cuda_device, act):
    for x_codes in (True, False):
        args = backward_inputs(257, 520, 650, torch.float16, x_codes)
        check_gradients(bwd.run(*args, act), args, act, torch.float16)


@pytest.mark.parametrize("act", ACTS)
def test_backward_of_very_large_projections(cuda_device, act):
    """|g| up to 2^104: f'(g) is 0 or 1 there, and the squares and cubes that the formulas name leave fp32's range."""
    args = list(backward_inputs(40, 64, 40, torch.bfloat16))
    args[6] = torch.exp2(torch.arange(40, device="cuda") * 2.0 + 18)[:, None].contiguous()       # times codes of up to 448
    check_gradients(bwd.run(*args, act), args, act, torch.bfloat16)


@pytest.mark.parametrize("m,k,f", [(512, 9472, 2820), (1100, 2056, 1900), (2000, 1024, 3000), (300, 520, 20000), (60, 4104, 6500)])
def test_backward_over_many_tiles(cuda_device, m, k, f):
    """Enough tiles for several rounds: dx and the weights' gradients in one launch, in two, and dx by the kernel for few rows."""
    args = backward_inputs(m, k, f, torch.bfloat16, x_codes=True)
    check_gradients(bwd.run(*args, "relu"), args, "relu", torch.bfloat16)


@pytest.mark.parametrize("m,k,f", [(3000, 136, 140), (9000, 264, 24), (520, 72, 9000), (70, 2056, 5000)])
def test_backward_in_shares(cuda_device, m, k, f):
    """Sizes whose tiles are too few, for the gradient of x or for those of the weights: the contraction is shared out."""
    for x_codes in (True, False):
        args = backward_inputs(m, k, f, torch.bfloat16, x_codes)
        check_gradients(bwd.run(*args, "silu"), args, "silu", torch.bfloat16)


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_backward_takes_codes_at_odd_addresses(cuda_device, offset):
    args = list(backward_inputs(33, 72, 136, torch.float16))
    want = bwd.run(*args, "relu")

    def moved(t):
        flat = torch.zeros(t.numel() + 16, dtype=torch.uint8, device="cuda")
        flat[offset:offset + t.numel()] = t.view(torch.uint8).flatten()
        return flat[offset:offset + t.numel()].view(t.shape).view(t.dtype)
    for i in (3, 5, 7):
        args[i] = moved(args[i])
    assert all(torch.equal(a, b) for a, b in zip(bwd.run(*args, "relu"), want))


def test_backward_takes_a_strided_input(cuda_device):
    args = list(backward_inputs(70, 136, 200, torch.bfloat16, x_codes=False))
    wide = torch.zeros(70, 160, dtype=torch.bfloat16, device="cuda")
    wide[:, :136] = args[3]
    want = bwd.run(*args, "silu")
    args[3] = wide[:, :136]
    assert all(torch.equal(a, b) for a, b in zip(bwd.run(*args, "silu"), want))


def test_backward_is_the_gradient_of_the_forward(cuda_device):
    """Small whole numbers: the projections fit in 8 bits exactly, so the operators' own chain, forward with
    checkpoints and backward, is the derivative that 64-bit autograd gives, up to the roundings of dg, du and the outputs."""
    g = gen(17)
    x = torch.randint(-1, 2, (150, 16), generator=g, device="cuda").to(torch.bfloat16)
    wg, wu = (torch.randint(-1, 2, (137, 16), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    dh = normal(g, 150, 137, dtype=torch.bfloat16)
    for act in ACTS:
        t = [v.double().requires_grad_() for v in (x, wg, wu)]
        a = t[0] @ t[1].t()
        ((torch.relu(a) if act == "relu" else tensors.gate(a, act)[0]) * (t[0] @ t[2].t())).backward(dh.double())  # relu'(0) = 0
        h, gq, gs, uq, us = ffn.run(x, wg, wu, act, checkpoint=True)
        args = (dh, wg, wu, *save.run(x), gq, gs, uq, us)
        got = bwd.run(*args, act)
        check_gradients(got, args, act, torch.bfloat16)
        sums = backward64(*args, act)[0]
        for a, b in zip(sums, t):
            assert torch.allclose(a, b.grad, rtol=1e-12, atol=1e-12)


def test_no_tokens(cuda_device):
    x = torch.empty(0, 64, dtype=torch.float16, device="cuda")
    wg, wu = (normal(gen(1), 48, 64, dtype=torch.float16) for _ in range(2))
    assert ffn.run(x, wg, wu).shape == (0, 48)
    h, gq, gs, uq, us = ffn.run(x, wg, wu, checkpoint=True)
    assert gq.shape == (0, 48) and us.shape == (0, 1)
    xq, xs = save.run(x)
    assert restore.run(xq, xs).shape == (0, 64)
    for xin in ((xq, xs), (x, None)):
        dx, dwg, dwu = bwd.run(torch.empty(0, 48, dtype=torch.float16, device="cuda"), wg, wu, *xin, gq, gs, uq, us)
        assert dx.shape == (0, 64) and not dwg.any() and not dwu.any()


# ---- together, captured, on other streams -------------------------------------------------------------

def train_step(x, wg, wu, dh, act):
    xq, xs = save.run(x)
    h, gq, gs, uq, us = ffn.run(x, wg, wu, act, checkpoint=True)
    return (h, *bwd.run(dh, wg, wu, xq, xs, gq, gs, uq, us, act))


@pytest.mark.parametrize("m,k,f", [(1, 64, 130), (77, 200, 333), (512, 1024, 1408)])
def test_training_step_by_hand(cuda_device, m, k, f):
    """Save, forward, backward and an update of the weights, several times over, each step against 64 bits."""
    x, wg, wu = block_inputs(m, k, f, torch.bfloat16)
    for step in range(3):
        dh = normal(gen(step), m, f, scale=0.1, dtype=torch.bfloat16)
        xq, xs = save.run(x)
        h, gq, gs, uq, us = ffn.run(x, wg, wu, "silu", checkpoint=True)
        check_h(h, x, wg, wu, "silu")
        args = (dh, wg, wu, xq, xs, gq, gs, uq, us)
        dx, dwg, dwu = bwd.run(*args, "silu")
        check_gradients((dx, dwg, dwu), args, "silu", torch.bfloat16)
        wg, wu = (w - 0.1 * d for w, d in ((wg, dwg), (wu, dwu)))


@pytest.mark.parametrize("m", [1, 8, 50, 300])
def test_captured_steps_replay_on_new_inputs(cuda_device, m):
    """Two graphs that live at once, replayed in turn on inputs that change, bit for bit as the eager calls."""
    state, graphs = [], []
    for i, act in enumerate(("silu", "gelu")):
        x, wg, wu = block_inputs(m, 136, 200, torch.float16, seed=i)
        dh = normal(gen(i), m, 200, dtype=torch.float16)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            train_step(x, wg, wu, dh, act), ffn.run(x, wg, wu, act)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = (*train_step(x, wg, wu, dh, act), ffn.run(x, wg, wu, act))
        state.append((x, wg, wu, dh, act, out))
        graphs.append(graph)
    for turn in range(3):
        for i in range(2):
            x, wg, wu, dh, act, out = state[i]
            x.copy_(normal(gen(100 * turn + i), m, 136))
            dh.copy_(normal(gen(200 * turn + i), m, 200))
            graphs[i].replay()
        for x, wg, wu, dh, act, out in state:
            want = (*train_step(x, wg, wu, dh, act), ffn.run(x, wg, wu, act))
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("m", [1, 40, 300])
def test_captured_behind_copies_fills_and_another_stream(cuda_device, m):
    """What a call waits for may be a copy, a fill or another stream's work instead of a kernel."""
    x, wg, wu = block_inputs(m, 136, 200, torch.bfloat16)
    dh = normal(gen(m), m, 200, dtype=torch.bfloat16)
    source, weight = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in (x, wg)]
    into, w, zeros = torch.empty_like(source), torch.empty_like(weight), torch.ones_like(source)
    side = torch.cuda.Stream()

    def step():
        into.copy_(source)
        plain = ffn.run(into, wg, wu)
        zeros.zero_()
        none = ffn.run(zeros, wg, wu)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            w.copy_(weight)
            w.mul_(2.0)
        out = train_step(into, wg, wu, dh, "silu")
        torch.cuda.current_stream().wait_stream(side)
        return (plain, none, *out, ffn.run(into, w, wu), *train_step(into, w, wu, dh, "gelu"))

    def expected():
        a, b = source.clone(), weight * 2.0
        torch.cuda.synchronize()
        return (ffn.run(a, wg, wu), torch.zeros(m, 200, dtype=torch.bfloat16, device="cuda"), *train_step(a, wg, wu, dh, "silu"), ffn.run(a, b, wu),
                *train_step(a, b, wu, dh, "gelu"))
    source.copy_(x), weight.copy_(wg)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        source.copy_(normal(gen(turn), m, 136))
        weight.copy_(normal(gen(50 + turn), 200, 136, scale=0.1))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expected()))
        assert all(torch.equal(a, b) for a, b in zip(step(), expected()))
        torch.cuda.synchronize()


def test_first_call_of_a_process_inside_a_capture(cuda_device):
    """Nothing that a first call sets up is refused under capture."""
    code = """
import torch
from tilebench_b200 import native
from tilebench_b200.benchmarks.layers.ffn_gated import impl_cuda as ffn
from tilebench_b200.benchmarks.layers.ffn_gated_bwd import impl_cuda as bwd
native.load()
x, wg, wu, dh = (torch.randn(s, device="cuda").half() for s in ((200, 64), (136, 64), (136, 64), (200, 136)))
def step():
    h, *held = ffn.run(x, wg, wu, "gelu_tanh", checkpoint=True)
    return (h, *bwd.run(dh, wg, wu, x, None, *held, "gelu_tanh"), ffn.run(x[:3], wg, wu, "gelu_tanh"))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, step()))
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=REPO_ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_calls_on_two_streams_at_once(cuda_device):
    sets = [(*block_inputs(64 + 200 * i, 512, 640, torch.bfloat16, seed=i), normal(gen(i), 64 + 200 * i, 640, dtype=torch.bfloat16)) for i in range(2)]
    want = [train_step(x, wg, wu, dh, "silu") for x, wg, wu, dh in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(6):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(train_step(*sets[i], "silu"))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_repeated_calls_are_bit_identical(cuda_device):
    for m, k, f in ((1, 4096, 2816), (16, 4096, 2816), (100, 2048, 2816), (700, 1024, 2816)):
        x, wg, wu = block_inputs(m, k, f, torch.bfloat16)
        dh = normal(gen(m), m, f, dtype=torch.bfloat16)
        first, plain = train_step(x, wg, wu, dh, "silu"), ffn.run(x, wg, wu)
        for _ in range(20):
            assert all(torch.equal(a, b) for a, b in zip(train_step(x, wg, wu, dh, "silu"), first))
            assert torch.equal(ffn.run(x, wg, wu), plain)


# ---- refusals and the engine ---------------------------------------------------------------------------

def test_refusals(cuda_device):
    x, wg, wu = block_inputs(4, 64, 48, torch.float16)
    for bad in (lambda: ffn.run(x.t().contiguous().t(), wg, wu), lambda: ffn.run(x, wg.t().contiguous().t(), wu),
                lambda: ffn.run(x.bfloat16(), wg, wu), lambda: ffn.run(x, wg, wu.bfloat16()), lambda: ffn.run(x, wg, wu[:-1]),
                lambda: ffn.run(x[:, :56], wg, wu), lambda: ffn.run(x, wg.cpu(), wu), lambda: save.run(x.t()),
                lambda: restore.run(x.to(torch.float8_e4m3fn), torch.ones(4, 2, device="cuda")),
                lambda: restore.run(x, torch.ones(4, 1, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(TypeError):
        ffn.run(x.float(), wg.float(), wu.float())
    with pytest.raises(TypeError):
        save.run(x.double())
    with pytest.raises(TypeError):
        restore.run(x.to(torch.float8_e4m3fn), torch.ones(4, 1, device="cuda"), torch.int32)
    with pytest.raises(TypeError, match="multiple of 8"):
        ffn.run(x[:, :60].contiguous(), wg[:, :60].contiguous(), wu[:, :60].contiguous())
    with pytest.raises(ValueError, match="row stride"):
        ffn.run(normal(gen(1), 4, 68, dtype=torch.float16)[:, :64], wg, wu)
    h, gq, gs, uq, us = ffn.run(x, wg, wu, checkpoint=True)
    dh = torch.ones_like(h)
    xq, xs = save.run(x)
    for bad in (lambda: bwd.run(dh[:, :40], wg, wu, xq, xs, gq, gs, uq, us), lambda: bwd.run(dh, wg, wu, x, xs, gq, gs, uq, us),
                lambda: bwd.run(dh, wg, wu, xq, None, gq, gs, uq, us), lambda: bwd.run(dh, wg, wu, xq, xs, gq[:3], gs, uq, us),
                lambda: bwd.run(dh, wg, wu, xq, xs, gq, gs[:, :0], uq, us), lambda: bwd.run(dh.bfloat16(), wg, wu, xq, xs, gq, gs, uq, us)):
        with pytest.raises(RuntimeError):
            bad()
    ext = native.load()
    small = torch.empty(16, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="workspace"):
        ext.ffn_gated_bwd(dh, wg, wu, xq, xs, gq, gs, uq, us, torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu), 0, small)


@pytest.mark.parametrize("op,cases", [("act_checkpoint_fp8", [0, 4, 8]), ("act_restore_fp8", [0, 4, 8]), ("ffn_gated", [0, 5, 8, 12]),
                                      ("ffn_gated_bwd", [0, 3])])
def test_through_the_engine(cuda_device, op, cases):
    rows = run_benchmark_suite(op, {"warmup": 1, "repeat": 1, "case_indices": cases}, ["cuda"])
    assert len(rows) == len(cases)
    for r in rows:
        assert r["cuda_ok"], f"{r['params']}: {r['cuda_err']}"
        assert r["cuda_ms"] > 0 and r["cuda_stats"]["mode"] == "graph"
