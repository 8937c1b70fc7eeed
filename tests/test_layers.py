"""The layer operators on CPU: their formulas in the package against 64-bit statements, their place in the harness, and
the refusals of the C ABI (arguments are checked on the host before anything is launched)."""
import ctypes
import math

import pytest
import torch
import yaml

from tilebench_b200 import native
from tilebench_b200.data import tensors
from tilebench_b200.paths import list_layer_operators, list_operators, operator_config, operator_package

LAYERS = ["act_checkpoint_fp8", "act_restore_fp8", "ffn_gated", "ffn_gated_bwd"]
ACTS = ("silu", "gelu", "gelu_tanh", "relu")
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def scale64(amax: float) -> float:
    """The smallest power of two >= 2^-126 with amax <= 448 * scale, 1 for amax 0 (64-bit search)."""
    if amax == 0:
        return 1.0
    e = -126
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def nearest_code64(y: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 number to y (|y| <= 448), ties to even, from the list of all numbers."""
    grid = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    a = y.abs()
    hi = torch.searchsorted(grid, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - grid[lo], grid[hi] - a
    even = torch.where(lo % 2 == 0, lo, hi)
    pick = torch.where(dl < dh, lo, torch.where(dh < dl, hi, even))
    pick = torch.where(a == grid[hi], hi, pick)
    return torch.copysign(grid[pick], y)


def test_layer_operators_are_listed_and_their_grids_expand():
    assert list_layer_operators() == LAYERS
    assert not set(LAYERS) & set(list_operators())
    for op, n in zip(LAYERS, (9, 9, 16, 8)):
        assert operator_package(op) == f"tilebench_b200.benchmarks.layers.{op}"
        cfg = yaml.safe_load(open(operator_config(op)))
        cases = tensors.expand_cases(op, cfg)
        assert len(cases) == n and cfg["benchmark"]["use_cuda_graph"] is True
        assert tensors.infer_problem_size(op, cases[0]) > 1
        assert op in tensors.GENERATORS
    assert operator_package("gemm_w4a16") == "tilebench_b200.benchmarks.operators.gemm_w4a16"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 127), (2, 128), (5, 129), (4, 300)])
def test_checkpoint_formula(rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * 1000 + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))).to(dtype)
    x[0, 0] = 0
    q, s = tensors.checkpoint_fp8(x)
    assert q.shape == x.shape and s.shape == (rows, -(-cols // 128))
    for r in range(rows):
        for b in range(s.shape[1]):
            part = x[r, 128 * b:128 * (b + 1)].double()
            want = scale64(float(part.abs().max()))
            assert float(s[r, b]) == want
            assert torch.equal(q[r, 128 * b:128 * (b + 1)].double(), nearest_code64(part / want))
    # a code is off by half a step at most: 2^-4 of the value, or half of the smallest step
    back = tensors.restore_fp8(q, s, torch.float32).double()
    step = s.double().repeat_interleave(128, dim=1)[:, :cols] * 2.0 ** -10
    assert bool(((back - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, step)).all())


def test_checkpoint_special_values():
    inf, nan = math.inf, math.nan
    x = torch.zeros(8, 128)
    x[1, :4] = torch.tensor([448.0, -448.0, 1.0, 2.0 ** -9])
    x[2, :3] = torch.tensor([inf, -inf, nan])
    x[3, :4] = torch.tensor([inf, 3.0, nan, -5.0])
    x[4, 0] = 2.0 ** -149                                   # the smallest subnormal number
    x[5, 0] = torch.finfo(torch.float32).max
    x[6, 0] = 448.0000305                                   # just above a border of the scale
    x[7, :2] = torch.tensor([-0.0, 0.0])
    q, s = tensors.checkpoint_fp8(x)
    assert s[:, 0].tolist() == [1.0, 1.0, 1.0, 2.0 ** -6, 2.0 ** -126, 2.0 ** 120, 2.0, 1.0]
    assert q[1, :4].float().tolist() == [448.0, -448.0, 1.0, 2.0 ** -9]
    assert q[2, :3].float().isnan().all() and not q[2, 3:].float().any()
    assert q[3].float().isnan().nonzero().flatten().tolist() == [0, 2]
    assert q[3, [1, 3]].float().tolist() == [192.0, -320.0]
    for dtype in DTYPES:                                    # an amax that was rounded up stays finite
        top = torch.finfo(dtype).max
        t = torch.tensor([[top, -top, 1.0]], dtype=dtype)
        back = tensors.restore_fp8(*tensors.checkpoint_fp8(t), dtype)
        assert back[0, 0] == top and back[0, 1] == -top


@pytest.mark.parametrize("act", ACTS)
def test_gate_values_and_derivatives(act):
    z = torch.linspace(-12, 12, 4801, dtype=torch.float64) + 1e-4
    f, df = tensors.gate(z, act)
    ref = {"silu": lambda v: v / (1 + torch.exp(-v)), "gelu": lambda v: torch.nn.functional.gelu(v),
           "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh"), "relu": lambda v: torch.relu(v)}[act]
    assert torch.allclose(f, ref(z), atol=1e-14, rtol=1e-9)
    step = 1e-5                                             # differences: error step^2 f''' / 6 + 2^-53 |f| / step < 1e-9
    diff = (tensors.gate(z + step, act)[0] - tensors.gate(z - step, act)[0]) / (2 * step)
    assert torch.allclose(df, diff, atol=2e-9, rtol=0)
    with pytest.raises(ValueError):
        tensors.gate(z, "swish")
    with pytest.raises(ValueError):
        native.activation("swish")


@pytest.mark.parametrize("act", ACTS)
def test_plain_backward_is_the_gradient(act):
    """impl_torch of the backward pass against autograd in 64 bits, where the 8-bit forms hold g, u and x exactly."""
    from tilebench_b200.benchmarks.layers.ffn_gated import impl_torch as fwd
    from tilebench_b200.benchmarks.layers.ffn_gated_bwd import impl_torch as bwd
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-1, 2, (9, 16), generator=g).double().requires_grad_()
    wg, wu = (torch.randint(-1, 2, (13, 16), generator=g).double().requires_grad_() for _ in range(2))
    dh = torch.randn(9, 13, generator=g).to(torch.bfloat16)
    a = x @ wg.t()
    f = (torch.relu(a) if act == "relu" else tensors.gate(a, act)[0]) * (x @ wu.t())       # relu'(0) = 0
    f.backward(dh.double())
    low = [t.detach().to(torch.bfloat16) for t in (x, wg, wu)]
    h, gq, gs, uq, us = fwd.run(*low, act, checkpoint=True)
    assert torch.equal(tensors.restore_fp8(gq, gs, torch.float32).double(), a.detach())
    # bf16 outputs: half a step, 2^-8 of the value; the 32-bit sums are off by less than 2^-18
    assert torch.allclose(h.double(), f.detach(), rtol=2.0 ** -8, atol=2.0 ** -18)
    for xq, xs in (tensors.checkpoint_fp8(low[0]), (low[0], None)):
        for got, want in zip(bwd.run(dh, low[1], low[2], xq, xs, gq, gs, uq, us, act), (x.grad, wg.grad, wu.grad)):
            assert torch.allclose(got.double(), want, rtol=2.0 ** -8, atol=2.0 ** -18)


# ---- refusals: checked on the host, nothing is launched ------------------------------------------

ARG, ALIGN, UNSUPPORTED, WORKSPACE = 1, 2, 3, 5
P = ctypes.c_void_p(1 << 20)                                # never dereferenced: every call below is refused


@pytest.fixture(scope="module")
def lib():
    from tilebench_b200.csrc import build
    build.build_all()
    return native.capi()


def test_refusals_of_save_and_restore(lib):
    fp = ctypes.c_void_p(1 << 20)
    assert lib.tb200_act_checkpoint_fp8(P, P, fp, -1, 8, 8, 0, None) == ARG
    assert lib.tb200_act_checkpoint_fp8(P, P, fp, 4, 0, 8, 0, None) == ARG
    assert lib.tb200_act_checkpoint_fp8(None, P, fp, 4, 8, 8, 0, None) == ARG
    assert lib.tb200_act_checkpoint_fp8(P, P, fp, 4, 8, 7, 0, None) == ARG          # rows overlap
    assert lib.tb200_act_checkpoint_fp8(P, P, fp, 4, 8, 8, native.DT_F8E4M3, None) == UNSUPPORTED
    assert lib.tb200_act_checkpoint_fp8(P, P, fp, 1 << 31, 256, 256, 0, None) == UNSUPPORTED
    assert lib.tb200_act_checkpoint_fp8(ctypes.c_void_p(2), P, fp, 4, 8, 8, 0, None) == ALIGN
    assert lib.tb200_act_restore_fp8(P, fp, None, 4, 8, 0, None) == ARG
    assert lib.tb200_act_restore_fp8(P, fp, P, 4, 8, 7, None) == UNSUPPORTED
    assert lib.tb200_act_restore_fp8(P, fp, ctypes.c_void_p(1), 4, 8, 1, None) == ALIGN
    assert lib.tb200_act_restore_fp8(P, ctypes.c_void_p(2), P, 4, 8, 1, None) == ALIGN
    assert "aligned" in native.last_error()


def test_refusals_of_the_forward_block(lib):
    def call(x=P, wg=P, wu=P, h=P, ckpt=(None,) * 4, m=4, f=16, k=64, ldx=64, act=0, dtype=native.DT_BF16):
        return lib.tb200_ffn_gated(x, wg, wu, h, *ckpt, m, f, k, ldx, act, dtype, None)
    assert call(m=-1) == ARG and call(f=0) == ARG and call(k=0) == ARG
    assert call(x=None) == ARG and call(wg=None) == ARG and call(wu=None) == ARG and call(h=None) == ARG
    assert call(ckpt=(P, P, P, None)) == ARG and "together" in native.last_error()
    assert call(k=60) == UNSUPPORTED and "multiple of 8" in native.last_error()
    assert call(dtype=native.DT_F32) == UNSUPPORTED and call(act=4) == UNSUPPORTED and call(act=-1) == UNSUPPORTED
    assert call(ldx=56) == ALIGN and call(ldx=68) == ALIGN
    assert call(x=ctypes.c_void_p(8)) == ALIGN and call(wu=ctypes.c_void_p(24)) == ALIGN
    assert call(m=1 << 31) == UNSUPPORTED
    odd = ctypes.c_void_p((1 << 20) + 1)
    assert call(h=odd) == ALIGN and call(ckpt=(P, odd, P, P)) == ALIGN and call(ckpt=(P, P, P, odd)) == ALIGN


def test_refusals_of_the_backward_block(lib):
    need = lib.tb200_ffn_gated_bwd_workspace_bytes(4, 17, 64, 1)
    assert need == 2 * 512 + 512                            # dg, du: 4 rows of 128 bytes; x: the same
    assert lib.tb200_ffn_gated_bwd_workspace_bytes(4, 17, 64, 0) == 2 * 512
    assert lib.tb200_ffn_gated_bwd_workspace_bytes(0, 17, 64, 1) == 0

    def call(dh=P, wg=P, wu=P, x=P, xs=P, gq=P, gs=P, uq=P, us=P, dx=P, dwg=P, dwu=P, m=4, f=17, k=64, ldx=64, act=0,
             dtype=native.DT_F16, ws=P, nbytes=need):
        return lib.tb200_ffn_gated_bwd(dh, wg, wu, x, xs, gq, gs, uq, us, dx, dwg, dwu, m, f, k, ldx, act, dtype, ws, nbytes, None)
    for name in ("dh", "wg", "wu", "x", "gq", "gs", "uq", "us", "dx", "dwg", "dwu"):
        assert call(**{name: None}) == ARG, name
    assert call(m=-1) == ARG and call(k=12) == UNSUPPORTED and call(dtype=native.DT_F32) == UNSUPPORTED and call(act=9) == UNSUPPORTED
    assert call(xs=None, ldx=60) == ALIGN and call(xs=None, x=ctypes.c_void_p(8)) == ALIGN and call(dx=ctypes.c_void_p(8)) == ALIGN
    assert call(ws=None) == WORKSPACE and call(nbytes=need - 1) == WORKSPACE and call(ws=ctypes.c_void_p(128)) == WORKSPACE
    assert str(need) in native.last_error()
    odd = ctypes.c_void_p((1 << 20) + 2)
    assert all(call(**{name: odd}) == ALIGN for name in ("gs", "us", "xs")) and call(dh=ctypes.c_void_p(1)) == ALIGN


def test_operators_refuse_host_tensors(lib):
    from tilebench_b200.benchmarks.layers.act_checkpoint_fp8 import impl_cuda as save
    from tilebench_b200.benchmarks.layers.act_restore_fp8 import impl_cuda as restore
    from tilebench_b200.benchmarks.layers.ffn_gated import impl_cuda as ffn
    from tilebench_b200.benchmarks.layers.ffn_gated_bwd import impl_cuda as bwd
    x, w = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(16, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        save.run(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        restore.run(x.to(torch.float8_e4m3fn), torch.ones(4, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        ffn.run(x, w, w)
    with pytest.raises(ValueError, match="activation"):
        ffn.run(x, w, w, "swish")
    held = (torch.zeros(4, 16, dtype=torch.float8_e4m3fn), torch.ones(4, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        bwd.run(x[:, :16], w, w, x, None, *held, *held)
