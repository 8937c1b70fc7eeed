"""Calls whose kernels go round their loops more than once, and other uses of the layer operators' results.

The sizes are those at which a CTA, or a pair of CTAs, of a device with 148 SMs has a second and a third tile; with another number of SMs
the results have to be the same.  Blocks of 128 hidden units differ in size by powers of two, so that a maximum that stays from the tile
before shows."""
import pytest
import torch

from tilebench_b200.benchmarks.layers.act_checkpoint_fp8 import impl_cuda as save
from tilebench_b200.benchmarks.layers.act_restore_fp8 import impl_cuda as restore
from tilebench_b200.benchmarks.layers.ffn_gated import impl_cuda as ffn
from tilebench_b200.benchmarks.layers.ffn_gated_bwd import impl_cuda as bwd
from tilebench_b200.benchmarks.operators.gemm_fp8_blockscaled import impl_cuda as blockscaled
from tilebench_b200.data import tensors
from test_gpu_layers import (backward_inputs, block_inputs, check_gradients, check_h, check_held, clean_status, depth_error,    # noqa: F401
                             forward64, gen, half_step, normal)

pytestmark = pytest.mark.gpu


def uneven(m, k, f, dtype, seed=0):
    x, wg, wu = block_inputs(m, k, f, dtype, seed=seed, pad=8)
    g = gen(seed + f)
    blocks = -(-f // 128)
    for w in (wg, wu):
        size = torch.exp2(torch.randint(-3, 4, (blocks,), generator=g, device="cuda").float()).repeat_interleave(128)[:f]
        w.mul_(size[:, None].to(dtype))
    x.mul_(torch.exp2(torch.randint(-2, 3, (m, 1), generator=g, device="cuda").float()).to(dtype))
    return x, wg, wu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,f", [(65, 72, 28677), (300, 136, 10237), (1100, 136, 4104), (513, 200, 9999)])
def test_checkpoints_of_several_tiles_per_pair(cuda_device, m, k, f, dtype):
    """160 to 237 tiles of 256 rows x 128 hidden units on 74 pairs: both accumulators in turn, and their maxima cleared between tiles."""
    x, wg, wu = uneven(m, k, f, dtype)
    x[m // 3, 1] = float("inf")                              # a row whose maxima are taken twice
    clean = torch.arange(m, device="cuda") != m // 3
    h, gq, gs, uq, us = ffn.run(x, wg, wu, "silu", checkpoint=True)
    assert not gq[m // 3].float().isfinite().any() and bool((us[m // 3] == 1).all())
    x = x[clean]
    check_h(h[clean], x, wg, wu, "silu")
    _, g, u, eg, eu = forward64(x, wg, wu, "silu")
    check_held(gq[clean], gs[clean], g, eg)
    check_held(uq[clean], us[clean], u, eu)


@pytest.mark.parametrize("m", [1, 16, 33, 64])
@pytest.mark.parametrize("f", [28672, 40001])
def test_checkpoints_of_few_rows_and_several_tiles_per_cta(cuda_device, m, f):
    x, wg, wu = uneven(m, 72, f, torch.bfloat16)
    h, gq, gs, uq, us = ffn.run(x, wg, wu, "gelu", checkpoint=True)
    check_h(h, x, wg, wu, "gelu")
    _, g, u, eg, eu = forward64(x, wg, wu, "gelu")
    check_held(gq, gs, g, eg)
    check_held(uq, us, u, eu)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,f", [(1, 72, 28672), (16, 136, 40001), (64, 72, 40008), (65, 136, 28672), (128, 72, 40001), (100, 136, 40008)])
def test_decoding_over_several_tiles_per_cta(cuda_device, m, k, f, dtype):
    x, wg, wu = uneven(m, k, f, dtype)
    check_h(ffn.run(x, wg, wu, "silu"), x, wg, wu, "silu")


@pytest.mark.parametrize("m,k,f", [(490, 128, 5281), (735, 64, 2722), (865, 80, 2728), (300, 136, 10237)])
def test_blocks_of_rows_over_several_tiles_per_cta(cuda_device, m, k, f):
    x, wg, wu = uneven(m, k, f, torch.bfloat16)
    check_h(ffn.run(x, wg, wu, "gelu_tanh"), x, wg, wu, "gelu_tanh")


@pytest.mark.parametrize("m,k,f", [(1524, 72, 716), (1579, 200, 637), (1239, 72, 984), (1481, 136, 1690), (1145, 72, 2629), (1328, 200, 1095),
                                   (1415, 72, 3411), (1162, 136, 2931), (1424, 72, 2372), (1100, 72, 4100), (2100, 72, 6401)])
def test_prompts_on_tiles_of_every_width(cuda_device, m, k, f):
    """Tiles of 64, 80, 96, 112 and 128 hidden units, one to four per pair."""
    x, wg, wu = uneven(m, k, f, torch.bfloat16)
    check_h(ffn.run(x, wg, wu, "silu"), x, wg, wu, "silu")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 16, 64])
@pytest.mark.parametrize("k,f", [(4096, 4000), (4096, 6100), (4096, 6300), (1032, 30500)])
def test_backward_of_few_rows_and_weights_of_either_size(cuda_device, m, k, f, dtype):
    """Weights of 63 to 126 MB: dx by the launch that makes the weights' gradients, and by a kernel of its own."""
    args = backward_inputs(m, k, f, dtype, x_codes=m != 16)
    check_gradients(bwd.run(*args, "silu"), args, "silu", dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k", [(1, 128), (40, 512), (300, 1024)])
def test_codes_are_an_operand_of_the_block_scaled_product(cuda_device, m, k, dtype):
    """x saved, then multiplied as it is held: against the product of the restored numbers in 64 bits."""
    g = gen(m + k)
    x = normal(g, m, k, dtype=dtype) * torch.exp2(torch.randint(-4, 5, (m, 1), generator=g, device="cuda").float()).to(dtype)
    xq, xs = save.run(x)
    _, _, bq, sb = tensors.generate_gemm_fp8_blockscaled_inputs(M=1, N=256, K=k, device="cuda")
    a = restore.run(xq, xs, torch.float32).double()
    b = bq.double() * sb.double().repeat_interleave(128, dim=0).repeat_interleave(128, dim=1)
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    tol = (depth_error(k) + k / 128 * 2.0 ** -22) * size     # each block's sum is scaled, rounded and added in 32 bits
    tol = tol + half_step(torch.bfloat16) * (want.abs() + tol)
    assert bool(((blockscaled.run(xq, xs, bq, sb).double() - want).abs() <= tol).all())
