import torch

from tilebench_b200.core.dtypes import full_fp32_matmul
from tilebench_b200.data.tensors import checkpoint_fp8, gate


def run(x: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, act: str = "silu", checkpoint: bool = False, **kwargs):
    """h = f(x Wg^T) * (x Wu^T) in fp32, rounded once; with `checkpoint` also the 8-bit forms of both projections."""
    x32 = x.to(torch.float32)
    with full_fp32_matmul():
        g, u = x32 @ wg.to(torch.float32).t(), x32 @ wu.to(torch.float32).t()
    h = (gate(g, act)[0] * u).to(x.dtype)
    return (h, *checkpoint_fp8(g), *checkpoint_fp8(u)) if checkpoint else h
