"""cuda backend of ffn_gated: both projections, the gate and the product in one kernel (tb200_ffn_gated)."""
import torch

from tilebench_b200 import native


def run(x: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, act: str = "silu", checkpoint: bool = False, **kwargs):
    """h [m, f] = f(x Wg^T) * (x Wu^T) for x [m, k] (any row stride that is a multiple of 8) and wg, wu [f, k], fp16
    or bf16; act: silu, gelu, gelu_tanh or relu.  With `checkpoint`: (h, gq, gs, uq, us), where gq, gs and uq, us
    are the 8-bit forms (act_checkpoint_fp8's) of the two projections, which ffn_gated_bwd reads."""
    ext = native.load()
    code = native.activation(act)
    m, f = x.shape[0], wg.shape[0]
    h = torch.empty((m, f), dtype=x.dtype, device=x.device)
    if not checkpoint:
        ext.ffn_gated(x, wg, wu, h, code, None, None, None, None)
        return h
    gq, uq = (torch.empty((m, f), dtype=torch.float8_e4m3fn, device=x.device) for _ in range(2))
    gs, us = (torch.empty((m, -(-f // 128)), dtype=torch.float32, device=x.device) for _ in range(2))
    ext.ffn_gated(x, wg, wu, h, code, gq, gs, uq, us)
    return h, gq, gs, uq, us
