"""cuda backend of ffn_gated: both projections, the gate and the product in one kernel (tb200_ffn_gated)."""
import torch

from tilebench_b200 import native


def run(x: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, act: str = "silu", checkpoint: bool = False, **kwargs):
    """h [m, f] = f(x Wg^T) * (x Wu^T) for x [m, k] (any row stride that is a multiple of 8) and wg, wu [f, k], fp16
    or bf16; act: silu, gelu, gelu_tanh or relu.  With `checkpoint`: (h, gq, gs, uq, us), where gq, gs and uq, us
    are the 8-bit forms (act_checkpoint_fp8's) of the two projections, which ffn_gated_bwd reads."""
    ext = native.load()
    run = ext.ffn_gated_checkpoint_new if checkpoint else ext.ffn_gated_new
    return run(x, wg, wu, native.activation(act))
