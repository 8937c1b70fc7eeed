"""cuda backend of ffn_gated: both projections, the gate and the product in one kernel (tb200_ffn_gated)."""
import warnings

import torch

from tilebench_b200 import native


def run(x: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, act: str = "silu", checkpoint: bool = False, **kwargs):
    """h [m, f] = f(x Wg^T) * (x Wu^T) for x [m, k] (any row stride that is a multiple of 8) and wg, wu [f, k], fp16
    or bf16; act: silu, gelu, gelu_tanh or relu.  With `checkpoint`: (h, gq, gs, uq, us), where gq, gs and uq, us
    are the 8-bit forms (act_checkpoint_fp8's) of the two projections, which ffn_gated_bwd reads.  Autograd records neither
    form: gradients come from ffn_gated_bwd alone, and a call without checkpoints on tensors that require one warns."""
    ext = native.load()
    if not checkpoint and torch.is_grad_enabled() and (x.requires_grad or wg.requires_grad or wu.requires_grad):
        warnings.warn("ffn_gated: autograd does not record this call, no gradient will reach x, wg or wu through it; use checkpoint=True "
                      "with ffn_gated_bwd to train, torch.no_grad() where no gradient is wanted", stacklevel=2)
    run = ext.ffn_gated_checkpoint_new if checkpoint else ext.ffn_gated_new
    return run(x, wg, wu, native.activation(act))
