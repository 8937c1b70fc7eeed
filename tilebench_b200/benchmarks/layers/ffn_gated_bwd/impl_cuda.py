"""cuda backend of ffn_gated_bwd (tb200_ffn_gated_bwd): one streaming kernel makes the gradients of both projections
from the 8-bit checkpoints, one tcgen05 kernel the gradients of x and of both weights (few rows and large weights: two)."""
import torch

from tilebench_b200 import native


def run(dh: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, x: torch.Tensor, xs: torch.Tensor | None, gq: torch.Tensor,
        gs: torch.Tensor, uq: torch.Tensor, us: torch.Tensor, act: str = "silu", **kwargs):
    """(dx [m, k], dWg [f, k], dWu [f, k]) of ffn_gated from dh [m, f] and the checkpoints it returned.  x is the
    block's input: its codes with scales xs (act_checkpoint_fp8), or as it was with xs None."""
    return native.load().ffn_gated_bwd_new(dh, wg, wu, x, xs, gq, gs, uq, us, native.activation(act))
