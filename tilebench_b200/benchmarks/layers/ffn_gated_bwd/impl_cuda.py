"""cuda backend of ffn_gated_bwd (tb200_ffn_gated_bwd): one streaming kernel makes the gradients of both projections
from the 8-bit checkpoints, one tcgen05 kernel the gradient of x, one those of both weights."""
import torch

from tilebench_b200 import native


def run(dh: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, x: torch.Tensor, xs: torch.Tensor | None, gq: torch.Tensor,
        gs: torch.Tensor, uq: torch.Tensor, us: torch.Tensor, act: str = "silu", **kwargs):
    """(dx [m, k], dWg [f, k], dWu [f, k]) of ffn_gated from dh [m, f] and the checkpoints it returned.  x is the
    block's input: its codes with scales xs (act_checkpoint_fp8), or as it was with xs None."""
    ext = native.load()
    code = native.activation(act)
    m, (f, k) = dh.shape[0], wg.shape
    dx = torch.empty((m, k), dtype=wg.dtype, device=dh.device)
    dwg, dwu = torch.empty_like(wg), torch.empty_like(wu)
    ws = torch.empty(ext.ffn_gated_bwd_workspace_bytes(m, f, k, xs is not None), dtype=torch.uint8, device=dh.device)
    ext.ffn_gated_bwd(dh, wg, wu, x, xs, gq, gs, uq, us, dx, dwg, dwu, code, ws)
    return dx, dwg, dwu
