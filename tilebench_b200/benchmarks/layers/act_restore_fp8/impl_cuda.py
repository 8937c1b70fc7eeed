"""cuda backend of act_restore_fp8: one streaming kernel (tb200_act_restore_fp8)."""
import torch

from tilebench_b200 import native


def run(q: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16, **kwargs):
    """The activation that act_checkpoint_fp8 (or ffn_gated with checkpoints) stored, as fp32, fp16 or bf16."""
    return native.load().act_restore_fp8_new(q, scales, dtype)
