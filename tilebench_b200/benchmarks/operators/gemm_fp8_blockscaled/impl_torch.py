import torch

from tilebench_b200.core.dtypes import full_fp32_matmul


def run(aq: torch.Tensor, sa: torch.Tensor, bq: torch.Tensor, sb: torch.Tensor, BLOCK: int = 128, **kwargs):
    a = aq.to(torch.float32) * sa.repeat_interleave(BLOCK, dim=1)
    b = bq.to(torch.float32) * sb.repeat_interleave(BLOCK, dim=0).repeat_interleave(BLOCK, dim=1)
    with full_fp32_matmul():
        return torch.matmul(a, b.t()).to(torch.bfloat16)
