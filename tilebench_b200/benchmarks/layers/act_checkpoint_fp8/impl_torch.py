import torch

from tilebench_b200.data.tensors import checkpoint_fp8


def run(x: torch.Tensor, **kwargs):
    """(codes e4m3 [rows, cols], scales fp32 [rows, ceil(cols / 128)])"""
    return checkpoint_fp8(x)
