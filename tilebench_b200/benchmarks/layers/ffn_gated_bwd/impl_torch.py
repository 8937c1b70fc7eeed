import torch

from tilebench_b200.core.dtypes import full_fp32_matmul
from tilebench_b200.data.tensors import gate, restore_fp8


def run(dh, wg, wu, x, xs, gq, gs, uq, us, act: str = "silu", **kwargs):
    """(dx, dWg, dWu) in fp32 from the restored activations, rounded once."""
    f32 = torch.float32
    x = x.to(f32) if xs is None else restore_fp8(x, xs, f32)
    g, u = restore_fp8(gq, gs, f32), restore_fp8(uq, us, f32)
    a, da = gate(g, act)
    dh = dh.to(f32)
    dg, du = dh * u * da, dh * a
    with full_fp32_matmul():
        grads = (dg @ wg.to(f32) + du @ wu.to(f32), dg.t() @ x, du.t() @ x)
    return tuple(t.to(wg.dtype) for t in grads)
