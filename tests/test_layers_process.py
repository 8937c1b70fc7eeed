"""What the operators leave behind in the process that calls them, and what they say to a caller who expects a gradient."""
import importlib
import warnings

import pytest
import torch

from tilebench_b200.data import tensors
from tilebench_b200.paths import operator_package

CASES = {"ffn_gated": dict(M=3, K=16, F=5), "ffn_gated_bwd": dict(M=3, K=16, F=5), "gemm_w4a16": dict(M=3, K=128, N=8),
         "gemm_fp8_blockscaled": dict(M=3, N=128, K=128)}


@pytest.mark.parametrize("allowed", [True, False])
@pytest.mark.parametrize("op", sorted(CASES))
def test_references_leave_the_precision_of_products_as_they_found_it(op, allowed, monkeypatch):
    monkeypatch.setattr(torch.backends.cuda.matmul, "allow_tf32", allowed)
    seen = []
    product = torch.Tensor.t
    monkeypatch.setattr(torch.Tensor, "t", lambda s: seen.append(torch.backends.cuda.matmul.allow_tf32) or product(s))   # beside each product
    impl = importlib.import_module(f"{operator_package(op)}.impl_torch")
    monkeypatch.setattr(torch.backends.cuda.matmul, "allow_tf32", allowed)            # an import may set it
    impl.run(*tensors.get_generator(op)(**CASES[op], device="cpu"))
    assert torch.backends.cuda.matmul.allow_tf32 is allowed
    assert False in seen


def test_a_lost_gradient_is_said_aloud():
    """Host tensors: the call is refused after the warning, which needs no GPU."""
    from tilebench_b200.benchmarks.layers.ffn_gated import impl_cuda as ffn
    from tilebench_b200.csrc import build
    build.build_all()
    x, wg, wu = (torch.zeros(s, dtype=torch.float16) for s in ((4, 64), (16, 64), (16, 64)))
    for which in range(3):
        args = [t.clone().requires_grad_(i == which) for i, t in enumerate((x, wg, wu))]
        with pytest.warns(UserWarning, match="autograd does not record"), pytest.raises(RuntimeError, match="CUDA"):
            ffn.run(*args)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
                ffn.run(*args)
            with pytest.raises(RuntimeError, match="CUDA"):  # gradients by hand
                ffn.run(*args, checkpoint=True)
            with pytest.raises(RuntimeError, match="CUDA"):
                ffn.run(x, wg, wu)
