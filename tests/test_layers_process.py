"""What the operators leave behind in the process that calls them."""
import importlib

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
