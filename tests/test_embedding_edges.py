"""Token embedding where the kernels do not apply."""

import pytest
import torch

from optimizers_b200.models import fused_ops

F32, F64 = torch.float32, torch.float64


@pytest.mark.parametrize("dtype", [F32, F64, torch.float16])
def test_embedding_without_kernels_gives_nan_for_tokens_outside_the_table(dtype):
    """What a GPU runs for types that the kernels do not take: a lookup there must never see such a token."""
    torch.manual_seed(0)
    table = torch.randn(11, 6).to(dtype).requires_grad_()
    ids = torch.tensor([[3, -1, 10], [11, 3, 2**40]])
    y = fused_ops._embedding_of_known(ids, table)
    known = (ids >= 0) & (ids < 11)
    assert torch.equal(y[known], table[ids[known]]) and y[~known].isnan().all() and y.dtype == dtype
    dy = torch.randn(2, 3, 6).to(dtype)
    dy[~known] = float("nan")
    (grad,) = torch.autograd.grad(y, table, dy)
    want = torch.zeros(11, 6, dtype=F64).index_add_(0, ids[known], dy[known].double())
    assert torch.allclose(grad.double(), want, rtol=torch.finfo(dtype).eps, atol=2 * torch.finfo(dtype).eps)  # one sum of two values below four
    empty = torch.randn(0, 6, dtype=dtype, requires_grad=True)
    y = fused_ops._embedding_of_known(ids, empty)
    assert y.shape == (2, 3, 6) and y.isnan().all()
    assert torch.autograd.grad(y.sum(), empty)[0].shape == (0, 6)
    assert fused_ops._embedding_of_known(ids, torch.randn(4, 0, dtype=dtype)).shape == (2, 3, 0)
