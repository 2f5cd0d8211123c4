"""Edges of the decoder's operators on the GPU: types without kernels, modes of autograd, hooks on saved tensors."""

import pytest
import torch

from optimizers_b200.models import fp8, fused_ops

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _x(rows, cols, dtype=BF16, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=gen) * torch.exp(torch.randn(rows, 1, device="cuda", generator=gen))
    return (x * torch.exp(torch.randn(1, cols, device="cuda", generator=gen))).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_tokens_outside_the_table_in_types_without_kernels(dtype):
    table = torch.randn(11, 6, device="cuda").to(dtype).requires_grad_()
    ids = torch.tensor([[3, -1, 10], [11, 3, 2**40]], device="cuda")
    y = fused_ops.embedding(ids, table, scale=2.0)
    known = (ids >= 0) & (ids < 11)
    assert torch.equal(y[known], table.detach()[ids[known]] * 2) and y[~known].isnan().all()
    (grad,) = torch.autograd.grad(y, table, torch.ones_like(y))
    want = torch.zeros(11, 6, device="cuda").to(dtype)
    want[3], want[10] = 4, 2
    assert torch.equal(grad, want)
    assert fused_ops.embedding(ids, table[:0]).isnan().all()
