"""Token embedding and the gradient of its table on the GPU against 64-bit sums."""

import pytest
import torch

from optimizers_b200.models import GPT2, GPT2Config, fused_ops

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _ids(n, V, kind, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "same":
        return torch.full((n,), V - 1, device="cuda")
    if kind == "ramp":
        return torch.arange(n, device="cuda") % V
    if kind == "skewed":
        u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
        ids = (float(V) ** u).long().clamp_(1, V) - 1
        return torch.where(torch.rand(n, device="cuda", generator=gen) < 0.4, V // 2, ids)
    return torch.randint(0, V, (n,), device="cuda", generator=gen)


def _check(ids, V, C, dtype, out, scale, seed=0, known=None):
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    n = ids.numel()
    table = torch.randn(V, C, device="cuda", generator=gen).to(dtype).requires_grad_()
    dy = torch.randn(n, C, device="cuda", generator=gen).to(out)
    y = fused_ops.embedding(ids, table, scale=scale, out_dtype=out)
    y.backward(dy.view(y.shape))
    known = torch.ones(n, dtype=torch.bool, device="cuda") if known is None else known
    flat = ids.reshape(-1).long()
    exact = table.detach().double()[torch.where(known, flat, 0)] * scale
    got = y.detach().double().view(n, C)
    # forward: one product rounded to fp32, one rounding to the output's type
    tol = torch.finfo(out).eps / 2 + 2**-23
    assert ((got - exact).abs()[known] <= tol * exact.abs()[known]).all()
    assert got[~known].isnan().all()
    # gradient: a token's m rows are added in chains of at most 32 within a piece and 1/8 of its pieces (or in order where few), so the error
    # is below (m + 8) * 2^-24 times the sum of magnitudes, then the scale and one rounding
    want = torch.zeros(V, C, dtype=torch.float64, device="cuda").index_add_(0, flat[known], dy.double()[known]) * scale
    size = torch.zeros(V, C, dtype=torch.float64, device="cuda").index_add_(0, flat[known], dy.double().abs()[known]) * abs(scale)
    count = torch.bincount(flat[known], minlength=V).double().unsqueeze(1)
    bound = (count.clamp(max=2000) + 8) * 2**-24 * size + (torch.finfo(dtype).eps / 2 + 2**-23) * want.abs()
    assert table.grad.dtype == dtype
    assert ((table.grad.double() - want).abs() <= bound).all()
    return table.grad


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 1000, 8192, 8193, 20000, 40000])
@pytest.mark.parametrize("kind", ["uniform", "skewed", "same", "ramp"])
def test_lengths_and_distributions(n, kind):
    V = 1000
    _check(_ids(n, V, kind), V, 24, F32, F32, 1.0)


@pytest.mark.parametrize("V", [1, 2, 255, 256, 257, 65535, 65536, 70000])
def test_table_heights_around_the_digits_of_the_sort(V):
    _check(_ids(3000, V, "uniform"), V, 8, F32, F32, 0.5)


@pytest.mark.parametrize("C", [1, 3, 8, 12, 16, 100, 333, 768, 1337, 2048, 5000])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
def test_widths_and_types(C, dtype, out):
    _check(_ids(777, 500, "skewed"), 500, C, dtype, out, 3.25)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_batches_beyond_the_capacity_of_the_sort(dtype):
    for n in (65536, 65537, 150001):
        _check(_ids(n, 900, "skewed"), 900, 16, dtype, dtype, 1.0)


def test_shapes_types_and_strides_of_tokens():
    ids = _ids(60, 50, "uniform").view(3, 20)
    a = _check(ids, 50, 16, F32, F32, 1.0)
    b = _check(ids.int(), 50, 16, F32, F32, 1.0)
    c = _check(ids.t().contiguous().t(), 50, 16, F32, F32, 1.0)
    assert torch.equal(a, b) and torch.equal(a, c)
    table = torch.randn(50, 16, device="cuda", requires_grad=True)
    y = fused_ops.embedding(ids[:0], table)
    assert y.shape == (0, 20, 16)
    y.sum().backward()
    assert not table.grad.any()
    one = fused_ops.embedding(ids[0, 0], table)
    assert one.shape == (16,) and torch.equal(one, table[ids[0, 0]])


def test_tokens_outside_the_table():
    ids = _ids(500, 64, "uniform")
    ids[[3, 77, 499]] = torch.tensor([-1, 64, 1 << 40], device="cuda")
    known = (ids >= 0) & (ids < 64)
    _check(ids, 64, 24, F32, F32, 1.0, known=known)


def test_incoming_gradients_of_other_strides_and_broadcasts():
    ids = _ids(100, 40, "uniform")
    table = torch.randn(40, 12, device="cuda", requires_grad=True)
    fused_ops.embedding(ids, table).sum().backward()  # an expanded gradient
    count = torch.bincount(ids, minlength=40).float()
    assert torch.equal(table.grad, count.unsqueeze(1).expand(40, 12))
    wide = torch.randn(12, 100, device="cuda")
    (g,) = torch.autograd.grad(fused_ops.embedding(ids, table), table, wide.t())
    (h,) = torch.autograd.grad(fused_ops.embedding(ids, table), table, wide.t().contiguous())
    assert torch.equal(g, h)


def test_same_inputs_give_the_same_bits():
    ids = _ids(20000, 300, "skewed")
    a, b = (_check(ids, 300, 40, F32, BF16, 1.0) for _ in range(2))
    assert torch.equal(a, b)


def test_captured_backward_with_other_tokens_and_a_side_stream():
    ids = _ids(3000, 700, "skewed")
    table = torch.randn(700, 48, device="cuda", requires_grad=True)
    dy = torch.randn(3000, 48, device="cuda")

    def call():
        return torch.autograd.grad(fused_ops.embedding(ids, table, scale=2.0), table, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(warm, call())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (1, 2):
        ids.copy_(_ids(3000, 700, "uniform", seed))
        graph.replay()
        assert torch.equal(got, call())


def test_gpt2_with_the_fused_embedding_matches_the_module():
    cfg = dict(n_layer=1, vocab_size=1000, d_model=256, n_head=4, d_mlp=512, n_ctx=64)
    models = []
    for fused in (True, False):
        torch.manual_seed(0)
        models.append(GPT2(GPT2Config(fused_embedding=fused, **cfg)).cuda())
    idx = torch.randint(0, 1000, (4, 65), device="cuda")
    for m in models:
        m(idx[:, :-1], idx[:, 1:]).backward()
    a, b = (m.wte.weight.grad for m in models)
    # the rows' sums of at most 256 terms in two orders
    assert (a - b).abs().max() <= 256 * 2**-24 * 4 * b.abs().max()
