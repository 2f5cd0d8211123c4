"""Gradient norm and clipping on the GPU against 64-bit formulas."""

import math

import pytest
import torch

from optimizers_b200 import clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _params(shapes, dtype=F32, offset=0, seed=0):
    """Parameters whose gradients are packed behind one another, the first ``offset`` elements into a buffer."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    sizes = [math.prod(s) for s in shapes]
    flat = torch.randn(offset + sum(sizes) + 8, device="cuda", generator=gen).to(dtype)
    params, at = [], offset
    for s, n in zip(shapes, sizes):
        p = torch.nn.Parameter(torch.empty(s, device="cuda", dtype=dtype))
        p.grad = flat[at : at + n].view(s)
        params.append(p)
        at += n
    return params, flat


def _check(params, max_norm, given=None):
    """Clips ``given`` (by default the distinct ``params``) and compares with the formula over ``params``."""
    before = [p.grad.clone() for p in params]
    true = math.sqrt(sum(float(g.double().square().sum()) for g in before))
    got = clip_grad_norm_(params if given is None else given, max_norm)
    # The norm: an fp32 sum of n squares added in chains of at most a few hundred and then in a tree; each of the terms is positive, so its
    # relative error is below (chain + tree + 2) * 2^-24 < 512 * 2^-24 = 3e-5, and half of that after the root.
    assert got.shape == () and got.dtype == F32
    assert abs(float(got) - true) <= 1.6e-5 * true
    factor = min(1.0, max_norm / (true + 1e-6))
    for p, g in zip(params, before):
        # one rounding to the gradient's type, the factor's own error, one product rounded to fp32
        tol = torch.finfo(g.dtype).eps / 2 + 2e-5 + 2**-24
        want = g.double() * factor
        small = torch.finfo(g.dtype).smallest_normal  # fp16: below it the step is absolute
        assert ((p.grad.double() - want).abs() <= tol * want.abs() + small * torch.finfo(g.dtype).eps).all()
    return got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_odd_sizes_and_alignments(dtype, offset):
    params, flat = _params([(1,), (7,), (3, 5), (129,), (1000, 13), (4097,), (2,), (64, 64), (33000,)], dtype, offset)
    edge = (flat[:offset].clone(), flat[-8:].clone())
    _check(params, 1.0)
    assert torch.equal(flat[:offset], edge[0]) and torch.equal(flat[-8:], edge[1])  # neighbours of the gradients stay


@pytest.mark.parametrize("count", [1, 31, 32, 33, 180, 181, 1500, 1501, 3100])
def test_numbers_of_gradients_around_the_table_sizes(count):
    params, _ = _params([(5 + i % 7,) for i in range(count)])
    _check(params, 0.5)


def test_large_gradients_span_many_chunks():
    params, _ = _params([(3000, 2777), (11,), (5000, 1024)], F32, 1)
    _check(params, 2.0)


def test_mixed_types_and_layouts():
    a, _ = _params([(40, 30), (17,)], F32)
    b, _ = _params([(50, 20), (9,)], BF16)
    c, _ = _params([(64,)], F16)
    conv = torch.nn.Parameter(torch.empty(8, 4, 3, 3, device="cuda").to(memory_format=torch.channels_last))
    conv.grad = torch.randn(8, 4, 3, 3, device="cuda").to(memory_format=torch.channels_last)
    strided = torch.nn.Parameter(torch.empty(10, 6, device="cuda"))
    wide = torch.randn(10, 12, device="cuda")
    strided.grad = wide[:, ::2]
    rest = wide[:, 1::2].clone()
    none = torch.nn.Parameter(torch.empty(3, device="cuda"))
    empty = torch.nn.Parameter(torch.empty(0, device="cuda"))
    empty.grad = torch.empty(0, device="cuda")
    _check(a + b + c + [conv, strided, empty], 0.7)
    assert torch.equal(wide[:, 1::2], rest)
    assert float(clip_grad_norm_([none], 1.0)) == 0.0 and float(clip_grad_norm_([empty], 1.0)) == 0.0
    assert float(clip_grad_norm_([], 1.0)) == 0.0


def test_small_norms_are_left_alone_bit_for_bit():
    params, flat = _params([(100, 100), (33,)], BF16)
    before = flat.clone()
    _check(params, 1e6)
    assert torch.equal(flat, before)
    clip_grad_norm_(params, math.inf)
    assert torch.equal(flat, before)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_norms_that_are_not_finite(value):
    params, flat = _params([(100, 10), (33,)])
    params[0].grad[3, 4] = value
    before = flat.clone()
    with pytest.raises(RuntimeError, match="norm"):
        clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
    assert torch.equal(flat.nan_to_num(7.0), before.nan_to_num(7.0))
    got = clip_grad_norm_(params, 1.0)
    norm = torch.linalg.vector_norm(before[:1033])
    want = before[:1033] * (1.0 / (norm + 1e-6)).clamp(max=1.0)
    assert torch.equal(got.isnan(), norm.isnan()) and (got.isnan() or torch.isinf(got))
    assert torch.equal(flat[:1033].isnan(), want.isnan())
    assert torch.equal(flat[:1033].nan_to_num(0.0), want.nan_to_num(0.0))


def test_zero_gradients_and_zero_bound():
    params, flat = _params([(100,)])
    flat.zero_()
    assert float(clip_grad_norm_(params, 1.0)) == 0.0 and not flat.any()
    params, flat = _params([(100,)])
    clip_grad_norm_(params, 0.0)
    assert not flat[:100].any()


def test_same_parameter_twice_counts_once_and_shared_memory_is_refused():
    params, flat = _params([(50, 20)])
    once = float(grad_norm(params))
    assert float(grad_norm(params + params)) == once
    _check(params, 1.0, given=params + params)
    other = torch.nn.Parameter(torch.empty(18, device="cuda"))
    other.grad = flat[990:1008]
    before = flat.clone()
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_(params + [other], 1.0)
    assert torch.equal(flat, before)


def test_same_inputs_give_the_same_bits():
    params, flat = _params([(3000, 777), (55,)])
    before = flat.clone()
    results = set()
    for _ in range(5):
        flat.copy_(before)
        results.add(float(clip_grad_norm_(params, 1.0)))
    assert len(results) == 1


def test_on_another_stream_and_captured():
    params, flat = _params([(300, 77), (55,)])
    before = flat.clone()
    want = float(clip_grad_norm_(params, 1.0))
    after = flat.clone()
    flat.copy_(before)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = clip_grad_norm_(params, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert float(got) == want and torch.equal(flat, after)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(params, 1.0)
    for scale in (1.0, 3.0, 1e-9):
        flat.copy_(before * scale)
        graph.replay()
        expected = before * scale
        p2, f2 = _params([(300, 77), (55,)])
        f2.copy_(expected)
        eager = clip_grad_norm_(p2, 1.0)
        assert torch.equal(norm, eager) and torch.equal(flat, f2)


def test_grad_norm_matches_and_changes_nothing():
    params, flat = _params([(300, 77), (55,)], BF16, 3)
    before = flat.clone()
    true = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
    assert abs(float(grad_norm(params)) - true) <= 1.6e-5 * true
    assert torch.equal(flat, before)
