"""Residual addition + RMSNorm on the GPU against 64-bit formulas, its gradients, and its 8-bit form."""

import pytest
import torch

from optimizers_b200.models import fp8, fused_ops

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
KINDS = [(BF16, F32), (BF16, BF16), (F32, F32), (F32, BF16)]
EPS = 1e-5


def _inputs(rows, C, x_dtype, r_dtype, seed=0, offset=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def make(dtype):
        flat = torch.randn(rows * C + offset, device="cuda", generator=gen).to(dtype)
        return flat[offset:].view(rows, C)

    return make(x_dtype), make(r_dtype), 1 + 0.3 * torch.randn(C, device="cuda", generator=gen)


def _check(x, r, w, seed=1):
    rows, C = x.shape
    gen = torch.Generator(device="cuda").manual_seed(seed)
    leaves = [t.detach().requires_grad_() for t in (x, r, w)]
    y, h = fused_ops.add_rms_norm(*leaves, eps=EPS)
    wide = torch.promote_types(x.dtype, r.dtype)
    assert y.dtype == x.dtype and h.dtype == wide
    hd = h.detach().double()
    hx = x.double() + r.double()
    assert ((hd - hx).abs() <= (torch.finfo(wide).eps / 2 + 2**-24) * hx.abs()).all()
    rs = (hd.square().mean(1, keepdim=True) + EPS).rsqrt()
    z, wd = hd * rs, w.double()
    # C squares in chains of at most 16 and trees, the mean, the root (2 units) and two products: under 40 units of 2^-24 relative
    tol = 40 * 2**-24
    assert ((y.double() - z * wd).abs() <= (torch.finfo(y.dtype).eps / 2 + tol) * (z * wd).abs()).all()
    dy = torch.randn(rows, C, device="cuda", generator=gen).to(y.dtype)
    dh = torch.randn(rows, C, device="cuda", generator=gen).to(h.dtype)
    dx, dr, dw = torch.autograd.grad((y, h), leaves, (dy, dh))
    assert (dx.dtype, dr.dtype, dw.dtype) == (x.dtype, r.dtype, w.dtype)
    g = dy.double() * wd
    mean = (g * z).mean(1, keepdim=True)
    want = dh.double() + rs * (g - z * mean)
    # the terms' own roundings: under 60 units of their magnitudes (the mean's are those of the magnitudes it adds)
    size = dh.double().abs() + rs * (g.abs() + z.abs() * (g * z).abs().mean(1, keepdim=True))
    for got in (dx, dr):
        extra = torch.finfo(wide).eps / 2 if got.dtype != wide else 0.0  # dr of a bf16 residual next to an fp32 x
        assert ((got.double() - want).abs() <= (torch.finfo(got.dtype).eps / 2 + extra) * want.abs() + 60 * 2**-24 * size).all()
    dwant, dsize = (dy.double() * z).sum(0), (dy.double() * z).abs().sum(0)
    # a column is added in chains of rows / 592 (at least 1) per CTA, then of at most 74, then 8: under 300 units here
    assert ((dw.double() - dwant).abs() <= torch.finfo(dw.dtype).eps / 2 * dwant.abs() + 300 * 2**-24 * dsize).all()
    return y, h, dx, dr, dw


@pytest.mark.parametrize("C", [1, 2, 7, 8, 31, 128, 200, 256, 257, 264, 512, 520, 768, 1000, 1024, 1032, 1337, 2048, 4096, 4104, 8192, 8200, 12345, 16384])
@pytest.mark.parametrize("kinds", KINDS)
def test_widths_and_types(C, kinds):
    _check(*_inputs(19, C, *kinds))


@pytest.mark.parametrize("rows", [1, 2, 3, 7, 8, 9, 600, 5000])
@pytest.mark.parametrize("C", [96, 768, 2048])
def test_numbers_of_rows(rows, C):
    _check(*_inputs(rows, C, BF16, F32))


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_unaligned_rows(offset):
    x, r, w = _inputs(9, 512, BF16, F32, offset=offset)
    a = _check(x, r, w)
    b = _check(x.clone(), r.clone(), w)
    for s, t in zip(a, b):
        assert torch.equal(s, t)


def test_bf16_weight_shapes_and_strides():
    x, r, w = _inputs(24, 300, BF16, F32)
    _check(x, r, w.to(BF16))
    y, h = fused_ops.add_rms_norm(x.view(2, 3, 4, 300), r.view(2, 3, 4, 300), w, eps=EPS)
    y2, h2 = fused_ops.add_rms_norm(x, r, w, eps=EPS)
    assert y.shape == (2, 3, 4, 300) and torch.equal(y.view(24, 300), y2) and torch.equal(h.view(24, 300), h2)
    xt, rt = x.t().contiguous().t(), r.t().contiguous().t()
    y3, _ = fused_ops.add_rms_norm(xt, rt, w, eps=EPS)
    assert torch.equal(y3, y2)
    e, f = fused_ops.add_rms_norm(x[:0], r[:0], w, eps=EPS)
    assert e.shape == (0, 300) and f.shape == (0, 300)


def test_partial_gradients():
    x, r, w = _inputs(33, 640, BF16, F32)
    leaves = [t.detach().requires_grad_() for t in (x, r, w)]
    y, h = fused_ops.add_rms_norm(*leaves, eps=EPS)
    dy, dh = torch.randn_like(y), torch.randn_like(h)
    both = torch.autograd.grad((y, h), leaves, (dy, dh), retain_graph=True)
    only_y = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    zero = torch.autograd.grad((y, h), leaves, (dy, torch.zeros_like(dh)), retain_graph=True)
    for a, b in zip(only_y, zero):
        assert torch.equal(a, b)
    only_h = torch.autograd.grad(h, leaves, dh, retain_graph=True)
    assert torch.equal(only_h[0], dh.to(BF16)) and torch.equal(only_h[1], dh) and not only_h[2].any()
    assert torch.equal(both[2], only_y[2])
    leaves[0].requires_grad_(False)
    y, h = fused_ops.add_rms_norm(leaves[0], leaves[1], leaves[2], eps=EPS)
    dr, dw = torch.autograd.grad((y, h), leaves[1:], (dy, dh))
    assert torch.equal(dr, both[1]) and torch.equal(dw, both[2])


def test_zero_and_non_finite_rows_stay_in_their_rows():
    x, r, w = _inputs(6, 384, BF16, F32)
    x[1] = 0
    r[1] = 0
    clean = fused_ops.add_rms_norm(x, r, w, eps=EPS)[0]
    assert not clean[1].any()
    x[3, 5], x[4, 5] = float("inf"), float("nan")
    got = fused_ops.add_rms_norm(x, r, w, eps=EPS)[0]
    for row in (0, 1, 2, 5):
        assert torch.equal(got[row], clean[row])
    assert got[3, 5].isnan() and got[4].isnan().all() and not got[3, 6:].any()


def test_autocast_gives_bf16():
    x, r, w = _inputs(5, 256, F32, F32)
    with torch.autocast("cuda", dtype=BF16):
        y, h = fused_ops.add_rms_norm(x, r, w, eps=EPS)
    assert y.dtype == BF16 and h.dtype == F32


def test_gradients_against_differences():
    torch.manual_seed(0)
    x, r, w = (torch.randn(3, 72, device="cuda") for _ in range(3))
    w = w[0].contiguous()
    cy, ch = torch.randn(3, 72, device="cuda"), torch.randn(3, 72, device="cuda")

    def value(*t):
        y, h = fused_ops.add_rms_norm(*t, eps=EPS)
        return (y.double() * cy).sum() + (h.double() * ch).sum()

    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = fused_ops.add_rms_norm(*leaves, eps=EPS)
    grads = torch.autograd.grad((y, h), leaves, (cy, ch))
    for i, g in enumerate(grads):
        d = torch.randn_like(leaves[i])
        step = 2**-6
        moved = [[t.detach() + (s * step * d if j == i else 0) for j, t in enumerate(leaves)] for s in (1, -1)]
        slope = float(value(*moved[0]) - value(*moved[1])) / (2 * step)
        # fp32 values of order 10 give the difference an error of about 216 * 2^-24 * 10 / step = 0.01; the cubic term is of order step^2 * |d|^3
        assert abs(slope - float((g.double() * d).sum())) <= 0.05 + 5e-3 * abs(slope)


@pytest.mark.parametrize("C", [1, 16, 100, 127, 128, 129, 256, 1000, 1337, 2048, 4100, 8192, 16000])
@pytest.mark.parametrize("kinds", KINDS)
def test_eight_bit_rows(C, kinds):
    x, r, w = _inputs(11, C, *kinds)
    rows, h = fp8.add_rms_norm(x, r, w, eps=EPS)
    y, h2 = fused_ops.add_rms_norm(x.float(), r.float(), w, eps=EPS) if h.dtype == F32 else fused_ops.add_rms_norm(x, r, w, eps=EPS)
    assert torch.equal(h, h2)
    hd = h.double()
    want = hd * (hd.square().mean(1, keepdim=True) + EPS).rsqrt() * w.double()
    padded = torch.nn.functional.pad(want, (0, -C % 128)).view(11, -1, 128)
    top = padded.abs().amax(2)
    assert rows.scale.shape == top.shape and ((rows.scale.double() * 448 - top).abs() <= 42 * 2**-24 * top).all()
    got = rows.dequantize().double()
    # half a step of e4m3 relative to the value (2^-4), or half of its smallest step (2^-10) times the scale; and the norm's own error
    scale = rows.scale.double().repeat_interleave(128, 1)[:, :C]
    assert ((got - want).abs() <= (2**-4 + 42 * 2**-24) * want.abs() + 2**-10 * scale).all()
    alone, same = fp8.add_rms_norm(h.to(x.dtype), None, w, eps=EPS)
    assert same.shape == h.shape
    if h.dtype == x.dtype:
        assert torch.equal(alone.data.view(torch.uint8), rows.data.view(torch.uint8)) and torch.equal(alone.scale, rows.scale)


def test_captured_forward_and_backward():
    x, r, w = _inputs(130, 768, BF16, F32)
    leaves = [t.detach().requires_grad_() for t in (x, r, w)]
    dy, dh = torch.randn(130, 768, device="cuda").to(BF16), torch.randn(130, 768, device="cuda")

    def call():
        y, h = fused_ops.add_rms_norm(*leaves, eps=EPS)
        return (y, h, *torch.autograd.grad((y, h), leaves, (dy, dh)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (3, 4):
        with torch.no_grad():
            for t, new in zip(leaves, _inputs(130, 768, BF16, F32, seed)):
                t.copy_(new)
        graph.replay()
        for a, b in zip(got, call()):
            assert torch.equal(a, b)
