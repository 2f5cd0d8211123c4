"""Products of 8-bit operands with a scale per block of 128: formats, products, the linear layer and its gradients."""

import pytest
import torch

from optimizers_b200.models import Llama, LlamaConfig, fp8, fused_ops

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _x(rows, cols, dtype=BF16, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=gen) * torch.exp(torch.randn(rows, 1, device="cuda", generator=gen))
    return (x * torch.exp(torch.randn(1, cols, device="cuda", generator=gen))).to(dtype)


def _held(x, down):
    """The format's definition on 64-bit numbers, step by step; the steps that are 32-bit numbers are rounded to them."""
    rows, cols = x.shape
    p = torch.nn.functional.pad(x.double(), (0, -cols % 128, 0, -rows % down))
    b = p.view(p.shape[0] // down, down, p.shape[1] // 128, 128)
    top = b.abs().amax((1, 3), keepdim=True).clamp_min(float(torch.tensor(1e-30)))
    v = (b * (448 / top).float().double()).float().double()
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
    q = torch.round(v / step) * step
    return q.view_as(p)[:rows, :cols], (top / 448).float().view(b.shape[0], b.shape[2])


def _full(q, scale, down):
    return q * scale.double().repeat_interleave(down, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]


def _both(x):
    """Both layouts from the kernel: ((values, scales), (values, scales of the transpose))."""
    raw, scale, raw_t, scale_t = fused_ops._ext().fp8_both(x)
    return (fp8._e4m3(raw, x.shape[1]), scale.t()), (fp8._e4m3(raw_t, x.shape[0]), scale_t.t())


def _squares(w):
    raw, raw_t, scale = fused_ops._ext().fp8_squares(w, True)
    return (fp8._e4m3(raw, w.shape[1]), scale), (fp8._e4m3(raw_t, w.shape[0]), scale.t())


def _product(a, b, column, out, addend=None):
    return fused_ops._ext().fp8_matmul(
        a[0].view(torch.uint8), a[1], b[0].view(torch.uint8), b[1], column, out == BF16, addend, fp8._status_of(a[0].device)
    )


SHAPES = [(1, 1), (1, 16), (3, 127), (5, 128), (7, 129), (128, 128), (127, 300), (129, 256), (257, 1000), (300, 1337)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_formats_are_the_definition_bit_for_bit(shape, dtype):
    x = _x(*shape, dtype)
    q, s = _held(x, 1)
    rows = fp8.quantize_rows(x)
    assert torch.equal(rows.scale, s) and torch.equal(rows.data.double(), q)
    (a, sa), (b, sb) = _both(x)
    assert torch.equal(sa, s) and torch.equal(a.double(), q)
    qt, st = _held(x.t(), 1)
    assert torch.equal(sb, st) and torch.equal(b.double(), qt)
    qw, sw = _held(x, 128)
    (c, sc), (d, sd) = _squares(x)
    assert torch.equal(sc, sw) and torch.equal(c.double(), qw)
    assert torch.equal(sd, sw.t()) and torch.equal(d.double(), qw.t())
    w = fp8.quantize_weight(x)
    assert torch.equal(w.scale, sw) and torch.equal(w.data.double(), qw)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_formats_of_strided_unaligned_and_extreme_sources(dtype):
    wide = _x(40, 700, dtype)
    for view in (wide[:, 3:300], wide[:, 8:264], wide[::2, :256], wide.t(), wide[5:6, 1:2]):
        for got, want in zip(fp8._rows(view, True), fp8._rows(view.contiguous(), True)):
            assert torch.equal(got.float(), want.float())
        source = fp8._source(view)
        for got, want in zip(_both(source), _both(view.contiguous())):
            assert torch.equal(got[0].float(), want[0].float()) and torch.equal(got[1], want[1])
    x = torch.zeros(4, 256, device="cuda", dtype=dtype)
    x[1, :128] = 1e-38
    x[2] = 3e38
    x[3, 128:] = -1e-29
    rows = fp8.quantize_rows(x)
    q, s = _held(x, 1)
    assert torch.equal(rows.scale, s) and torch.equal(rows.data.double(), q)
    assert not rows.dequantize()[0].any()
    x[0, 5], x[1, 200] = float("nan"), float("inf")
    rows = fp8.quantize_rows(x)
    v = rows.dequantize()
    assert v[0, :128].isnan().all() and not v[0, 128:].any() and v[1, 128:].isnan().all() and torch.equal(v[2:], _full(q, s, 1)[2:].float())


def _product_case(M, N, K, column, out, addend, seed=0):
    a, sa = fp8._rows(_x(M, K, F32, seed), True)
    b, sb = fp8._rows(_x(N, K, F32, seed + 1), True) if column else fp8._squares(_x(N, K, F32, seed + 1), True)
    add = _x(M, N, F32, seed + 2) if addend else None
    got = _product((a, sa), (b, sb), column, out, add)
    fa, fb = _full(a.double(), sa, 1), _full(b.double(), sb, 1 if column else 128)
    want = fa @ fb.t() + (add.double() if addend else 0)
    size = fa.abs() @ fb.abs().t() + (add.double().abs() if addend else 0)
    # a group: 128 exact products added in 32 bits by the tensor core (at most 128 units of 2^-23, it may cut instead of round); scales: two
    # products; groups: one unit each
    units = (128 + 4 + K / 128) * 2**-23
    assert got.dtype == out and ((got.double() - want).abs() <= torch.finfo(out).eps / 2 * want.abs() + units * size).all()
    return got


SIZES = [
    (1, 1, 1), (1, 64, 128), (2, 65, 129), (4, 2048, 1024), (128, 128, 128), (127, 127, 127), (129, 257, 300), (1, 1000, 4000), (200, 16, 4096),
    (16, 333, 1337), (1001, 333, 1337), (1024, 1024, 512), (2500, 1111, 640), (4096, 4100, 300), (100, 20000, 256), (20000, 100, 256),
]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("column", [False, True])
@pytest.mark.parametrize("out", [F32, BF16])
def test_products(size, column, out):
    _product_case(*size, column, out, addend=False)


@pytest.mark.parametrize("size", [(1, 1, 1), (129, 257, 300), (1001, 333, 1337), (4096, 4096, 256)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_products_with_an_addend(size, out):
    _product_case(*size, False, out, addend=True)


def test_products_leave_their_neighbours_alone_and_repeat():
    first = _product_case(300, 270, 500, False, F32, False)
    for _ in range(3):
        assert torch.equal(first, _product_case(300, 270, 500, False, F32, False))
    fp8.check_status()


def test_non_finite_groups_reach_their_rows_only():
    x, w = _x(70, 384), _x(130, 384, F32, 1)
    clean = fp8.linear(x, w)
    x[7, 200] = float("nan")
    x[9, 1] = float("inf")
    got = fp8.linear(x, w)
    assert got[7].isnan().all() and got[9].isnan().all()
    keep = [i for i in range(70) if i not in (7, 9)]
    assert torch.equal(got[keep], clean[keep])


def _linear_case(T, N, K, x_dtype, w_dtype, seed=0):
    x = _x(T, K, x_dtype, seed).requires_grad_()
    w = _x(N, K, w_dtype, seed + 1).requires_grad_()
    y = fp8.linear(x, w)
    dy = _x(T, N, y.dtype, seed + 2)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert (y.dtype, dx.dtype, dw.dtype) == (x_dtype, x_dtype, w_dtype)
    fw, fx, fd = _full(*_held(w, 128), 128), _full(*_held(x, 1), 1), _full(*_held(dy, 1), 1)
    fxt, fdt = _full(*_held(x.t(), 1), 1), _full(*_held(dy.t(), 1), 1)
    for got, a, b in ((y, fx, fw.t()), (dx, fd, fw), (dw, fdt, fxt.t())):
        want, size = a @ b, a.abs() @ b.abs()
        units = (132 + a.shape[1] / 128) * 2**-23
        assert ((got.double() - want).abs() <= torch.finfo(got.dtype).eps / 2 * want.abs() + units * size).all()
    return y, dx, dw


@pytest.mark.parametrize("size", [(1, 1, 1), (1, 256, 128), (5, 33, 200), (128, 256, 384), (333, 257, 129), (1001, 333, 1337), (2048, 1024, 768)])
@pytest.mark.parametrize("kinds", [(BF16, F32), (BF16, BF16), (F32, F32)])
def test_linear_and_its_gradients(size, kinds):
    _linear_case(*size, *kinds)


def test_linear_is_near_the_unrounded_layer():
    # e4m3 rounds each operand by at most 2^-4 of its value (rms about 0.026); products of independent roundings average out
    x, w = torch.randn(300, 512, device="cuda"), torch.randn(200, 512, device="cuda")
    y = fp8.linear(x, w).double()
    want = x.double() @ w.double().t()
    assert (y - want).norm() <= 2 * 2**-4 * want.norm()


def test_gradients_against_differences_of_the_held_operands():
    """Steps that stay on the grid of the format: the product is bilinear in the held values, so differences are exact to rounding."""
    torch.manual_seed(0)
    x = torch.randint(-8, 9, (4, 128), device="cuda").float()
    w = torch.randint(-8, 9, (6, 128), device="cuda").float()
    x[:, 0] = 448.0  # factors of one for x's rows, and for its columns' groups once every column has it
    w[0, 0] = 448.0
    c = torch.randint(-8, 9, (4, 6), device="cuda").float()
    c[0, :] = 448.0
    c[:, 0] = 448.0
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = fp8.linear(xr, wr)
    (dx,) = torch.autograd.grad(y, xr, c, retain_graph=True)
    for i, j in ((0, 1), (2, 5), (3, 127)):
        moved = x.clone()
        moved[i, j] += 1.0
        diff = ((fp8.linear(moved, w) - y.detach()).double() * c.double()).sum()
        assert abs(float((diff - dx[i, j]).detach())) <= 1e-5 * float((c.double().abs() @ w.double().abs())[i, j]) + 2**-23 * float(y.detach().abs().max()) * 448 * 6


def test_several_weights_share_x():
    x = _x(150, 320).requires_grad_()
    ws = [_x(n, 320, F32, n).requires_grad_() for n in (64, 200, 33)]
    ys = fp8.linear(x, tuple(ws))
    dys = [_x(150, n, BF16, n + 1) for n in (64, 200, 33)]
    got = torch.autograd.grad(ys, [x, *ws], dys)
    total = torch.zeros(150, 320, dtype=torch.float64, device="cuda")
    size = total.clone()
    for w, y, dy, dw in zip(ws, ys, dys, got[1:]):
        one = fp8.linear(x, w)
        assert torch.equal(one, y)
        dx1, dw1 = torch.autograd.grad(one, (x, w), dy)
        assert torch.equal(dw, dw1)
        a, b = _full(*_held(dy, 1), 1), _full(*_held(w, 128), 128)
        total += a @ b
        size += a.abs() @ b.abs()
    assert ((got[0].double() - total).abs() <= 2**-8 * total.abs() + 140 * 2**-23 * size).all()
    part = fp8.linear(x, tuple(ws))
    dx, dw = torch.autograd.grad(part[1], (x, ws[1]), dys[1])  # the other results are not used
    one = torch.autograd.grad(fp8.linear(x, ws[1]), (x, ws[1]), dys[1])
    assert torch.equal(dx, one[0]) and torch.equal(dw, one[1])


def test_parts_of_the_gradient():
    x, w = _x(77, 200), _x(50, 200, F32, 1)
    dy = _x(77, 50, BF16, 2)
    full = torch.autograd.grad(fp8.linear(a := x.clone().requires_grad_(), b := w.clone().requires_grad_()), (a, b), dy)
    (dx,) = torch.autograd.grad(fp8.linear(a, w), a, dy)
    (dw,) = torch.autograd.grad(fp8.linear(x, b), b, dy)
    assert torch.equal(dx, full[0]) and torch.equal(dw, full[1])
    (gx,) = torch.autograd.grad(fp8.linear(a, w).sum(), a)  # an expanded gradient
    (hx,) = torch.autograd.grad(fp8.linear(a, w), a, torch.ones(77, 50, device="cuda", dtype=BF16))
    assert torch.equal(gx, hx)
    (tx,) = torch.autograd.grad(fp8.linear(a, w), a, dy.t().contiguous().t())
    assert torch.equal(tx, full[0])


def test_held_operands_give_the_same_bits():
    x, w = _x(30, 500), _x(260, 500, F32, 1)
    with torch.no_grad():
        want = fp8.linear(x, w)
        held = fp8.quantize_weight(w)
        rows = fp8.quantize_rows(x)
        assert torch.equal(fp8.linear(x, held), want) and torch.equal(fp8.linear(rows, held), want) and torch.equal(fp8.linear(rows, w), want)
        packed = fp8.Weight(held.data.contiguous(), held.scale.t().contiguous().t())  # rows 500 bytes apart, other strides of the scales
        assert torch.equal(fp8.linear(x, packed), want)
        loose = fp8.Rows(rows.data.contiguous(), rows.scale.contiguous())
        assert torch.equal(fp8.linear(loose, packed, out_dtype=F32).to(BF16), want)
    assert torch.equal(fp8.linear(x.clone().requires_grad_(), w).detach(), want)


def test_empty_operands():
    w = _x(40, 200, F32).requires_grad_()
    x = torch.empty(0, 200, device="cuda", dtype=BF16, requires_grad=True)
    y = fp8.linear(x, w)
    assert y.shape == (0, 40)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert dx.shape == (0, 200) and not dw.any()


def test_other_streams_and_capture():
    x, w = _x(300, 256).requires_grad_(), _x(512, 256, F32, 1).requires_grad_()
    dy = _x(300, 512, BF16, 2)

    def call():
        y = fp8.linear(x, w)
        # (an autograd graph of the same leaves that was built outside must not be alive while one is captured: hence detach)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (5, 6):
        with torch.no_grad():
            x.copy_(_x(300, 256, BF16, seed))
            w.copy_(_x(512, 256, F32, seed + 1))
        graph.replay()
        for a, b in zip(got, call()):
            assert torch.equal(a, b)


def _llama(**kw):
    torch.manual_seed(0)
    cfg = dict(vocab_size=500, n_layer=2, n_head=4, d_model=256, d_ffn=640, max_seq=64)
    return Llama(LlamaConfig(**(cfg | kw))).cuda()


def test_llama_runs_all_of_it_together():
    """Embedding, residual norms, 8-bit layers, loss and clipping in one training step; evaluation with and without kept weights."""
    from optimizers_b200 import clip_grad_norm_

    model, plain = _llama(fp8=True, fused_embedding=True), _llama()
    idx = torch.randint(0, 500, (3, 34), device="cuda")
    count = fused_ops.launches()
    losses = []
    for m in (model, plain):
        with torch.autocast("cuda", dtype=BF16):
            loss = m(idx[:, :-1], idx[:, 1:])
        loss.backward()
        losses.append(float(loss))
    assert fused_ops.launches() > count
    # two layers whose products are off by about 2^-5 rms each, in a loss of about log 500 over random weights of 0.02
    assert abs(losses[0] - losses[1]) < 0.05
    for (name, a), (_, b) in zip(model.named_parameters(), plain.named_parameters()):
        assert a.grad is not None and a.grad.isfinite().all(), name
        cosine = float(torch.nn.functional.cosine_similarity(a.grad.flatten(), b.grad.flatten(), dim=0))
        assert cosine > 0.9, (name, cosine)
    norm = clip_grad_norm_(model.parameters(), 1e-3)
    after = torch.sqrt(sum(p.grad.double().square().sum() for p in model.parameters()))
    assert float(norm) > 1e-3 and abs(float(after) - 1e-3) < 1e-6
    model.eval()
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        logits = model(idx)
        model.hold_fp8_weights()
        held = model(idx)
        reference = plain(idx)
    assert torch.equal(logits, held)
    assert torch.nn.functional.cosine_similarity(logits.float().flatten(), reference.float().flatten(), dim=0) > 0.95
    model.train()
    assert all(layer._held is None for layer in model.layers)
    fp8.check_status()


def test_inference_mode():
    x, w, r = _x(20, 256), _x(64, 256, F32, 1), _x(20, 256, F32, 2)
    weight, table, ids = torch.ones(256, device="cuda"), _x(30, 16, F32), torch.arange(10, device="cuda")
    with torch.inference_mode():
        y = fp8.linear(x, (w, w))[1]
        n, h = fused_ops.add_rms_norm(x, r, weight)
        rows, h8 = fp8.add_rms_norm(x, r, weight)
        e = fused_ops.embedding(ids, table)
        z = fp8.linear(rows, fp8.quantize_weight(w))
    with torch.no_grad():
        assert torch.equal(y, fp8.linear(x, w)) and torch.equal(h, h8) and torch.equal(e, table[:10])
        m, k = fused_ops.add_rms_norm(x, r, weight)
        assert torch.equal(n, m) and torch.equal(h, k)
        assert torch.equal(z, fp8.linear(rows, w))


def test_differentiating_a_gradient_again_is_refused():
    x, w = _x(9, 130, F32).requires_grad_(), _x(20, 130, F32, 1).requires_grad_()
    r, n, table = _x(9, 130, F32, 2).requires_grad_(), torch.ones(130, device="cuda", requires_grad=True), _x(30, 16, F32).requires_grad_()
    for out, leaf in (
        (fp8.linear(x, w), x), (fused_ops.add_rms_norm(x, r, n)[0], x), (fused_ops.embedding(torch.arange(4, device="cuda"), table), table)
    ):
        (g,) = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="again"):
            g.sum().backward()
        with pytest.raises(RuntimeError):  # (nothing leads from the gradient back to the leaf)
            torch.autograd.grad(g.sum(), leaf)


def test_in_place_changes_of_what_the_backward_pass_needs_are_found():
    x, r, n = _x(9, 128, F32).requires_grad_(), _x(9, 128, F32, 1).requires_grad_(), torch.ones(128, device="cuda", requires_grad=True)
    y, h = fused_ops.add_rms_norm(x, r, n)
    with torch.no_grad():
        h += 1.0
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_batches_of_incoming_gradients_are_refused():
    x, w = _x(9, 130, F32).requires_grad_(), _x(20, 130, F32, 1).requires_grad_()
    r, n, table = _x(9, 130, F32, 2).requires_grad_(), torch.ones(130, device="cuda", requires_grad=True), _x(30, 16, F32).requires_grad_()
    for out, leaf in (
        (fp8.linear(x, w), x), (fused_ops.add_rms_norm(x, r, n)[0], x), (fused_ops.embedding(torch.arange(4, device="cuda"), table), table)
    ):
        with pytest.raises(RuntimeError, match="one gradient at a time"):
            torch.autograd.grad(out, leaf, torch.ones(3, *out.shape, device="cuda"), is_grads_batched=True)
