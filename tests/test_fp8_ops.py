"""The decoder's operators on the CPU: formulas, gradients and refusals."""

import pytest
import torch

from optimizers_b200.examples import train
from optimizers_b200.models import Llama, LlamaConfig, fp8, fused_ops

F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64


@pytest.mark.parametrize("shape", [(1, 1), (3, 128), (5, 200), (130, 300)])
def test_formats(shape):
    torch.manual_seed(0)
    x = torch.randn(shape)
    rows, w = fp8.quantize_rows(x), fp8.quantize_weight(x)
    groups = -(-shape[1] // 128)
    assert rows.data.dtype == torch.float8_e4m3fn and rows.scale.shape == (shape[0], groups) and w.scale.shape == (-(-shape[0] // 128), groups)
    for held, scale in ((rows, rows.scale.repeat_interleave(128, 1)), (w, w.scale.repeat_interleave(128, 0)[: shape[0]].repeat_interleave(128, 1))):
        s = scale[:, : shape[1]]
        # half a step: 2^-4 of the value, or half of the smallest step (2^-9) of the scale; two products rounded to 32 bits
        assert ((held.dequantize() - x).abs() <= (2**-4 + 2**-22) * x.abs() + 2**-10 * s).all()
    assert (rows.data.float().abs().amax(1) == 448).all() or shape[1] > 128


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, F32), (BF16, BF16)])
def test_linear_and_gradients_on_held_values(kinds):
    torch.manual_seed(0)
    x = torch.randn(2, 7, 200).to(kinds[0]).requires_grad_()
    w = torch.randn(40, 200).to(kinds[1]).requires_grad_()
    y = fp8.linear(x, w)
    dy = torch.randn(2, 7, 40).to(y.dtype)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.shape == (2, 7, 40) and (y.dtype, dx.dtype, dw.dtype) == (kinds[0], kinds[0], kinds[1])
    x2, d2 = x.detach().view(14, 200), dy.view(14, 40)
    hw, hx, hd = fp8.quantize_weight(w).dequantize().double(), fp8.quantize_rows(x2).dequantize().double(), fp8.quantize_rows(d2).dequantize().double()
    hxt, hdt = fp8.quantize_rows(x2.t()).dequantize().double(), fp8.quantize_rows(d2.t()).dequantize().double()
    for got, a, b in ((y.view(14, 40), hx, hw.t()), (dx.view(14, 200), hd, hw), (dw, hdt, hxt.t())):
        size = a.abs() @ b.abs()
        # the dequantised operands are 32-bit products; sums of up to 200 terms
        assert ((got.double() - a @ b).abs() <= torch.finfo(got.dtype).eps / 2 * (a @ b).abs() + 210 * 2**-24 * size).all()


def test_linear_with_several_weights_and_held_operands():
    torch.manual_seed(0)
    x = torch.randn(9, 150)
    ws = (torch.randn(20, 150), torch.randn(7, 150))
    with torch.no_grad():
        a, b = fp8.linear(x, ws)
        assert torch.equal(a, fp8.linear(x, ws[0])) and torch.equal(b, fp8.linear(x, fp8.quantize_weight(ws[1])))
        assert torch.equal(fp8.linear(fp8.quantize_rows(x), ws[0], out_dtype=F32), a)
        assert fp8.linear(fp8.quantize_rows(x), ws[0]).dtype == BF16


def test_linear_without_rows():
    w = torch.randn(4, 5, requires_grad=True)
    y = fp8.linear(torch.randn(0, 5, requires_grad=True), w)
    y.sum().backward()
    assert y.shape == (0, 4) and not w.grad.any()


def test_first_use_inside_a_capture_is_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(fp8, "_status", {})
    with pytest.raises(RuntimeError, match="before capturing"):
        fp8._status_of(torch.device("cpu"))


def test_refusals_of_linear():
    x, w = torch.randn(4, 130), torch.randn(6, 130)
    with pytest.raises(ValueError, match="fit"):
        fp8.linear(x, torch.randn(6, 131))
    with pytest.raises(ValueError, match="weight"):
        fp8.linear(x, ())
    for empty in (torch.randn(4, 0), torch.tensor(1.0)):
        with pytest.raises(ValueError, match="at least one value"):
            fp8.linear(empty, torch.randn(6, 0))
    with pytest.raises(ValueError, match="floating"):
        fp8.linear(x, w, out_dtype=torch.int32)
    with pytest.raises(ValueError, match="floating"):
        fp8.linear(x.long(), w, out_dtype=F32)
    held = fp8.quantize_weight(w)
    with pytest.raises(ValueError, match="no gradient"):
        fp8.linear(x.requires_grad_(), held)
    with pytest.raises(ValueError, match="no gradient"):
        fp8.linear(fp8.quantize_rows(x), w.requires_grad_())
    with pytest.raises(ValueError, match="matrix"):
        fp8.quantize_weight(torch.randn(3))
    data, scale = held.data, held.scale
    for bad in ((data.float(), scale), (data, scale[:, :1]), (data, scale.double()), (data[0], scale)):
        with pytest.raises(ValueError):
            fp8.Weight(*bad)
    with pytest.raises(ValueError):
        fp8.Rows(data, scale)
    y = fp8.linear(x, w)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, F32), (BF16, BF16), (F32, BF16)])
def test_add_rms_norm(kinds):
    torch.manual_seed(0)
    x, r, w = torch.randn(2, 5, 48).to(kinds[0]), torch.randn(2, 5, 48).to(kinds[1]), torch.randn(48)
    y, h = fused_ops.add_rms_norm(x, r, w, eps=1e-5)
    assert y.dtype == kinds[0] and h.dtype == torch.promote_types(*kinds)
    hd = h.double()
    want = hd * (hd.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w.double()
    assert ((y.double() - want).abs() <= (torch.finfo(y.dtype).eps / 2 + 60 * 2**-24) * want.abs()).all()
    rows, h2 = fp8.add_rms_norm(x, r, w, eps=1e-5)
    assert torch.equal(h, h2) and rows.data.shape == (10, 48)
    assert ((rows.dequantize().double() - want.view(10, 48)).abs() <= (2**-4 + 2**-18) * want.view(10, 48).abs() + 2**-10 * rows.scale).all()


def test_refusals_of_add_rms_norm():
    x, w = torch.randn(3, 16), torch.randn(16)
    for bad in ((x, x[:2], w), (x, x, w[:8]), (x[:, :0], x[:, :0], w[:0]), (x, None, w), (x.long(), x, w)):
        with pytest.raises(ValueError):
            fused_ops.add_rms_norm(*bad)
    with pytest.raises(ValueError, match="no gradient"):
        fp8.add_rms_norm(x, x.clone().requires_grad_(), w)
    with torch.no_grad():
        fp8.add_rms_norm(x, x.clone().requires_grad_(), w)


@pytest.mark.parametrize("scale", [1.0, 2.5])
@pytest.mark.parametrize("out", [None, BF16])
def test_embedding(scale, out):
    torch.manual_seed(0)
    table = torch.randn(11, 6, requires_grad=True)
    ids = torch.randint(0, 11, (4, 5))
    y = fused_ops.embedding(ids, table, scale=scale, out_dtype=out)
    assert torch.equal(y, (table[ids] * scale).to(out or F32))
    y.sum().backward()
    assert torch.allclose(table.grad, torch.bincount(ids.flatten(), minlength=11).float().unsqueeze(1).expand(11, 6) * scale)


def test_refusals_of_embedding():
    table, ids = torch.randn(11, 6), torch.tensor([1, 2])
    with pytest.raises(ValueError, match="matrix"):
        fused_ops.embedding(ids, table[0])
    with pytest.raises(ValueError, match="int64 or int32"):
        fused_ops.embedding(ids.float(), table)
    with pytest.raises(ValueError, match="floating"):
        fused_ops.embedding(ids, table, out_dtype=torch.int32)
    with pytest.raises(IndexError):
        fused_ops.embedding(torch.tensor([11]), table)


def test_llama_fp8_trains_and_evaluates():
    torch.manual_seed(0)
    model = Llama(LlamaConfig(vocab_size=50, n_layer=2, n_head=2, d_model=32, d_ffn=48, fp8=True, fused_embedding=True))
    idx = torch.randint(0, 50, (2, 9))
    model(idx[:, :-1], idx[:, 1:]).backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())
    model.eval()
    with torch.no_grad():
        logits = model(idx)
        model.hold_fp8_weights()
        assert torch.equal(model(idx), logits)
    model.train()
    assert all(layer._held is None for layer in model.layers)
    with pytest.raises(ValueError, match="fp8"):
        Llama(LlamaConfig(vocab_size=50, n_layer=1, n_head=2, d_model=32, d_ffn=48)).hold_fp8_weights()


def test_trainer_options():
    run = ["--steps", "2", "--batch-size", "2", "--seq-len", "16", "--small", "--device", "cpu"]
    assert train.main(["--model", "llama", "--fp8", "--fused-embedding", "--max-grad-norm", "1.0", "--optimizer", "gpa_adamw", *run]) > 0
    assert train.main(["--model", "gpt2", "--fused-embedding", "--optimizer", "adamw", *run]) > 0
    for bad in (["--model", "gpt2", "--fp8"], ["--model", "mlp", "--fused-embedding"]):
        with pytest.raises(SystemExit):
            train.main(bad + run)
