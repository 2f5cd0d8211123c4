"""The decoder's 8-bit operators on the CPU: derivatives that they do not have, modes, types."""

import pytest
import torch

from optimizers_b200.models import fp8, fused_ops

F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64


def test_forward_mode_derivatives_are_refused():
    x, w, t = torch.randn(4, 130), torch.randn(6, 130), torch.randn(4, 130)
    held, ones, learning = fp8.quantize_weight(w), torch.ones(130), w.clone().requires_grad_()
    calls = [
        lambda a: fp8.linear(a, w), lambda a: fp8.linear(a, learning), lambda a: fp8.linear(a, held), lambda a: fp8.linear(a, (w, held)),
        lambda a: fp8.linear(x, a[:, :130]), lambda a: fp8.linear(fp8.quantize_rows(x), a), lambda a: fp8.add_rms_norm(a, x, ones)[1], lambda a: fp8.add_rms_norm(x, a, ones)[1],
    ]
    for call in calls:
        with pytest.raises(ValueError, match="forward-mode"):
            torch.func.jvp(call, (x,), (t,))
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(x, t)
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                    call(dual)
            call(x.clone())  # the level alone changes nothing


def test_fp64_is_computed_in_64_bits():
    torch.manual_seed(0)
    x, r, w = (torch.randn(5, 48, dtype=F64), torch.randn(5, 48, dtype=F64), torch.randn(48, dtype=F64))
    y, h = fused_ops.add_rms_norm(x, r, w, eps=1e-5)
    assert y.dtype == h.dtype == F64 and torch.equal(h, x + r)
    want = h * (h.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w
    assert ((y - want).abs() <= 60 * 2**-53 * want.abs()).all()  # a mean of 48 squares, its root, two products
    assert torch.equal(fp8.add_rms_norm(x, r, w)[1], h) and torch.equal(fused_ops.add_rms_norm(x.float(), r, w)[1], x.float().double() + r)
    table, ids = torch.randn(11, 6, dtype=F64), torch.randint(0, 11, (20,))
    assert torch.equal(fused_ops.embedding(ids, table, scale=1 / 3), table[ids] * (1 / 3))


def test_status_words_made_in_inference_mode_serve_every_mode(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(fp8, "_status", {})
    with torch.inference_mode():
        status = fp8._status_of(torch.device("cpu"))
    assert not status.is_inference() and fp8._status_of(torch.device("cpu")) is status
    fp8.check_status()
    status.fill_(1)
    with pytest.raises(RuntimeError, match="gave up a wait"):
        fp8.check_status()
    fp8.check_status()


def test_second_derivatives_are_never_lost_silently():
    """dx depends on the weight and dW on x, also where what comes in is a constant: a sum of a gradient with other terms has to raise."""
    x, w = torch.randn(4, 130, requires_grad=True), torch.randn(6, 130, requires_grad=True)
    for leaf, other in ((x, w), (w, x)):
        (g,) = torch.autograd.grad(fp8.linear(x, w).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="again"):
            (g.square().sum() + other.sum()).backward()
    # where only one side learns its gradient is a constant
    (g,) = torch.autograd.grad(fp8.linear(x, w.detach()).sum(), x, create_graph=True)
    assert not g.requires_grad
    (g,) = torch.autograd.grad(fp8.linear(x, w.detach()).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="again"):
        g.sum().backward()
