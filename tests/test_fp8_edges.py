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
