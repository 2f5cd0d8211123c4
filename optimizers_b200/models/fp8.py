"""Linear layers whose products take 8-bit operands with a scale per block of 128.

Format: e4m3 values with one fp32 scale per group.  For the largest magnitude ``a`` of a group (at least 1e-30) the scale is
``a / 448`` and a value x is held as ``e4m3(x * (448 / a))``.  Groups are runs of 128 along the dimension that a product sums
over (the last run may be shorter) for activations and gradients, and squares of 128 x 128 for weights.  A NaN or an infinity
makes every product that its group takes part in NaN.

``linear(x, weight)``
    ``x @ weight.T``.  In training all three products run in 8 bits: ``y = x W'``, ``dx = dy W`` and ``dW = dy' x``; x and dy are
    brought into both layouts by one pass each, the weight's squares serve W and its transpose.  Group sums are added in fp32,
    results are rounded once.  Several weights share one conversion of x: ``linear(x, (w_a, w_b))`` returns a tuple.
``Weight`` / ``quantize_weight(weight)``
    a weight that a program keeps in 8 bits (evaluation); taken in place of the tensor.
``Rows`` / ``quantize_rows(x)`` / ``add_rms_norm(x, residual, weight)``
    activations in 8 bits, the last straight from the residual addition and RMSNorm that precede a layer (no gradient).

On a B200 these are this package's kernels (``ops/csrc/fp8_kernels.cu``, ``ops/csrc/residual_norm.cu``) on the current stream; elsewhere,
and for other types, the same formulas run in PyTorch on the dequantised values.  ``check_status()`` raises if a product gave up a
wait inside its pipeline (its result is NaN then).  No reference counterpart.
"""

from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from optimizers_b200.models import fused_ops

GROUP = 128
_MOST = 448.0
_LEAST = 1e-30
_E4M3 = torch.float8_e4m3fn
_SOURCES = (torch.float32, torch.bfloat16)
_status: dict[torch.device, Tensor] = {}


def _groups(n: int) -> int:
    return -(-n // GROUP)


@dataclass(frozen=True)
class Rows:
    """[T, K] e4m3 values and fp32 scales [T, ceil(K / 128)]."""

    data: Tensor
    scale: Tensor

    def __post_init__(self) -> None:
        _check_held(self.data, self.scale, self.data.shape[0] if self.data.dim() == 2 else -1)

    def dequantize(self) -> Tensor:
        return _values(self.data, self.scale, 1)


@dataclass(frozen=True)
class Weight:
    """[N, K] e4m3 values and fp32 scales [ceil(N / 128), ceil(K / 128)] of a linear layer's weight."""

    data: Tensor
    scale: Tensor

    def __post_init__(self) -> None:
        _check_held(self.data, self.scale, _groups(self.data.shape[0]) if self.data.dim() == 2 else -1)

    def dequantize(self) -> Tensor:
        return _values(self.data, self.scale, GROUP)


def _check_held(data: Tensor, scale: Tensor, rows: int) -> None:
    if data.dim() != 2 or data.dtype != _E4M3:
        raise ValueError(f"values are a float8_e4m3fn matrix, got {data.dtype} of shape {tuple(data.shape)}")
    if scale.dtype != torch.float32 or scale.shape != (rows, _groups(data.shape[1])) or scale.device != data.device:
        raise ValueError(
            f"scales of {tuple(data.shape)} values are fp32 [{rows}, {_groups(data.shape[1])}] on {data.device}, "
            f"got {scale.dtype} {tuple(scale.shape)} on {scale.device}"
        )


def _values(data: Tensor, scale: Tensor, down: int) -> Tensor:
    full = scale if down == 1 else scale.repeat_interleave(down, 0)[: data.shape[0]]
    return data.float() * full.repeat_interleave(GROUP, 1)[:, : data.shape[1]]


def check_status() -> None:
    """Raise ``RuntimeError`` if a product of this process gave up a wait (one synchronisation per device)."""
    for device, status in _status.items():
        if int(status.item()):
            status.zero_()
            raise RuntimeError(f"an 8-bit product on {device} gave up a wait inside its pipeline; its result is NaN")


def _status_of(device: torch.device) -> Tensor:
    status = _status.get(device)
    if status is None:
        status = _status[device] = torch.zeros(1, dtype=torch.int32, device=device)
    return status


# --------------------------------------------------------------------------------------------------
# The steps, natively and plainly.  Operands are (values, scales) with scales [rows or row blocks, groups].
# --------------------------------------------------------------------------------------------------
def _plain_groups(x: Tensor, down: int) -> tuple[Tensor, Tensor]:
    rows, cols = x.shape
    p = torch.nn.functional.pad(x.float(), (0, -cols % GROUP, 0, -rows % down))
    blocks = p.view(p.shape[0] // down, down, p.shape[1] // GROUP, GROUP)
    top = blocks.abs().amax((1, 3)).clamp_min(_LEAST)
    most = torch.full_like(top, _MOST)  # (a number would be divided by as a product with its reciprocal)
    data = (blocks * (most / top)[:, None, :, None]).view_as(p).to(_E4M3)
    return data[:rows, :cols], top / most


def _e4m3(raw: Tensor, cols: int) -> Tensor:
    return raw.view(_E4M3)[:, :cols]


def _source(x: Tensor) -> Tensor:
    return x if x.shape[1] <= 1 or x.stride(1) == 1 else x.contiguous()


def _rows(x: Tensor, native: bool) -> tuple[Tensor, Tensor]:
    if not native:
        return _plain_groups(x, 1)
    raw, scale = fused_ops._ext().fp8_rows(_source(x))
    fused_ops._count()
    return _e4m3(raw, x.shape[1]), scale.t()


def _both(x: Tensor, native: bool) -> tuple[tuple[Tensor, Tensor], tuple[Tensor, Tensor]]:
    """x and its transpose, each in groups along its own rows."""
    if not native:
        return _plain_groups(x, 1), _plain_groups(x.t(), 1)
    raw, scale, raw_t, scale_t = fused_ops._ext().fp8_both(_source(x))
    fused_ops._count()
    return (_e4m3(raw, x.shape[1]), scale.t()), (_e4m3(raw_t, x.shape[0]), scale_t.t())


def _squares(w: Tensor, transpose: bool, native: bool) -> tuple[tuple[Tensor, Tensor], tuple[Tensor, Tensor] | None]:
    if not native:
        data, scale = _plain_groups(w, GROUP)
        return (data, scale), (data.t(), scale.t())
    raw, raw_t, scale = fused_ops._ext().fp8_squares(_source(w), transpose)
    fused_ops._count()
    return (_e4m3(raw, w.shape[1]), scale), (_e4m3(raw_t, w.shape[0]), scale.t()) if transpose else None


def _product(a, b, column_scales: bool, dtype: torch.dtype, native: bool, addend: Tensor | None = None) -> Tensor:
    """``a @ b.T`` (+ addend, fp32) in ``dtype``; b has a scale per row (``column_scales``) or per 128 rows."""
    if native:
        out = fused_ops._ext().fp8_matmul(
            a[0].view(torch.uint8), a[1], b[0].view(torch.uint8), b[1], column_scales, dtype == torch.bfloat16, addend, _status_of(a[0].device)
        )
        fused_ops._count()
        return out
    with torch.autocast(a[0].device.type, enabled=False):
        out = _values(*a, 1) @ _values(*b, 1 if column_scales else GROUP).t()
    return (out if addend is None else out + addend).to(dtype)


def _aligned(data: Tensor) -> Tensor:
    """Values whose rows start at multiples of 16 bytes, as the kernels read them."""
    if data.stride(1) == 1 and data.stride(0) % 16 == 0 and data.stride(0) >= data.shape[1] and data.data_ptr() % 16 == 0:
        return data
    rows, cols = data.shape
    raw = torch.empty(rows, (cols + 15) // 16 * 16, dtype=torch.uint8, device=data.device)
    raw[:, :cols] = data.view(torch.uint8)
    return raw.view(_E4M3)[:, :cols]


# --------------------------------------------------------------------------------------------------
# Public functions
# --------------------------------------------------------------------------------------------------
def _is_native(x: Tensor) -> bool:
    return fused_ops._native(x) and x.numel() > 0


def quantize_rows(x: Tensor) -> Rows:
    """``x`` [..., K] in 8 bits as [T, K], a scale per 128 columns of each row (no gradient)."""
    x2 = x.detach().reshape(-1, x.shape[-1])
    return Rows(*_rows(x2, _is_native(x2) and x2.dtype in _SOURCES))


def quantize_weight(weight: Tensor) -> Weight:
    """A linear layer's ``weight`` [N, K] in 8 bits, a scale per 128 x 128 square (no gradient)."""
    if weight.dim() != 2:
        raise ValueError(f"a weight is a matrix, got shape {tuple(weight.shape)}")
    w = weight.detach()
    return Weight(*_squares(w, False, _is_native(w) and w.dtype in _SOURCES)[0])


@torch.no_grad()
def _norm_rows(x: Tensor, residual: Tensor | None, weight: Tensor, eps: float) -> tuple[Rows, Tensor]:
    C = x.shape[-1]
    x2, r2 = fused_ops._norm_operands(x, residual)
    if fused_ops._add_norm_native(x2, r2, weight):
        raw, scale, h, _ = fused_ops._ext().add_norm_fwd(x2, r2, weight.contiguous(), eps, 2, False)
        fused_ops._count()
        return Rows(_e4m3(raw, C), scale.t()), (x if residual is None else h.view(x.shape))
    h = x if residual is None else (x.float() + residual.float()).to(torch.promote_types(x.dtype, residual.dtype))
    hf = h.float().reshape(-1, C)
    y = hf * torch.rsqrt(hf.pow(2).mean(-1, keepdim=True) + eps) * weight.float()
    return Rows(*_plain_groups(y, 1)), h


def add_rms_norm(x: Tensor, residual: Tensor | None, weight: Tensor, eps: float = 1e-6) -> tuple[Rows, Tensor]:
    """``fused_ops.add_rms_norm`` whose normalised rows come in 8 bits: ``(Rows [T, C], h)``.  The rows are rounded once, from 32 bits.
    No gradient: in training, ``fused_ops.add_rms_norm`` and ``linear`` on its result."""
    fused_ops._check_add_norm(x, residual, weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        raise ValueError("8-bit rows carry no gradient; use fused_ops.add_rms_norm in training, or torch.no_grad()")
    return _norm_rows(x, residual, weight, eps)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, dtype: torch.dtype, native: bool, *weights: Tensor):  # type: ignore[override]
        need_dx, need_dw = ctx.needs_input_grad[0], any(ctx.needs_input_grad[3:])
        rows, columns = _both(x, native) if need_dw else (_rows(x, native), None)
        saved, out = [], []
        for w in weights:
            straight, turned = _squares(w, need_dx, native)
            out.append(_product(rows, straight, False, dtype, native))
            saved += list(turned) if need_dx else []
        ctx.save_for_backward(*(columns or ()), *saved)
        ctx.meta = (need_dw, need_dx, native, x.shape, x.dtype, [(w.shape, w.dtype) for w in weights])
        ctx.set_materialize_grads(False)
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):  # type: ignore[override]
        need_dw, need_dx, native, x_shape, x_dtype, metas = ctx.meta
        saved = list(ctx.saved_tensors)
        columns = (saved.pop(0), saved.pop(0)) if need_dw else None
        live = [i for i, dy in enumerate(grads) if dy is not None]
        dx, dws = None, [None] * len(metas)
        for i in live:
            dy = grads[i]
            if dy.dtype not in _SOURCES:
                dy = dy.float()
            want_dw = ctx.needs_input_grad[3 + i]
            across, down = _both(dy, native) if want_dw else (_rows(dy, native) if need_dx else None, None)
            if need_dx:
                last = i == live[-1]  # sums over several layers stay in 32 bits until then
                dx = _product(across, (saved[2 * i], saved[2 * i + 1]), False, x_dtype if last else torch.float32, native, dx)
            if want_dw:
                dws[i] = _product(down, columns, True, metas[i][1], native)
        return (dx, None, None, *dws)


def linear(x: Tensor | Rows, weight: Tensor | Weight | Sequence[Tensor | Weight], out_dtype: torch.dtype | None = None):
    """``x @ weight.T`` from 8-bit operands, for ``x`` [..., K] and ``weight`` [N, K]; a tuple of results for a sequence of weights.

    ``out_dtype``: fp32 or bf16; by default the autocast dtype, or x's (bf16 for ``Rows``).  Gradients flow to ``x`` and to weights that
    are tensors; a ``Weight`` or ``Rows`` takes no gradient, and combining one with an operand that needs one raises ``ValueError``.
    """
    several = not isinstance(weight, (Tensor, Weight))
    weights = tuple(weight) if several else (weight,)
    if not weights:
        raise ValueError("linear needs a weight")
    held_x = isinstance(x, Rows)
    source = x.data if held_x else x
    for w in weights:
        shape = w.data.shape if isinstance(w, Weight) else w.shape
        if len(shape) != 2 or shape[1] != source.shape[-1]:
            raise ValueError(f"a weight of shape {tuple(shape)} does not fit rows of {source.shape[-1]}")
        if (w.data if isinstance(w, Weight) else w).device != source.device:
            raise ValueError(f"weight on {w.data.device}, x on {source.device}")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if held_x else fused_ops._compute_dtype(x)
    if not out_dtype.is_floating_point or (not held_x and not x.is_floating_point()):
        raise ValueError("linear takes and returns floating-point tensors")
    tensors = [w for w in weights if isinstance(w, Tensor)]
    learns = torch.is_grad_enabled() and (any(w.requires_grad for w in tensors) or (not held_x and x.requires_grad))
    empty = source.numel() == 0 or any((w.data if isinstance(w, Weight) else w).numel() == 0 for w in weights)
    native = (
        fused_ops._native(source) and not empty and out_dtype in _SOURCES and (held_x or x.dtype in _SOURCES)
        and all(w.dtype in _SOURCES for w in tensors)
    )
    if learns:
        if held_x or len(tensors) < len(weights):
            raise ValueError("operands held in 8 bits carry no gradient: pass tensors for x and every weight in training, or use torch.no_grad()")
        out = _Linear.apply(x.reshape(-1, x.shape[-1]), out_dtype, native, *weights)
        out = tuple(y.view(*x.shape[:-1], y.shape[-1]) for y in out)
    else:
        with torch.no_grad():
            rows = (x.data, x.scale) if held_x else _rows(x.reshape(-1, x.shape[-1]), native)
            if native and held_x:
                rows = (_aligned(rows[0]), rows[1])
            shape = x.data.shape[:1] if held_x else x.shape[:-1]
            out = []
            for w in weights:
                held = _squares(w, False, native)[0] if isinstance(w, Tensor) else (_aligned(w.data) if native else w.data, w.scale)
                out.append(_product(rows, held, False, out_dtype, native).view(*shape, held[0].shape[0]))
            out = tuple(out)
    return out if several else out[0]
