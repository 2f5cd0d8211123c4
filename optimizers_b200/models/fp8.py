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
from torch.autograd import forward_ad

from optimizers_b200.models import fused_ops

GROUP = 128
_MOST = 448.0
_LEAST = 1e-30
_E4M3 = torch.float8_e4m3fn
_SOURCES = (torch.float32, torch.bfloat16)
_status: dict[torch.device, Tensor] = {}


def _groups(n: int) -> int:
    return -(-n // GROUP)


@dataclass(frozen=True, eq=False)
class Rows:
    """[T, K] e4m3 values and fp32 scales [T, ceil(K / 128)]."""

    data: Tensor
    scale: Tensor

    def __post_init__(self) -> None:
        _check_held(self.data, self.scale, self.data.shape[0] if self.data.dim() == 2 else -1)

    def dequantize(self) -> Tensor:
        return _values(self.data, self.scale, 1)


@dataclass(frozen=True, eq=False)
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
        if torch.cuda.is_current_stream_capturing():  # it would live in that graph's memory
            raise RuntimeError("call fp8.linear once on this device before capturing it into a CUDA graph")
        with torch.inference_mode(False):  # it serves the calls of every mode
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


def _squares(w: Tensor, native: bool) -> tuple[Tensor, Tensor]:
    if not native:
        return _plain_groups(w, GROUP)
    raw, _, scale = fused_ops._ext().fp8_squares(_source(w), False)
    fused_ops._count()
    return _e4m3(raw, w.shape[1]), scale


def _product(a, b, dtype: torch.dtype, native: bool, shape) -> Tensor:
    """``a @ b.T`` in ``dtype`` as a tensor of ``shape``, for rows a and a weight's squares b."""
    if not native:
        return _plain_product(a, b, GROUP, dtype).view(shape)
    out = fused_ops._ext().fp8_matmul(
        a[0].view(torch.uint8), a[1], b[0].view(torch.uint8), b[1], False, dtype == torch.bfloat16, None, _status_of(a[0].device), shape
    )
    fused_ops._count()
    return out


def _plain_product(a, b, down: int, dtype: torch.dtype) -> Tensor:
    with torch.autocast(a[0].device.type, enabled=False):
        return (_values(*a, 1) @ _values(*b, down).t()).to(dtype)


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
    return fused_ops._kernels_take(x) and x.numel() > 0


def _has_tangent(*tensors: Tensor) -> bool:
    """Whether a forward-mode derivative is being taken along one of these."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # none is being taken (the look below costs a microsecond a tensor)
        return False
    return any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _rows_of(data: Tensor, scale: Tensor) -> Rows:
    """Rows without the checks, for results of the kernels."""
    rows = object.__new__(Rows)
    object.__setattr__(rows, "data", data)
    object.__setattr__(rows, "scale", scale)
    return rows


def quantize_rows(x: Tensor) -> Rows:
    """``x`` [..., K] in 8 bits as [T, K], a scale per 128 columns of each row (no gradient)."""
    x2 = x.detach().reshape(-1, x.shape[-1])
    return Rows(*_rows(x2, _is_native(x2)))


def quantize_weight(weight: Tensor) -> Weight:
    """A linear layer's ``weight`` [N, K] in 8 bits, a scale per 128 x 128 square (no gradient)."""
    if weight.dim() != 2:
        raise ValueError(f"a weight is a matrix, got shape {tuple(weight.shape)}")
    w = weight.detach()
    return Weight(*_squares(w, _is_native(w)))


@torch.no_grad()
def _norm_rows(x: Tensor, residual: Tensor | None, weight: Tensor, eps: float) -> tuple[Rows, Tensor]:
    C = x.shape[-1]
    given = (x, weight) if residual is None else (x, weight, residual)
    if fused_ops._kernels_take(*given) and 0 < C <= fused_ops._MOST_COLUMNS and x.numel() > 0:
        if residual is not None and x.dtype == torch.float32 and residual.dtype == torch.bfloat16:
            residual = residual.float()  # an fp32 x is added to a residual in fp32
        raw, scale, h, _ = fused_ops._ext().add_norm_fwd(
            x.contiguous(), None if residual is None else residual.contiguous(), weight.contiguous(), eps, 2, False
        )
        fused_ops._count()
        return _rows_of(_e4m3(raw, C), scale.t()), (x if residual is None else h)
    h = x if residual is None else fused_ops._sum_of(x, residual)
    hf = h.float().reshape(-1, C)
    y = hf * torch.rsqrt(hf.pow(2).mean(-1, keepdim=True) + eps) * weight.float()
    return Rows(*_plain_groups(y, 1)), h


def add_rms_norm(x: Tensor, residual: Tensor | None, weight: Tensor, eps: float = 1e-6) -> tuple[Rows, Tensor]:
    """``fused_ops.add_rms_norm`` whose normalised rows come in 8 bits: ``(Rows [T, C], h)``.  The rows are rounded once, from 32 bits.
    No gradient: in training, ``fused_ops.add_rms_norm`` and ``linear`` on its result."""
    fused_ops._check_add_norm(x, residual, weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        raise ValueError("8-bit rows carry no gradient; use fused_ops.add_rms_norm in training, or torch.no_grad()")
    if _has_tangent(*(t for t in (x, residual, weight) if t is not None)):
        raise ValueError("8-bit rows carry no forward-mode derivative; use fused_ops.add_rms_norm")
    return _norm_rows(x, residual, weight, eps)


class _Once(torch.autograd.Function):
    """A gradient that raises an error where somebody differentiates it again."""

    @staticmethod
    def forward(ctx, grad: Tensor):  # type: ignore[override]
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, grad: Tensor):  # type: ignore[override]
        raise RuntimeError("this operator's gradient cannot be differentiated again")


class _Linear(torch.autograd.Function):
    """The plain form of the layer; the kernels' is a node of the extension."""

    @staticmethod
    def forward(ctx, x: Tensor, dtype: torch.dtype, *weights: Tensor):  # type: ignore[override]
        rows = _plain_groups(x, 1)
        squares = [_plain_groups(w, GROUP) for w in weights]
        ctx.save_for_backward(*_plain_groups(x.t(), 1), *(t for sq in squares for t in sq))
        ctx.meta = (x.dtype, [w.dtype for w in weights])
        ctx.set_materialize_grads(False)
        return tuple(_plain_product(rows, sq, GROUP, dtype) for sq in squares)

    @staticmethod
    def backward(ctx, *grads):  # type: ignore[override]
        learns = ctx.needs_input_grad
        # dx depends on the weights and dW on x, whether or not what comes in depends on a leaf
        again = torch.is_grad_enabled() and ((learns[0] and any(learns[2:])) or any(dy is not None and dy.requires_grad for dy in grads))
        with torch.no_grad():
            out = _Linear._gradients(ctx, grads)
        return tuple(None if g is None else _Once.apply(g.detach().requires_grad_()) if again else g for g in out)

    @staticmethod
    def _gradients(ctx, grads):
        x_dtype, w_dtypes = ctx.meta
        saved = ctx.saved_tensors
        dx, dws = None, [None] * len(w_dtypes)
        for i, dy in enumerate(grads):
            if dy is None:
                continue
            if ctx.needs_input_grad[0]:  # sums over several layers stay in 32 bits
                part = _plain_product(_plain_groups(dy, 1), (saved[2 + 2 * i].t(), saved[3 + 2 * i].t()), GROUP, torch.float32)
                dx = part if dx is None else dx + part
            if ctx.needs_input_grad[2 + i]:
                dws[i] = _plain_product(_plain_groups(dy.t(), 1), saved[:2], 1, w_dtypes[i])
        return (None if dx is None else dx.to(x_dtype), None, *dws)


def linear(x: Tensor | Rows, weight: Tensor | Weight | Sequence[Tensor | Weight], out_dtype: torch.dtype | None = None):
    """``x @ weight.T`` from 8-bit operands, for ``x`` [..., K] and ``weight`` [N, K]; a tuple of results for a sequence of weights.

    ``out_dtype``: fp32 or bf16; by default the autocast dtype, or x's (bf16 for ``Rows``).  Gradients flow to ``x`` and to weights that
    are tensors; a ``Weight`` or ``Rows`` takes no gradient, and combining one with an operand that needs one raises ``ValueError``.
    Forward-mode derivatives raise ``ValueError`` too.
    """
    several = not isinstance(weight, (Tensor, Weight))
    weights = tuple(weight) if several else (weight,)
    if not weights:
        raise ValueError("linear needs a weight")
    held_x = isinstance(x, Rows)
    source = x.data if held_x else x
    if source.dim() < 1 or source.shape[-1] == 0:
        raise ValueError(f"linear takes rows of at least one value, got shape {tuple(source.shape)}")
    tensors, empty = [], source.numel() == 0
    for w in weights:
        held = isinstance(w, Weight)
        data = w.data if held else w
        if data.dim() != 2 or data.shape[1] != source.shape[-1]:
            raise ValueError(f"a weight of shape {tuple(data.shape)} does not fit rows of shape {tuple(source.shape)}")
        if data.device != source.device:
            raise ValueError(f"weight on {data.device}, x on {source.device}")
        empty = empty or data.numel() == 0
        if not held:
            tensors.append(w)
    if out_dtype is None:
        out_dtype = torch.bfloat16 if held_x else fused_ops._compute_dtype(x)
    if not out_dtype.is_floating_point or (not held_x and not x.is_floating_point()):
        raise ValueError("linear takes and returns floating-point tensors")
    operands = tensors if held_x else [x, *tensors]
    native = not empty and out_dtype in _SOURCES and (fused_ops._kernels_take(*operands) if operands else fused_ops._native(source))
    learns = torch.is_grad_enabled() and any(t.requires_grad for t in operands)
    if learns and (held_x or len(tensors) < len(weights)):
        raise ValueError("operands held in 8 bits carry no gradient: pass tensors for x and every weight in training, or use torch.no_grad()")
    if _has_tangent(*operands):
        raise ValueError("linear has no forward-mode derivative: its operands are rounded to 8 bits")
    if native and not held_x and len(tensors) == len(weights):
        out = fused_ops._ext().fp8_linear(x, tensors, out_dtype == torch.bfloat16, _status_of(x.device))
    elif native and not held_x and not tensors:
        out = fused_ops._ext().fp8_linear_held(
            x, [_aligned(w.data) for w in weights], [w.scale for w in weights], out_dtype == torch.bfloat16, _status_of(x.device)
        )
    elif learns:
        out = _Linear.apply(x.reshape(-1, x.shape[-1]), out_dtype, *tensors)
        out = [y.view(*x.shape[:-1], y.shape[-1]) for y in out]
    else:
        rows = (x.data, x.scale) if held_x else _rows(x.detach().reshape(-1, x.shape[-1]), native)
        if native and held_x:
            rows = (_aligned(rows[0]), rows[1])
        out = []
        for w in weights:
            if isinstance(w, Weight):
                held = (_aligned(w.data) if native else w.data, w.scale)
            else:
                held = _squares(w.detach(), native)
            out.append(_product(rows, held, out_dtype, native, [*source.shape[:-1], held[0].shape[0]]))
    return tuple(out) if several else out[0]
