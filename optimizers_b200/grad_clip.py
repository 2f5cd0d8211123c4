"""Norm over the gradients of a model, and their scaling below a bound, between ``backward()`` and ``step()``.

``norm = sqrt(sum of g^2)`` over every gradient; ``clip_grad_norm_`` then multiplies each gradient by
``min(1, max_norm / (norm + 1e-6))`` in place.  On a B200 both are two launches of this package's kernels
(``ops/csrc/clip_kernels.cu``) whatever the number of gradients, without a copy from the host: they run on the current
stream, can be captured into a CUDA graph, and add in a fixed order.  Elsewhere, and for gradients of other types, the same
formulas run in PyTorch.  Squares are summed in 32 bits (a gradient beyond 1.8e19 makes the norm infinite); bf16 and fp16
gradients are rounded once.

Gradients that are shards (``FullyShardedDataParallel``, ``fully_shard``) take ``shard_group``, the process group that one
whole gradient is spread over: the sum of squares is added up over it.  No reference counterpart.
"""

from __future__ import annotations

import math
from collections.abc import Iterable

import torch
import torch.distributed as dist
from torch import Tensor

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_on_sm100: dict[int | None, bool] = {}


def _sm100(device: torch.device) -> bool:
    known = _on_sm100.get(device.index)
    if known is None:
        known = _on_sm100[device.index] = torch.cuda.get_device_capability(device)[0] == 10
    return known


def _gradients(parameters: Tensor | Iterable[Tensor], shard_group) -> list[Tensor]:
    """The gradients of distinct parameters (a parameter listed twice counts once)."""
    seen: set[int] = set()
    grads = []
    for p in [parameters] if isinstance(parameters, Tensor) else parameters:
        if not isinstance(p, Tensor):
            raise TypeError(f"parameters are tensors, got {type(p).__name__}")
        g = p.grad
        if g is None or id(p) in seen:
            continue
        seen.add(id(p))
        if type(g) is not Tensor:
            g = _local_shard(g, shard_group)
        if g.layout != torch.strided:
            raise ValueError(f"gradients are dense tensors, got one of layout {g.layout}")
        if not g.is_floating_point():
            raise ValueError(f"gradients are real floating-point tensors, got one of dtype {g.dtype}")
        grads.append(g)
    return grads


def _local_shard(g: Tensor, shard_group) -> Tensor:
    from torch.distributed.tensor import DTensor, Replicate, Shard

    if not isinstance(g, DTensor):
        return g.detach() if isinstance(g, torch.nn.Parameter) else g
    shards = sum(isinstance(pl, Shard) for pl in g.placements)
    if shards + sum(isinstance(pl, Replicate) for pl in g.placements) != len(g.placements):
        raise ValueError(f"gradients are sharded or replicated, got placements {g.placements}")
    if shards > 1 or (shards == 1) != (shard_group is not None):
        raise ValueError(f"a gradient with placements {g.placements} needs the process group of its one sharded dimension as shard_group")
    return g.to_local()


def _native(grads: list[Tensor]) -> bool:
    d = grads[0].device
    return (
        d.type == "cuda"
        and all(type(g) is Tensor and g.device == d and g.dtype in _FLOATS for g in grads)
        and _sm100(d)
    )


def _sum_over_group(sumsq: Tensor, shard_group) -> Tensor:
    total = sumsq.sum().reshape(1).double()  # one type on every rank, whatever gradients it holds
    dist.all_reduce(total, group=shard_group)
    return total.to(sumsq.dtype)


def _plain_sumsq(grads: list[Tensor]) -> Tensor:
    first = grads[0].device
    sums = [g.detach().to(torch.promote_types(g.dtype, torch.float32)).square().sum().to(first) for g in grads]
    return torch.stack(sums).sum().reshape(1)


def _dense(g: Tensor) -> bool:
    """Whether the elements fill one stretch of memory, in any order of the dimensions."""
    expect = 1
    for st, n in sorted((st, n) for st, n in zip(g.stride(), g.shape) if n != 1):
        if st != expect:
            return False
        expect *= n
    return True


def _share_a_value(a: Tensor, b: Tensor) -> bool:
    """Whether some byte belongs to an element of each.  An element of ``a`` and one of ``b`` meet where the distance of the two starts is a sum of
    strides times differences of indices (a byte within an element counts as a last dimension of stride one): looked for from the
    largest stride down, among the multiples that the smaller strides can still make up for."""
    reach: dict[int, list[int]] = {}  # stride in bytes -> least and greatest multiple
    for t, low in ((a, False), (b, True)):
        size = t.element_size()
        for n, st in [*((n, st * size) for n, st in zip(t.shape, t.stride())), (size, 1)]:
            span = reach.setdefault(st, [0, 0])
            span[0 if low else 1] += (1 - n) if low else (n - 1)
    steps = [(st, lo, hi) for st, (lo, hi) in sorted(reach.items(), reverse=True) if st > 0 and lo < hi]
    below = [(0, 0)]  # what the steps behind each one can add up to
    for st, lo, hi in reversed(steps):
        below.append((below[-1][0] + st * lo, below[-1][1] + st * hi))
    below.reverse()
    tries = 100_000  # (layouts that take more do not come up; they count as shared)
    work = [(0, b.data_ptr() - a.data_ptr())]
    while work and tries > 0:
        k, left = work.pop()
        tries -= 1
        if k == len(steps):
            if left == 0:
                return True
            continue
        st, lo, hi = steps[k]
        least, most = below[k + 1]
        first, last = max(lo, -((most - left) // st)), min(hi, (left - least) // st)
        work.extend((k + 1, left - st * t) for t in range(first, min(last, first + tries) + 1))
    return bool(work)


def _check_disjoint(grads: list[Tensor]) -> None:
    """Raise ``ValueError`` for two gradients that share memory."""
    spans = []
    for g in grads:
        if type(g) is Tensor and g.numel() > 0 and g.device.type != "meta":
            reach = sum((n - 1) * st for n, st in zip(g.shape, g.stride())) + 1
            spans.append((str(g.device), g.data_ptr(), g.data_ptr() + reach * g.element_size(), g))
    spans.sort(key=lambda span: span[:3])
    open_spans: list = []
    for device, start, end, g in spans:
        open_spans = [o for o in open_spans if o[0] == device and o[2] > start]
        for o in open_spans:
            if _share_a_value(o[3], g):
                raise ValueError("clip: two gradients share memory; each value can be scaled once only")
        open_spans.append((device, start, end, g))


def _packed(grads: list[Tensor]) -> list[Tensor]:
    """The gradients, with copies in place of those that leave gaps in their memory."""
    return [g if g.is_contiguous() or _dense(g) else g.contiguous() for g in grads]


def _no_gradients(parameters, shard_group) -> Tensor:
    """The sum of squares where this rank holds no gradient (others may)."""
    device = next((p.device for p in ([parameters] if isinstance(parameters, Tensor) else parameters)), None)
    if device is None:
        device = torch.device("cuda" if shard_group is not None and dist.get_backend(shard_group) == "nccl" else "cpu")
    zero = torch.zeros(1, device=device)
    return _sum_over_group(zero, shard_group) if shard_group is not None else zero


def _refuse_nonfinite(sumsq: Tensor) -> None:
    value = float(sumsq.sum().sqrt())
    if not math.isfinite(value):
        raise RuntimeError(f"The norm of the gradients is {value}, so they cannot be clipped")


@torch.no_grad()
def grad_norm(parameters: Tensor | Iterable[Tensor], *, shard_group: dist.ProcessGroup | None = None) -> Tensor:
    """The 2-norm over the gradients of ``parameters``, as a 0-dim tensor (the host does not wait for it)."""
    parameters = parameters if isinstance(parameters, Tensor) else list(parameters)
    grads = _gradients(parameters, shard_group)
    if not grads:
        return _no_gradients(parameters, shard_group).sqrt()[0]
    native = _native(grads)
    return _sumsq(_packed(grads) if native else grads, shard_group, native, disjoint=False).sum().sqrt()


def _sumsq(grads: list[Tensor], shard_group, native: bool, disjoint: bool) -> Tensor:
    if native:
        from optimizers_b200.ops import build

        sumsq = build.load().grad_sumsq(grads, disjoint)
    else:
        sumsq = _plain_sumsq(grads)
    return sumsq if shard_group is None else _sum_over_group(sumsq, shard_group)


@torch.no_grad()
def clip_grad_norm_(
    parameters: Tensor | Iterable[Tensor],
    max_norm: float,
    *,
    error_if_nonfinite: bool = False,
    shard_group: dist.ProcessGroup | None = None,
) -> Tensor:
    """Scale the gradients of ``parameters`` in place so that their 2-norm is at most ``max_norm``; returns the norm before.

    ``error_if_nonfinite`` raises ``RuntimeError`` for a norm that is NaN or infinite, before any gradient changes (the host then
    waits for the norm).  Without it such a norm makes the gradients NaN (an infinite one: those that are infinite, and 0
    the others).  A parameter listed twice counts once; two gradients that share memory raise ``ValueError``.
    """
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError(f"Invalid max_norm: {max_norm}")
    parameters = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    if shard_group is None and not error_if_nonfinite and parameters and getattr(parameters[0], "is_cuda", False) and _sm100(parameters[0].device):
        from optimizers_b200.ops import build

        norm = build.load().clip_parameters(parameters, max_norm)
        if norm is not None:
            return norm
    grads = _gradients(parameters, shard_group)
    if not grads:
        sumsq = _no_gradients(parameters, shard_group)
        if error_if_nonfinite:  # on every rank of the group or on none
            _refuse_nonfinite(sumsq)
        return sumsq.sqrt()[0]
    for g in grads:
        if any(st == 0 and n > 1 for st, n in zip(g.stride(), g.shape)):
            raise ValueError("a gradient with an expanded dimension cannot be scaled in place")
    native = _native(grads)
    work = _packed(grads) if native else grads
    if not native or any(w is not g for w, g in zip(work, grads)):  # (the kernels' entry looks at what it is given, which are copies then)
        _check_disjoint(grads)
    sumsq = _sumsq(work, shard_group, native, disjoint=True)
    if error_if_nonfinite:
        _refuse_nonfinite(sumsq)
    if native:
        from optimizers_b200.ops import build

        norm = build.load().clip_scale(work, sumsq, max_norm)
        for g, w in zip(grads, work):
            if w is not g:
                g.copy_(w)
        return norm
    norm = sumsq.sum().sqrt()
    factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    for g in grads:
        g.copy_((g.to(torch.promote_types(g.dtype, torch.float32)) * factor.to(g.device)).to(g.dtype))
    return norm
