"""Copies of parameters in another form that a model keeps between calls, and whether they are still what the parameters hold.

A copy is good as long as its parameter is the same tensor in the same memory and counts no change since: PyTorch counts every operation that
writes in place, ``load_state_dict`` and the optimizers' steps among them.  This package's kernels write parameters
without that count, so the optimizers tell of it by ``written``.  What neither sees: writes through ``.data``, a raw pointer or a collective, and the
replay of a captured CUDA graph.
"""

from __future__ import annotations

import weakref
from collections.abc import Iterable
from typing import Any

from torch import Tensor
from torch.nn import Parameter

_alive: weakref.WeakSet[Kept] = weakref.WeakSet()


class Kept:
    """``value``, made from ``source`` as it is now."""

    def __init__(self, source: Tensor, value: Any) -> None:
        if source.is_inference():
            raise ValueError("an inference tensor does not count its changes, so no copy of it can be kept")
        self.source, self.value = source, value
        self.memory = source.detach()  # while it lives, no other tensor gets this memory
        self.place = (source.data_ptr(), source.stride())
        self.version = source._version
        _alive.add(self)

    def of(self, source: Tensor) -> bool:
        """Whether ``value`` is still what would be made from ``source``."""
        return source is self.source and source._version == self.version and (source.data_ptr(), source.stride()) == self.place

    def __reduce__(self):  # a copy of the model makes its own
        return _Expired, ()


class _Expired:
    value = None

    def of(self, source: Tensor) -> bool:
        return False


def any_alive() -> bool:
    return len(_alive) > 0


def written(parameters: Iterable[Tensor]) -> None:
    """A kernel has written these parameters, or other parts of the memory that they lie in."""
    storages = {p.untyped_storage().data_ptr() for p in parameters if type(p) in (Tensor, Parameter)}
    for kept in list(_alive):
        if kept.memory.untyped_storage().data_ptr() in storages:
            kept.version = -1
