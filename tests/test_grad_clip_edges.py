"""Gradient clipping on the CPU: shared memory, other devices, ranks that hold other gradients."""

import math

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from optimizers_b200 import clip_grad_norm_, grad_norm


def _with_grads(*grads):
    params = [torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    return params


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_gradients_that_share_memory_are_refused(dtype):
    flat = torch.arange(1.0, 61.0).to(dtype)
    square = flat[:48].view(6, 8)
    for pair in (
        (flat[:20], flat[10:]), (flat, flat), (flat[:10], flat[9:10]), (square[:, :3], square[:, 2:5]), (square[::2], square[2:3]),
        (square.t()[1:3], square[:, 2]), (flat[0:40:3], flat[1:40:7]), (flat[::2], flat[40:44]), (flat.view(torch.uint8).view(dtype)[3:9], flat[8:12]),
    ):
        before = flat.clone()
        with pytest.raises(ValueError, match="share memory"):
            clip_grad_norm_(_with_grads(*pair), 1.0)
        assert torch.equal(flat, before)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_gradients_that_interleave_without_sharing_are_scaled_once(dtype):
    flat = torch.arange(1.0, 61.0).to(dtype)
    for parts in ((0, 2, 4), (1, 3, 5)):
        square = flat[:48].clone().view(6, 8)
        for grads in (
            [square[:, :2], square[:, 2:7], square[:, 7]], [square[::2], square[1::2]], [square.t()[: parts[0] + 1], square.t()[parts[0] + 1 :]],
            [square[:, parts[0]], square[:, parts[1]], square[:, parts[2]]], [square[:0], square[:3], square[3:]],
        ):
            before = [g.double().clone() for g in grads]
            true = math.sqrt(sum(float(g.square().sum()) for g in before))
            assert float(clip_grad_norm_(_with_grads(*grads), 1.0)) == pytest.approx(true, rel=1e-6)
            for g, b in zip(grads, before):
                assert torch.allclose(g.double(), b / (true + 1e-6), rtol=1e-6)
            for g, b in zip(grads, before):
                g.copy_(b)


def test_sharing_is_decided_as_by_listing_every_byte():
    import random

    from optimizers_b200 import grad_clip

    rng = random.Random(0)
    memory = torch.zeros(4000)
    halves = memory.view(torch.bfloat16)
    answers = set()
    for _ in range(400):
        views = []
        for _ in range(2):
            dims = rng.randint(1, 3)
            shape = [rng.randint(1, 5) for _ in range(dims)]
            stride = [rng.choice([0, 1, 2, 3, 5, 8, 13, 40]) for _ in range(dims)]
            views.append(rng.choice([memory, halves]).as_strided(shape, stride, rng.randint(0, 60)))
        cells = [
            {(v.storage_offset() + sum(i * s for i, s in zip(at, v.stride()))) * v.element_size() + byte for at in _indices(v.shape) for byte in range(v.element_size())}
            for v in views
        ]
        answers.add(bool(cells[0] & cells[1]))
        assert grad_clip._share_a_value(*views) == bool(cells[0] & cells[1])
    assert answers == {True, False}


def _indices(shape):
    import itertools

    return itertools.product(*(range(n) for n in shape))


class _OnAnotherGpu(torch.nn.Parameter):
    """A parameter that takes itself for one on a GPU without these kernels."""

    is_cuda = True


def test_other_gpus_do_without_the_extension(monkeypatch):
    from optimizers_b200 import grad_clip
    from optimizers_b200.ops import build

    def load():
        raise AssertionError("the extension was loaded")

    monkeypatch.setattr(build, "load", load)
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda device=None: (9, 0))
    monkeypatch.setattr(grad_clip, "_on_sm100", {}, raising=False)
    p = _OnAnotherGpu(torch.zeros(5))
    p.grad = torch.full((5,), 3.0)
    assert float(clip_grad_norm_([p], 1.0)) == pytest.approx(math.sqrt(45), rel=1e-6)
    assert p.grad.norm() == pytest.approx(1.0, rel=1e-5)
    assert float(grad_norm(p)) == pytest.approx(1.0, rel=1e-5)


def _uneven_worker(rank, port):
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
    p = torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))
    if rank == 0:
        p.grad = torch.full((4,), 3.0, dtype=torch.float64)
    # gradients of other types on other ranks, or none
    assert abs(float(clip_grad_norm_([p], 12.0, shard_group=dist.group.WORLD)) - 6.0) < 1e-6
    assert abs(float(grad_norm([p] if rank == 0 else [], shard_group=dist.group.WORLD)) - 6.0) < 1e-6
    if rank == 1:
        p = torch.nn.Parameter(torch.zeros(4))
        p.grad = torch.full((4,), 4.0)
    assert abs(float(grad_norm([p], shard_group=dist.group.WORLD)) - 10.0) < 1e-6
    # a norm that is refused is refused on every rank
    q = torch.nn.Parameter(torch.zeros(2))
    if rank == 0:
        q.grad = torch.tensor([1.0, math.inf])
    with pytest.raises(RuntimeError, match="norm of the gradients"):
        clip_grad_norm_([q], 1.0, shard_group=dist.group.WORLD, error_if_nonfinite=True)
    dist.destroy_process_group()


def test_ranks_with_other_gradients_or_none_agree():
    import socket

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_uneven_worker, args=(port,), nprocs=2, join=True)
