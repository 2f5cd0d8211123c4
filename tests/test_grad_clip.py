"""Gradient clipping on the CPU: the formula, refusals, and shards over a process group."""

import math

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from optimizers_b200 import clip_grad_norm_, grad_norm
from optimizers_b200.examples import train


def _params(*shapes, dtype=torch.float32):
    torch.manual_seed(0)
    out = [torch.nn.Parameter(torch.zeros(s, dtype=dtype)) for s in shapes]
    for p in out:
        p.grad = torch.randn(p.shape).to(dtype)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("max_norm", [0.0, 0.3, 1e3, math.inf])
def test_formula(dtype, max_norm):
    params = _params((7, 5), (1,), (40,), dtype=dtype)
    before = [p.grad.double().clone() for p in params]
    true = math.sqrt(sum(float(g.square().sum()) for g in before))
    assert float(grad_norm(params)) == pytest.approx(true, rel=1e-6)
    assert float(clip_grad_norm_(iter(params), max_norm)) == pytest.approx(true, rel=1e-6)
    for p, g in zip(params, before):
        tol = max(torch.finfo(dtype).eps / 2 + 2**-23, 1e-12) + 2e-7
        assert ((p.grad.double() - g * min(1.0, max_norm / (true + 1e-6))).abs() <= tol * g.abs()).all()


def test_one_tensor_no_gradients_and_repeats():
    (p,) = _params((9,))
    want = float(p.grad.norm())
    assert float(clip_grad_norm_(p, 1.0)) == pytest.approx(want, rel=1e-6)
    assert float(clip_grad_norm_([p, p], 1e9)) == pytest.approx(1.0, rel=1e-5)
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.zeros(2))], 1.0)) == 0.0
    assert float(grad_norm([])) == 0.0


def test_refusals():
    (p,) = _params((4,))
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], bad)
    with pytest.raises(TypeError):
        clip_grad_norm_([3.0], 1.0)
    q = torch.nn.Parameter(torch.zeros(4, 3))
    q.grad = torch.ones(1, 3).expand(4, 3)
    with pytest.raises(ValueError, match="expanded"):
        clip_grad_norm_([q], 1.0)
    emb = torch.nn.Embedding(5, 3, sparse=True)
    emb(torch.tensor([1])).sum().backward()
    with pytest.raises(ValueError, match="dense"):
        clip_grad_norm_(emb.parameters(), 1.0)
    z = torch.nn.Parameter(torch.zeros(2, dtype=torch.complex64))
    z.grad = torch.ones(2, dtype=torch.complex64)
    with pytest.raises(ValueError, match="floating"):
        clip_grad_norm_([z], 1.0)
    p.grad[0] = math.inf
    before = p.grad.clone()
    with pytest.raises(RuntimeError, match="norm"):
        clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert torch.equal(p.grad, before)


def _shard_worker(rank, port):
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Replicate, Shard, distribute_tensor

    torch.manual_seed(0)
    whole = torch.randn(6, 4)
    true = float(whole.norm())
    p = torch.nn.Parameter(torch.zeros(3, 4))
    p.grad = whole[3 * rank : 3 * rank + 3].clone()
    assert abs(float(grad_norm([p], shard_group=dist.group.WORLD)) - true) < 1e-5
    assert abs(float(clip_grad_norm_([p], 1.0, shard_group=dist.group.WORLD)) - true) < 1e-5
    assert torch.allclose(p.grad, whole[3 * rank : 3 * rank + 3] / true, rtol=1e-5)
    # a rank without gradients still takes part
    q = torch.nn.Parameter(torch.zeros(6, 4))
    if rank == 0:
        q.grad = whole.clone()
    assert abs(float(clip_grad_norm_([q], 1.0, shard_group=dist.group.WORLD)) - true) < 1e-5
    # sharded and replicated DTensor gradients
    mesh = init_device_mesh("cpu", (2,))
    d = torch.nn.Parameter(distribute_tensor(torch.zeros(6, 4), mesh, [Shard(0)]))
    d.grad = distribute_tensor(whole, mesh, [Shard(0)])
    for bad in (dict(shard_group=None),):
        try:
            clip_grad_norm_([d], 1.0, **bad)
            raise AssertionError("a shard without its group was accepted")
        except ValueError:
            pass
    assert abs(float(clip_grad_norm_([d], 1.0, shard_group=mesh.get_group())) - true) < 1e-5
    assert torch.allclose(d.grad.full_tensor(), whole / true, rtol=1e-5)
    r = torch.nn.Parameter(distribute_tensor(torch.zeros(6, 4), mesh, [Replicate()]))
    r.grad = distribute_tensor(whole, mesh, [Replicate()])
    assert abs(float(grad_norm([r])) - true) < 1e-5
    dist.destroy_process_group()


def test_shards_over_a_group():
    import socket

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_shard_worker, args=(port,), nprocs=2, join=True)


def test_trainer_option_runs():
    loss = train.main(["--model", "mlp", "--optimizer", "sgd", "--max-grad-norm", "0.5", "--steps", "2", "--batch-size", "4", "--device", "cpu"])
    assert loss == loss
    with pytest.raises(SystemExit):
        train.main(["--model", "mlp", "--max-grad-norm", "-1", "--steps", "1", "--device", "cpu"])
    with pytest.raises(SystemExit):
        train.main(["--model", "mlp", "--max-grad-norm", "1", "--parallelism", "ddp_fused", "--steps", "1", "--device", "cpu"])
