"""The decoders' fused forms as modules: hooks, sharding of single blocks, weights kept in 8 bits."""

import pytest
import torch

from optimizers_b200.models import Llama, LlamaConfig


def _held_llama():
    torch.manual_seed(0)
    model = Llama(LlamaConfig(vocab_size=50, n_layer=2, n_head=2, d_model=32, d_ffn=48, fp8=True)).eval()
    model.hold_fp8_weights()
    return model


def _fresh(model):
    """The logits of a model of the same weights that keeps none of them in 8 bits."""
    other = Llama(model.cfg)
    other.load_state_dict(model.state_dict())
    return other.eval()(_IDX)


_IDX = torch.arange(18).view(2, 9)


@pytest.mark.parametrize("change", ["load", "assign", "in_place", "new_parameter", "data", "transposed", "moved", "gpa_step", "shampoo_step", "kernel"])
def test_kept_weights_follow_the_weights(change):
    from optimizers_b200 import AdaGradPreconditionerConfig, DistributedShampoo, GPAAdamW
    from optimizers_b200.utils import kept

    model = _held_llama()
    with torch.no_grad():
        before = model(_IDX)
        assert torch.equal(before, _fresh(model)) and all(len(layer._held) == 7 for layer in model.layers)
        source = Llama(model.cfg)
        wo = model.layers[1].wo
        if change == "load":
            model.load_state_dict(source.state_dict())
        elif change == "assign":
            model.load_state_dict(source.state_dict(), assign=True)
        elif change == "in_place":
            wo.weight.mul_(-1.0)
        elif change == "new_parameter":
            wo.weight = torch.nn.Parameter(-wo.weight)
        elif change == "data":
            wo.weight.data = -wo.weight.data
        elif change == "transposed":
            wo.weight.data = wo.weight.data.t()
        elif change == "moved":
            model.double().float()
            model.layers[0].wq.weight.add_(1.0)
        elif change == "kernel":  # as this package's kernels write: without PyTorch's count
            wo.weight.data.mul_(-1.0)
            kept.written([wo.weight])
        else:
            for p in model.parameters():
                p.grad = torch.randn_like(p)
            if change == "gpa_step":
                optimizer = GPAAdamW(model.parameters(), lr=0.1)
                optimizer.train()
                optimizer.step()
            else:
                DistributedShampoo(model.parameters(), lr=0.1, precondition_frequency=1, grafting_config=AdaGradPreconditionerConfig(epsilon=1e-8)).step()
        after = model(_IDX)
        assert not torch.equal(after, before)
        assert torch.equal(after, _fresh(model))
        model.hold_fp8_weights()
        assert torch.equal(model(_IDX), after) and all(len(layer._held) == 7 for layer in model.layers)


def test_copies_of_a_model_that_keeps_weights():
    import copy
    import io

    model = _held_llama()
    with torch.no_grad():
        want = model(_IDX)
        twin = copy.deepcopy(model)
        file = io.BytesIO()
        torch.save(model, file)
        file.seek(0)
        loaded = torch.load(file, weights_only=False)
        for other in (twin, loaded):
            assert torch.equal(other(_IDX), want)
            other.layers[0].wq.weight.data.neg_()
            assert torch.equal(other(_IDX), _fresh(other))
        assert torch.equal(model(_IDX), want)


def test_weights_that_cannot_be_kept_are_refused():
    with torch.inference_mode():
        model = Llama(LlamaConfig(vocab_size=50, n_layer=1, n_head=2, d_model=32, d_ffn=48, fp8=True)).eval()
        model(_IDX)
        with pytest.raises(ValueError, match="inference tensor"):
            model.hold_fp8_weights()
        assert getattr(model.layers[0], "_held", None) is None
    model = _held_llama()
    model.layers[0].wq.weight = torch.nn.Parameter(torch.zeros(5))  # as a shard of a flat parameter is
    with pytest.raises(ValueError, match="whole weights"):
        model.hold_fp8_weights()


def _sharded_hold_worker(rank, port):
    import torch.distributed as dist
    from torch.distributed.fsdp import fully_shard

    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=1)
    torch.manual_seed(0)
    model = fully_shard(Llama(LlamaConfig(vocab_size=50, n_layer=1, n_head=2, d_model=32, d_ffn=48, fp8=True)).eval())
    with torch.no_grad():
        model(_IDX)
    model.reshard()
    with pytest.raises(ValueError, match="whole weights"):
        model.hold_fp8_weights()
    dist.destroy_process_group()


def test_sharded_weights_are_not_kept():
    import socket

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    torch.multiprocessing.spawn(_sharded_hold_worker, args=(port,), nprocs=1, join=True)


def _small_llama(**kw):
    torch.manual_seed(0)
    cfg = dict(vocab_size=50, n_layer=2, n_head=2, d_model=32, d_ffn=48, fp8=True, fused_embedding=True)
    return Llama(LlamaConfig(**(cfg | kw)))


def test_hooks_of_blocks_norms_and_embeddings_run():
    from optimizers_b200.models import GPT2, GPT2Config

    model = _small_llama()
    seen = []
    watched = [model.embed, *model.layers, *(n for b in model.layers for n in (b.attn_norm, b.ffn_norm)), model.norm]
    for m in watched:
        m.register_forward_hook(lambda module, args, out: seen.append(module))
    idx = torch.randint(0, 50, (2, 9))
    model(idx[:, :-1], idx[:, 1:])
    assert len(seen) == len(watched) and all(any(m is s for s in seen) for m in watched)
    seen.clear()
    with torch.no_grad():
        model(idx)
    assert len(seen) == len(watched)
    gpt = GPT2(GPT2Config(vocab_size=50, n_ctx=16, n_layer=1, n_head=2, d_model=32, d_mlp=48, fused_embedding=True))
    seen.clear()
    gpt.wte.register_forward_hook(lambda module, args, out: seen.append(module))
    gpt(idx)
    assert seen == [gpt.wte]


def test_an_embedding_put_in_place_of_the_models_is_read():
    model = _small_llama()
    idx = torch.randint(0, 50, (2, 9))
    want = model(idx)
    table = model.embed.weight.detach().clone()
    model.embed = torch.nn.Embedding(50, 32, _weight=table)
    assert torch.equal(model(idx), want)


def _sharded_worker(rank, port):
    import torch.distributed as dist
    from torch.distributed.fsdp import fully_shard

    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
    idx = torch.randint(0, 50, (2, 9), generator=torch.Generator().manual_seed(1))
    whole = _small_llama()
    loss = whole(idx[:, :-1], idx[:, 1:])
    loss.backward()
    model = _small_llama()
    for part in (model.embed, *model.layers, model.norm):
        fully_shard(part)
    fully_shard(model)
    got = model(idx[:, :-1], idx[:, 1:])
    got.backward()
    assert torch.equal(got, loss)
    for (name, p), q in zip(model.named_parameters(), whole.parameters()):
        assert torch.allclose(p.grad.full_tensor(), q.grad, rtol=1e-6, atol=1e-9), name  # the mean of two equal gradients
    model.eval()
    whole.eval()
    with torch.no_grad():
        assert torch.equal(model(idx), whole(idx))
    dist.destroy_process_group()


def test_blocks_norm_and_embedding_sharded_on_their_own():
    import socket

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    torch.multiprocessing.spawn(_sharded_worker, args=(port,), nprocs=2, join=True)


def test_writes_to_the_memory_of_a_kept_weight_through_another_tensor():
    """Parameters that are pieces of one buffer, which an optimizer's kernel writes as a whole."""
    from optimizers_b200.utils import kept

    model = _held_llama()
    weight = model.layers[0].wq.weight
    flat = torch.nn.Parameter(torch.cat([torch.zeros(7), weight.detach().flatten()]))
    weight.data = flat.detach()[7:].view(32, 32)
    with torch.no_grad():
        model.hold_fp8_weights()
        before = model(_IDX)
        flat.data.neg_()
        kept.written([flat, model.embed.weight])
        assert not torch.equal(model(_IDX), before) and torch.equal(model(_IDX), _fresh(model))
        assert sum(len(layer._held) for layer in model.layers) == 13
