"""Gradient clipping on rank processes of a host-memory communicator."""
from __future__ import annotations


def run_clip(rank: int, world: int):
    import torch
    from originccl_b200 import init_from_env
    from originccl_b200.models import TinyLlamaStack
    from originccl_b200.ops import gradients
    from originccl_b200.parallel import DataParallelSync, GradBuckets

    comm = init_from_env(n_channels=2, timeout_ms=30000)
    model = TinyLlamaStack(hidden=32, ffn=96, layers=1, seed=3, vocab=50)
    dp = DataParallelSync(comm, GradBuckets(model.named_parameters(), bucket_bytes=4096, small_bytes=1024))
    g = torch.Generator().manual_seed(rank)
    model(torch.randint(0, 50, (8, 5), generator=g)).square().mean().backward()
    dp.sync()
    synced = [p.grad.clone() for p in model.parameters()]
    exact = sum(float(t.double().square().sum()) for t in synced) ** 0.5
    norm = float(dp.clip_grad_norm_(exact / 3))
    assert abs(norm - exact) <= exact * 2 ** -23
    for p, t in zip(model.parameters(), synced):  # the norm, the quotient and the product are rounded
        assert torch.allclose(p.grad, t / 3, rtol=1e-5 / exact + 2 ** -20, atol=0)
    # Shards: every rank holds other parameters, the norm is that of all of them.
    shard = torch.full((10,), float(rank + 1))
    total = float(gradients.clip_grad_norm([shard], 1e9, comm=comm))
    want = (10.0 * sum((r + 1) ** 2 for r in range(world))) ** 0.5
    assert abs(total - want) <= want * 2 ** -23 and torch.equal(shard, torch.full((10,), float(rank + 1)))
    assert abs(float(dp.clip_grad_norm_(1e9, shards=comm)) - world ** 0.5 * exact / 3) <= exact * 1e-4
    dp.close()
    comm.destroy()
    return {"norm": norm, "total": total}


def run_replicated(rank: int, world: int):
    """A matrix split by rows over the ranks beside a vector and a matrix that all hold: the norm is that of the
    model that is not split."""
    import pytest
    import torch
    from originccl_b200 import init_from_env
    from originccl_b200.ops import gradients
    from originccl_b200.parallel import DataParallelSync, GradBuckets

    comm = init_from_env(n_channels=2, timeout_ms=30000)
    alone = comm.split(color=rank, key=0)
    g = torch.Generator().manual_seed(5)
    split = torch.randn(6 * world, 8, generator=g)
    norm_weight, router = torch.randn(8, generator=g), torch.randn(40, 30, generator=g)
    whole = sum(float(t.double().square().sum()) for t in (split, norm_weight, router)) ** 0.5
    mine = split[6 * rank:6 * rank + 6]
    buckets = GradBuckets([("split", (6, 8)), ("norm", (8,)), ("router", (40, 30))], dtype=torch.float32, small_bytes=64)
    dp = DataParallelSync(alone, buckets)

    def fill():
        for view, t in zip(buckets.views, (mine, norm_weight, router)):
            view.copy_(t)
    fill()
    dp.sync()
    norm = dp.clip_grad_norm_(whole / 2, shards=comm, replicated=["norm", "router"])
    assert abs(float(norm) - whole) <= whole * 2 ** -23
    for view, t in zip(buckets.views, (mine, norm_weight, router)):  # the norm, the quotient and the product are rounded
        assert torch.allclose(view, t / 2, rtol=1e-5 / whole + 2 ** -20, atol=0)
    fill()
    flags = [False, True, True]
    assert float(gradients.grad_norm(buckets.views, comm=comm, replicated=flags)) == float(norm)
    # Nothing named: every parameter counts as a shard, once per rank.
    shares = sum(float(t.double().square().sum()) * (world if r else 1) for t, r in zip((split, norm_weight, router), flags))
    assert abs(float(gradients.grad_norm(buckets.views, comm=comm)) - shares ** 0.5) <= shares ** 0.5 * 2 ** -23
    # A rank that holds nothing but what the others hold too; one rank; no communicator.
    everywhere = float(gradients.grad_norm([norm_weight], comm=comm, replicated=[True]))
    assert abs(everywhere - float(norm_weight.double().norm())) <= everywhere * 2 ** -23
    for c in (alone, None):
        got = float(gradients.grad_norm(buckets.views, comm=c, replicated=flags))
        assert abs(got - sum(float(t.double().square().sum()) for t in buckets.views) ** 0.5) <= got * 2 ** -23
    with pytest.raises(ValueError, match="nobody"):
        dp.clip_grad_norm_(1.0, shards=comm, replicated=["norm", "nobody"])
    with pytest.raises(ValueError, match="truth values"):
        gradients.grad_norm(buckets.views, comm=comm, replicated=[True])
    dp.close()
    alone.destroy()
    comm.destroy()
    return float(norm)
