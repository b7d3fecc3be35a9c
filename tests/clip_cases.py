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
