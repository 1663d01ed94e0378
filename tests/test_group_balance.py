"""CPU, world_size 2 over gloo: the host side of the losses over a group of ranks, with the operators' mathematics from the
oracle, and the order of checks and work."""
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

T, E, K = 96, 10, 3


def _batch():
    rng = np.random.default_rng(17)
    return torch.from_numpy(rng.standard_normal((2 * T, E)) * 2 + rng.standard_normal(E)), rng.random(2 * T) < 0.7


def _operators(ops, O):
    """Stands in for the two operators and the counts with the oracle's mathematics, differentiable by torch itself."""
    class Balance(torch.autograd.Function):
        @staticmethod
        def forward(ctx, logits, ids, mask, load, sigmoid):
            with torch.enable_grad():
                l = logits.detach().requires_grad_(True)
                out = O.losses(l, ids.numpy(), token_mask=mask.numpy(), load=None if load is None else load.numpy(), sigmoid=sigmoid)
            ctx.pair = l, out
            return out.detach()

        @staticmethod
        def backward(ctx, d):
            l, out = ctx.pair
            return torch.autograd.grad(out, l, d)[0], None, None, None, None

    def counts(ids, num_experts, mask=None, offsets=None):
        return torch.from_numpy(O.expert_counts(ids.numpy(), num_experts, None if mask is None else mask.numpy()))

    class Losses:
        @staticmethod
        def apply(logits, ids, mask, offsets, load, sigmoid):
            assert offsets is None
            return Balance.apply(logits, ids, mask, load, sigmoid), counts(ids, logits.shape[1], mask), None

    class Route:
        @staticmethod
        def apply(logits, topk, mask, offsets, sigmoid):
            ids = torch.from_numpy(O.select(logits.detach().numpy(), topk).copy())
            return ids, O.weights(logits, ids.numpy(), sigmoid), *Losses.apply(logits, ids, mask, offsets, None, sigmoid)
    ops.expert_counts = counts
    return Losses, Route


def _worker(rank, port, out):
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for p in (root, os.path.join(root, "mixture-of-kittens_b200")):
        sys.path.insert(0, p)
    from datetime import timedelta
    from oracle import training_oracle as O
    from mok import functional as F, ops
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2, timeout=timedelta(seconds=60))
    F._Balance, F._RouteBalanced = _operators(ops, O)
    logits, mask = _batch()
    mask[:T], mask[T:] = mask[:T], mask[:T][::-1]             # as many tokens that count on each rank
    ids = O.select(logits.numpy(), K)
    worst = 0.0
    for score in ("softmax", "sigmoid"):
        whole = logits.clone().requires_grad_(True)
        ref = O.losses(whole, ids, token_mask=mask, sigmoid=score == "sigmoid")
        ref_grad, = torch.autograd.grad(ref.sum(), whole)
        mine = slice(rank * T, (rank + 1) * T)
        x = logits[mine].clone().requires_grad_(True)
        local = torch.from_numpy(mask[mine].copy())
        experts, weights, bal = F.route_balanced(x, K, token_mask=local, score=score, group=dist.group.WORLD)
        finished = F.balance_loss(x, experts, token_mask=local, score=score, group=dist.group.WORLD)
        assert torch.equal(experts, torch.from_numpy(ids[mine].copy()))
        assert torch.equal(bal.counts, torch.from_numpy(O.expert_counts(ids[mine], E, mask[mine])))      # the rank's own
        assert torch.equal(bal.losses, finished.losses)
        grad, = torch.autograd.grad(bal.losses.sum(), x)
        mean = bal.losses.detach().clone()
        dist.all_reduce(mean)
        worst = max(worst, float((mean / 2 - ref.detach()).abs().max()), float((grad / 2 - ref_grad[mine]).abs().max()))
    seen = torch.tensor([worst], dtype=torch.float64)
    dist.all_reduce(seen, op=dist.ReduceOp.MAX)
    if rank == 0:
        open(out, "w").write(repr(float(seen)))
    dist.destroy_process_group()


def test_losses_over_two_ranks_are_those_of_the_whole_batch(tmp_path):
    """Averaged over ranks with as many tokens that count each: losses and gradients of the two ranks' batches as one.  64 bits
    throughout: sums of 2 T E terms below 30, 2000 roundings of 2^-53 at most."""
    out = str(tmp_path / "worst.txt")
    mp.spawn(_worker, args=(29537, out), nprocs=2)
    assert float(open(out).read()) <= 2000 * 2.0 ** -53 * 30


def test_a_group_with_sequences_is_refused_before_any_work(monkeypatch):
    """The refusal comes first: no launch, no count, no collective."""
    from mok import functional as F, ops
    stop = lambda *a, **k: pytest.fail("work before the refusal")                        # noqa: E731
    for name in ("router_topk_balance", "router_balance", "expert_counts"):
        monkeypatch.setattr(ops, name, stop)
    monkeypatch.setattr(F.dist, "all_reduce", stop)
    logits, offsets = torch.zeros(8, 4), torch.tensor([0, 8], dtype=torch.int32)
    with pytest.raises(ValueError, match="sequence_offsets"):
        F.route_balanced(logits, 2, sequence_offsets=offsets, group=object())
    with pytest.raises(ValueError, match="sequence_offsets"):
        F.balance_loss(logits, torch.zeros(8, 2, dtype=torch.int64), sequence_offsets=offsets, group=object())


def test_a_wrong_configuration_is_refused_before_any_work(monkeypatch):
    """As route_and_schedule does: nothing is routed and no count summed for a schedule that cannot be built."""
    import dataclasses
    from types import SimpleNamespace
    from mok import functional as F, ops
    stop = lambda *a, **k: pytest.fail("work before the refusal")                        # noqa: E731
    for name in ("router_topk_balance", "router_topk_gather", "router_balance", "expert_counts"):
        monkeypatch.setattr(ops, name, stop)
    monkeypatch.setattr(F, "_device_properties", lambda device: SimpleNamespace(multi_processor_count=148, shared_memory_per_block_optin=232448))
    fields = {f.name: None for f in dataclasses.fields(F.MoKWorkspace)}
    ws = F.MoKWorkspace(**{**fields, "device": torch.device("cpu"), "num_local_tokens": 512, "topk": 2, "ep_size": 1, "ep_rank": 0})
    logits = torch.zeros(512, 8)
    for route in (F.route_and_schedule, F.route_balanced_and_schedule):
        for config in (F.MoKConfig(fwd_num_comm_sms=3), F.MoKConfig(minibatch_size=100)):
            with pytest.raises(ValueError):
                route(ws, config, logits, num_local_experts=8)
        with pytest.raises(TypeError):
            route(ws, None, logits, num_local_experts=8)
