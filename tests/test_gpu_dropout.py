"""GPU: dropout from the counter-based generator with the residual, against the 64-bit oracle; the layer's training step with
routing losses, residual and dropout together.

Tolerance of an element: the kernel rounds x * factor + residual at most twice in f32 (the factor is rounded once more) and once to
the type: 3 * 2^-24 of the terms' magnitude, and 2^-8 of the value for bf16."""
import numpy as np
import pytest
import torch

from oracle import training_oracle as O

pytestmark = pytest.mark.gpu


def seed_of(dev, value):
    return torch.tensor([value - (1 << 64) if value >= 1 << 63 else value], dtype=torch.int64, device=dev)


def check(got, x, residual, seed, p, first=0):
    want = O.dropout_add(x.cpu(), None if residual is None else residual.cpu(), seed, p, first)
    scale = x.cpu().double().abs() / max(1 - p, 2.0 ** -16) + (0 if residual is None else residual.cpu().double().abs())
    bound = 3 * 2.0 ** -24 * scale + (want.abs() * 2.0 ** -8 if x.dtype == torch.bfloat16 else 0) + 1e-38
    err = (got.cpu().double() - want).abs()
    assert got.dtype == x.dtype and bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5, 11), (512, 256), (1001, 1021), (40000, 257)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_against_the_oracle(cuda_device, shape, dtype, residual):
    from mok import ops
    gen = torch.Generator(device=cuda_device).manual_seed(len(shape))
    x = torch.randn(shape, generator=gen, device=cuda_device).to(dtype)
    r = torch.randn(shape, generator=gen, device=cuda_device).to(dtype) if residual else None
    for seed, p in ((1, 0.1), (0xFEDCBA9876543210, 0.5)):
        check(ops.dropout_add(x, r, seed_of(cuda_device, seed), p), x, r, seed, p)
        check(ops.dropout_add_bwd(x, seed_of(cuda_device, seed), p), x, None, seed, p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_extreme_rates(cuda_device, dtype):
    from mok import ops
    x, r = (torch.randn(999, device=cuda_device).to(dtype) for _ in range(2))
    s = seed_of(cuda_device, 3)
    assert torch.equal(ops.dropout_add(x, None, s, 0.0), x) and torch.equal(ops.dropout_add(x, r, s, 1), r)
    assert int(ops.dropout_add(x, None, s, 1.0).count_nonzero()) == 0
    assert torch.equal(ops.dropout_add(x, None, s, 2.0 ** -18), x)                      # rounds to 0
    check(ops.dropout_add(x, r, s, 1 - 2.0 ** -16), x, r, 3, 1 - 2.0 ** -16)
    check(ops.dropout_add(x, r, s, 2.0 ** -16), x, r, 3, 2.0 ** -16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_any_address(cuda_device, dtype):
    """x, residual and gradient on no common boundary."""
    from mok import ops
    base = [torch.randn(10007, device=cuda_device).to(dtype) for _ in range(2)]
    s = seed_of(cuda_device, 77)
    for a, b in ((0, 1), (1, 0), (3, 3), (8, 5), (16, 8)):
        x, r = base[0][a:a + 9000], base[1][b:b + 9000]
        assert torch.equal(ops.dropout_add(x, r, s, 0.2), ops.dropout_add(x.clone(), r.clone(), s, 0.2))
        assert torch.equal(ops.dropout_add_bwd(x, s, 0.2), ops.dropout_add_bwd(x.clone(), s, 0.2))


def test_dropped_elements_are_zero_whatever_they_hold(cuda_device):
    from mok import ops
    x = torch.full((4096,), float("nan"), device=cuda_device)
    x[1::2] = float("inf")
    keep, _ = O.dropout_keep(5, 0, 4096, 0.5)
    out = ops.dropout_add(x, None, seed_of(cuda_device, 5), 0.5).cpu()
    assert bool((out[torch.from_numpy(~keep)] == 0).all()) and not bool(torch.isfinite(out[torch.from_numpy(keep)]).any())


def test_elements_beyond_32_bits(cuda_device):
    from mok import ops
    n = (1 << 31) + 1003
    x = torch.ones(n, dtype=torch.bfloat16, device=cuda_device)
    out = ops.dropout_add(x, None, seed_of(cuda_device, 9), 0.25)
    for first in (0, (1 << 31) - 64, n - 99):
        check(out[first:first + 99], x[first:first + 99], None, 9, 0.25, first)
    assert abs(float((out == 0).sum()) / n - 0.25) < 1e-4


def test_refusals(cuda_device):
    from mok import ops
    x = torch.zeros(4, 6, device=cuda_device)
    s = seed_of(cuda_device, 1)
    for args in ((x.half(), None, s, 0.1), (x, None, s.int(), 0.1), (x, x.bfloat16(), s, 0.1)):
        with pytest.raises(TypeError):
            ops.dropout_add(*args)
    for args in ((x.t(), None, s, 0.1), (x, x.t(), s, 0.1), (x, x[:3], s, 0.1), (x, x.cpu(), s, 0.1), (x, None, s.cpu(), 0.1),
                 (x, None, torch.cat([s, s]), 0.1), (x, None, s, 1.1), (x, None, s, float("nan"))):
        with pytest.raises(ValueError):
            ops.dropout_add(*args)
    assert ops.dropout_add(torch.zeros(0, 4, device=cuda_device), None, s, 0.1).shape == (0, 4)


def test_gradients_and_seeds(cuda_device):
    """The gradient uses the forward's mask; seeds come from torch's generator, so activation checkpoints repeat them."""
    from mok import functional as F, ops
    x = torch.randn(300, 70, device=cuda_device, requires_grad=True)
    r = torch.randn(300, 70, device=cuda_device, requires_grad=True)
    g = torch.randn(300, 70, device=cuda_device)
    s = seed_of(cuda_device, 42)
    d_x, d_r = torch.autograd.grad(F.dropout_add(x, r, p=0.3, seed=s), (x, r), g)
    assert torch.equal(d_r, g) and torch.equal(d_x, ops.dropout_add_bwd(g, s, 0.3))
    check(d_x, g, None, 42, 0.3)
    d_x2, d_r2 = torch.autograd.grad(ops.dropout_add(x, r, s, 0.3), (x, r), g)
    assert torch.equal(d_x2, d_x) and torch.equal(d_r2, d_r)
    d_x3, = torch.autograd.grad(F.dropout_add(x, p=0.3, seed=s).sum(), x)                # an expanded gradient
    check(d_x3, torch.ones_like(g), None, 42, 0.3)
    d_r4, = torch.autograd.grad(F.dropout_add(x.detach(), r, p=0.3, seed=s), r, g)
    assert torch.equal(d_r4, g)
    # against differences: the map is linear in x for a fixed seed
    with torch.no_grad():
        moved = F.dropout_add(x + 0.5 * g, r, p=0.3, seed=s) - F.dropout_add(x, r, p=0.3, seed=s)
        assert abs(float((moved * g).sum()) - 0.5 * float((d_x * g).sum())) < 1e-3 * float((g * g).sum())
    torch.manual_seed(11)
    a = F.dropout_add(x, r, p=0.3)
    b = F.dropout_add(x, r, p=0.3)
    torch.manual_seed(11)
    assert torch.equal(F.dropout_add(x, r, p=0.3), a) and not torch.equal(a, b)
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(12)
    plain = torch.autograd.grad(F.dropout_add(torch.sin(x), r, p=0.4).square().sum(), x)[0]
    torch.manual_seed(12)
    again = torch.autograd.grad(checkpoint(lambda v: F.dropout_add(torch.sin(v), r, p=0.4), x, use_reentrant=False).square().sum(), x)[0]
    assert torch.equal(plain, again)


# ---------------------------------------------------------------------------------------------- together, in the layer
def layer_and_inputs(dev, group, **kwargs):
    import mok
    cfg = mok.functional.MoKConfig(minibatch_size=256, macrobatch_size=131072, schedule_capacity_multiplier=2.0,
                                   all_gather_top_experts_chunk_bytes=16)
    layer = mok.nn.MoKLayer(512, 256, 8, 2, group=group, config=cfg, device=dev, seed=5, **kwargs)
    gen = torch.Generator(device=dev).manual_seed(6)
    t = lambda: torch.randn(1024, 512, generator=gen, device=dev).bfloat16()             # noqa: E731
    return layer, t(), t(), t()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_training_step_is_the_composition_of_its_parts(cuda_device, single_rank_group, score):
    import mok
    F = mok.functional
    layer, x, residual, g = layer_and_inputs(cuda_device, single_rank_group, score=score, dropout=0.2)
    mask = torch.arange(1024, device=cuda_device) % 7 != 0
    off = torch.tensor([0, 300, 1000], dtype=torch.int32, device=cuda_device)
    x1, r1 = x.clone().requires_grad_(True), residual.clone().requires_grad_(True)
    torch.manual_seed(21)
    out, bal = layer(x1, residual=r1, return_balance=True, token_mask=mask, sequence_offsets=off)
    params = list(layer.parameters())
    loss = (out.float() * g.float()).sum() + bal.losses @ torch.tensor([50.0, 5.0], device=cuda_device)
    got = torch.autograd.grad(loss, [x1, r1, *params])
    # the parts, one by one
    x2, r2 = x.clone().requires_grad_(True), residual.clone().requires_grad_(True)
    logits = torch.nn.functional.linear(x2, layer.router_weight.to(x2.dtype)).float()
    if score == "softmax":
        experts, weights = F.route(logits, 2)
        p = torch.softmax(logits, 1)
    else:
        experts = O_select(logits, 2)
        p = torch.sigmoid(logits)
        weights = p.gather(1, experts)
        weights = weights / weights.sum(1, keepdim=True)
        p = p / p.sum(1, keepdim=True)
    ws = F.get_workspace(layer.config, single_rank_group, device=x.device, num_local_tokens=1024, hidden_size=512, topk=2)
    sched = F.build_schedule(ws, layer.config, experts, num_local_experts=8)
    y = mok.nn.moe_experts(layer.config, ws, sched, x2, weights, layer.shared_gate, layer.shared_up, layer.shared_down,
                           layer.routed_gate, layer.routed_up, layer.routed_down)
    torch.manual_seed(21)
    seed = torch.randint(0, 2 ** 63 - 1, (1,), dtype=torch.int64, device=cuda_device)
    keep, factor = O.dropout_keep(int(seed), 0, x.numel(), 0.2)
    keep = torch.from_numpy(keep).to(cuda_device).view(x.shape)
    out2 = (torch.where(keep, y.float() * factor, 0.0) + r2.float()).bfloat16()
    balance = z = 0.0
    n = 0
    for a, b in ((0, 300), (300, 1000)):
        rows = torch.arange(a, b, device=cuda_device)[mask[a:b]]
        c = torch.bincount(experts[rows].flatten(), minlength=8).float()
        balance = balance + (8 * c / c.sum() * p[rows].mean(0)).sum() / 2
        z = z + (torch.logsumexp(logits[rows], 1) ** 2).sum()
        n += len(rows)
    loss2 = (out2.float() * g.float()).sum() + 50.0 * balance + 5.0 * z / n
    want = torch.autograd.grad(loss2, [x2, r2, *params])
    assert (out.float() - out2.float()).abs().max() <= 2.0 ** -7 * out2.float().abs().max()
    assert abs(float(bal.balance.detach()) - float(balance.detach())) < 1e-4
    assert abs(float(bal.z.detach()) - float(z.detach()) / n) < 1e-4 * float(z.detach()) / n
    for a, b in zip(got, want):                             # bf16 gradients of the same kernels from inputs a rounding apart
        assert float((a.float() - b.float()).norm()) <= 1e-2 * float(b.float().norm())
    layer.eval()
    assert torch.equal(layer(x, residual=residual), layer(x) + residual)


def O_select(logits, K):
    return torch.from_numpy(O.select(logits.detach().cpu().numpy(), K).copy()).to(logits.device)


def test_layer_without_the_new_arguments_is_what_it_was(cuda_device, single_rank_group):
    layer, x, _, g = layer_and_inputs(cuda_device, single_rank_group)
    out = layer(x)
    withb, bal = layer(x, return_balance=True)
    assert torch.equal(out, withb) or float((out.detach().float() - withb.detach().float()).abs().max()) <= 2.0 ** -7 * float(out.detach().float().abs().max())
    assert int(bal.counts.sum()) == 1024 * 2 and tuple(bal.counts.shape) == (1, 8)


def test_captured_training_step_draws_new_masks_and_keeps_its_gradients(cuda_device, single_rank_group):
    """Forward, losses and gradients captured once: each replay uses the seed that torch's generator gives it."""
    layer, x, residual, g = layer_and_inputs(cuda_device, single_rank_group, dropout=0.3)
    params = list(layer.parameters())

    def step():
        out, bal = layer(x, residual=residual, return_balance=True)
        loss = (out.float() * g.float()).sum() + bal.losses.sum()
        return (out.detach(), bal.losses.detach(), bal.counts, *torch.autograd.grad(loss, params))
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    outs = []
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        outs.append([t.clone() for t in captured])
    assert not torch.equal(outs[0][0], outs[1][0])                                       # other masks
    assert torch.equal(outs[0][1], outs[1][1]) and torch.equal(outs[0][2], outs[1][2])   # the routing does not depend on them
    kept = [(o[0] != residual).float().mean() for o in outs]
    assert all(abs(float(k) - 0.7) < 0.02 for k in kept)
    assert all(torch.isfinite(t.float()).all() for o in outs for t in o)
