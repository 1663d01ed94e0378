"""GPU: routing with its losses where rows hold NaN or the type's lowest value, and against bounds of each element's own size.

Bounds, in units u = 2^-24 (half a step of f32), from the order in which the kernels compute:
  * an exponential of a difference d: d rounded once, its product with log2(e) once, log2(e) itself once, the base-2
    exponential to 4 u: EXP(d) = (3 |d| + 4) u.  One of a logit l (no difference): (2 |l| + 4) u;
  * a scaled sigmoid of l in a row with maximum m: for m >= 0 an exponential of -l, which is 1 - sigma of the sum it is added to, an
    addition and a reciprocal of 2 u; for m < 0 exponentials of l - m and of l, the latter sigma of its sum, an addition, a
    reciprocal and a product: (3 |l - m| + 2 |l| (1 - sigma or sigma) + 14) u holds for both;
  * a sum of positive terms over a row: at most 32 + 5 additions, and over K routes at most 4 + 5; a reciprocal 2 u, a product u;
  * a loss adds per lane at most 6 rows here, then 3 + 1 + 8 sums of a block, at most 296 slots over 32 warps of 4 or 8 of 1
    (37 + 8 + 2), the coefficient (4 roundings), 5 lanes, at most 32 tiles' parts a thread and 10 lanes and warps: 116 u;
  * lse: the maximum plus ln 2 times a base-2 logarithm of 2^-22 relative, or absolute below 1, and the rounding of that product and
    of ln 2: (6 (1 + lse - m) + |lse|) u on top of the relative error of the sum;
  * bf16 results: half a step more, 2^-8 of the value.
"""
import numpy as np
import pytest
import torch

from oracle import training_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 2.0 ** -120                                      # results below 2^-126 are flushed to zero, before a few products


def make(T, E, dtype, seed, spread=2.0):
    rng = np.random.default_rng(seed)
    return torch.from_numpy((rng.standard_normal((T, E)) * spread + rng.standard_normal(E)).astype(np.float32)).to(dtype)


def spans(l64, sigmoid):
    """|l - m| (softmax) or the terms of a scaled sigmoid's bound without its constant, per element, in units of 3 u."""
    m = l64.max(1, keepdim=True).values
    d = (l64 - m).abs()
    return d + l64.abs() * torch.where(m >= 0, torch.sigmoid(-l64), torch.sigmoid(l64)) * 2 / 3 if sigmoid else d


# ------------------------------------------------------------------------------------------------ rows that do not count
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,K", [(12, 3), (30, 8), (60, 5), (100, 8), (200, 8), (256, 20), (500, 6), (1000, 32)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_nan_in_rows_that_do_not_count_reaches_no_gradient(cuda_device, E, K, sigmoid, dtype):
    """With the gradient of the router weights: a route of weight 0 takes none, whatever its logit holds."""
    from mok import ops
    T = 100
    logits = make(T, E, dtype, E)
    mask = torch.ones(T, dtype=torch.bool)
    mask[10:30] = False
    offsets = torch.tensor([0, 50, 90], dtype=torch.int32, device=cuda_device)
    dirty = logits.clone()
    dirty[10:20] = np.nan
    dirty[20:25, K - 1:] = np.nan                       # one number too few for the routes
    dirty[25:30, 1:] = -np.inf
    dirty[92] = np.nan
    d = torch.tensor([0.7, 0.1], device=cuda_device)
    d_w = torch.randn(T, K, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    grads = []
    for l in (logits.to(cuda_device), dirty.to(cuda_device)):
        experts, weights, losses, _, coef = ops.router_topk_balance(l, K, mask.to(cuda_device), offsets, sigmoid)
        assert bool(torch.isfinite(weights).all()) and bool(torch.isfinite(losses).all())
        grads.append(ops.router_balance_bwd(d, l, coef, mask.to(cuda_device), offsets, experts, weights, d_w, sigmoid).cpu())
    clean, got = grads
    assert bool(torch.isfinite(got).all())
    assert bool((got[10:20] == 0).all()) and bool((got[92] == 0).all())
    keep = mask.clone()
    keep[92] = False
    assert torch.equal(got[keep], clean[keep])
    # a row with K - 1 numbers: the formula over those alone
    l64 = dirty[20:25, :K - 1].double().requires_grad_(True)
    chosen = O.select(l64.detach().numpy(), K - 1)
    w = O.weights(l64, chosen, sigmoid)
    dw = d_w[20:25, :K - 1].cpu().double()
    want, = torch.autograd.grad((w * dw).sum(), l64)
    scale = torch.zeros_like(want).scatter_(1, torch.from_numpy(chosen), (w * (dw.abs() + (w * dw).abs().sum(1, keepdim=True))).detach())
    assert bool((got[20:25, K - 1:] == 0).all())
    bound = 240 * U * scale + (want.abs() * 2.0 ** -8 if dtype == torch.bfloat16 else 0) + TINY
    assert bool(((got[20:25, :K - 1].double() - want).abs() <= bound).all())


def test_layer_gradients_with_nan_padding_rows(cuda_device):
    """The same through the autograd call a trainer makes."""
    from mok import functional as F
    x = make(64, 16, torch.float32, 3)
    x[40:] = np.nan
    mask = (torch.arange(64) < 40).to(cuda_device)
    x = x.to(cuda_device).requires_grad_(True)
    for score in ("softmax", "sigmoid"):
        _, weights, bal = F.route_balanced(x, 4, token_mask=mask, score=score)
        grad, = torch.autograd.grad((weights * torch.arange(4, device=cuda_device)).sum() + bal.losses.sum(), x)
        assert bool(torch.isfinite(grad).all()) and bool((grad[40:] == 0).all()) and bool((grad[:40] != 0).any(1).all())


# ------------------------------------------------------------------------------------------------ bounds of an element's size
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,K", [(8, 8), (32, 17), (64, 32), (128, 8), (256, 8), (300, 32), (1024, 32)])
def test_small_weights_are_as_exact_as_large_ones(cuda_device, E, K, dtype, sigmoid):
    """Weights from 1 to far below 1e-6, each within a bound relative to itself: its exponential, the sum's, 9 additions and the
    reciprocal and product."""
    from mok import ops
    logits = make(500, E, dtype, K, spread=9.0)
    logits[:20] -= 60.0
    logits[20:40] += 60.0
    experts, weights = ops.router_topk_balance(logits.to(cuda_device), K, None, None, sigmoid)[:2]
    chosen = O.select(logits.float().numpy(), K)
    assert np.array_equal(experts.cpu().numpy(), chosen)
    l64 = logits.double()
    want = O.weights(l64, chosen, sigmoid)
    span = spans(l64, sigmoid).gather(1, torch.from_numpy(chosen))
    bound = want * U * (3 * (span + (want * span).sum(1, keepdim=True)) + 2 * 14 + 9 + 3) + TINY
    assert float(want.min()) < 1e-6
    err = (weights.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,K,S,mask", [(1, 9, 3, 0, False), (512, 8, 2, 0, False), (1500, 24, 5, 0, True), (2000, 64, 4, 37, True),
                                          (5000, 256, 8, 3, False), (4097, 128, 8, 0, False), (1111, 1000, 3, 5, True),
                                          (3000, 500, 6, 61, False), (20000, 4, 1, 2, True), (300, 33, 2, 500, False)])
def test_losses_within_the_roundings_of_their_sums(cuda_device, T, E, K, S, mask, dtype, sigmoid):
    from mok import ops
    logits = make(T, E, dtype, T)
    rng = np.random.default_rng(S)
    where = {}
    if mask:
        where["token_mask"] = rng.random(T) < 0.8
    if S:
        where["sequence_offsets"] = np.sort(rng.integers(0, T + 1, S + 1)).astype(np.int32)
    chosen = O.select(logits.float().numpy(), K)
    l64 = logits.double()
    want = O.losses(l64, chosen, sigmoid=sigmoid, **where)
    rows = torch.from_numpy(np.concatenate(O.counted_rows(T, **where)))
    l = l64[rows]
    # p of every row: its exponential and the row sum's, each within the row's largest bound weighed by p; the sum's 37, 2 + 1
    p = O._scores(l, sigmoid)
    span = spans(l, sigmoid)
    rel_p = U * (3 * (span.max(1).values + (p * span).sum(1)) + 2 * 14 + 37 + 3)
    loss_bound = float(want[0]) * (float(rel_p.max()) + 116 * U) + TINY
    soft = torch.softmax(l, 1)
    lse = torch.logsumexp(l, 1)
    d = l.max(1, keepdim=True).values - l
    lse_err = U * (3 * (soft * d).sum(1) + 4 + 37 + 6 * (1 + lse - l.max(1).values) + lse.abs())
    z_bound = float((2 * lse.abs() * lse_err + lse_err ** 2).sum()) / max(1, len(rows)) + float(want[1]) * 116 * U + TINY
    x = logits.to(cuda_device)
    on = {k: torch.from_numpy(v).to(cuda_device) for k, v in where.items()}
    for losses in (ops.router_topk_balance(x, K, sigmoid=sigmoid, **on)[2],
                   ops.router_balance(x, torch.from_numpy(chosen.copy()).to(cuda_device), sigmoid=sigmoid, **on)[0]):
        err = (losses.cpu().double() - want).abs()
        assert float(err[0]) <= loss_bound and float(err[1]) <= z_bound, (float(err[0]) / loss_bound, float(err[1]) / z_bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E", [6, 60, 120, 300, 1000])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_gradients_of_rows_of_the_lowest_value(cuda_device, E, dtype, sigmoid):
    """A row whose every logit is the type's lowest value is uniform: its gradients, element by element.  In 64 bits the formulas
    need no shift; lse^2 is out of f32's range, so no z-loss is asked for.  Terms of an element as in its formula: two factors of
    its probability's bound (exponential or sigmoid, the row sum's, 37 + 3), a dot product of 37, 10 products; sigmoid scores
    another exponential of l, an addition and a reciprocal for 1 - sigma."""
    from mok import ops
    T, K = 40, 4
    logits = make(T, E, dtype, E)
    logits[7:12] = torch.finfo(dtype).min
    logits[20, 3:] = torch.finfo(dtype).min
    x = logits.to(cuda_device)
    experts, weights, _, counts, coef = ops.router_topk_balance(x, K, sigmoid=sigmoid)
    chosen = O.select(logits.float().numpy(), K)
    assert np.array_equal(experts.cpu().numpy(), chosen)
    d_w = torch.randn(T, K, generator=torch.Generator().manual_seed(E))
    got = ops.router_balance_bwd(torch.tensor([1.0, 0.0], device=cuda_device), x, coef, None, None, experts, weights,
                                 d_w.to(cuda_device), sigmoid).cpu().double()
    l64 = logits.double().requires_grad_(True)
    w = O.weights(l64, chosen, sigmoid)
    want, = torch.autograd.grad(O.losses(l64, chosen, sigmoid=sigmoid)[0] + (w * d_w.double()).sum(), l64)
    assert bool(torch.isfinite(want).all())
    with torch.no_grad():
        p = O._scores(l64, sigmoid)
        a = torch.from_numpy(O.expert_counts(chosen, E)[0] * E / (T * K) / T)
        scale = p * (a + (p * a).sum(1, keepdim=True))
        dw = d_w.double().abs()
        scale.scatter_add_(1, torch.from_numpy(chosen), w * (dw + (w * dw).sum(1, keepdim=True)))
        span = spans(l64, sigmoid)
        units = 2 * (3 * (span + (p * span).sum(1, keepdim=True)) + 2 * 14 + 40) + 37 + 10
        if sigmoid:
            units = units + 2 * l64.abs() * torch.sigmoid(l64) + 7
        bound = U * units * scale + (want.abs() * 2.0 ** -8 if dtype == torch.bfloat16 else 0) + TINY
    assert bool((bound[7:12] < want[7:12].abs() / 4).any(1).all())          # no gradient at all would be out of bounds
    err = (got - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


# ------------------------------------------------------------------------------------------------ the losses of a group
def test_layer_with_a_balance_group(cuda_device, single_rank_group):
    """One rank: the group's counts are its own, so outputs and losses are those without a group."""
    import mok
    F = mok.functional
    cfg = F.MoKConfig(minibatch_size=256, macrobatch_size=131072, schedule_capacity_multiplier=2.0, all_gather_top_experts_chunk_bytes=16)
    layers = [mok.nn.MoKLayer(512, 256, 8, 2, group=single_rank_group, config=cfg, device=cuda_device, seed=5, score="sigmoid",
                              balance_group=g) for g in (None, single_rank_group)]
    x = torch.randn(1024, 512, generator=torch.Generator().manual_seed(8)).bfloat16().to(cuda_device)
    mask = torch.arange(1024, device=cuda_device) % 5 != 0
    seen = []
    for layer in layers:
        out, bal = layer(x, return_balance=True, token_mask=mask)
        d_router, = torch.autograd.grad(bal.losses @ torch.tensor([1.0, 0.1], device=cuda_device), layer.router_weight)
        seen.append((out.detach(), bal.losses.detach(), bal.counts, d_router))
    for a, b in zip(*seen):
        assert torch.equal(a, b)
    off = torch.tensor([0, 1024], dtype=torch.int32, device=cuda_device)
    with pytest.raises(ValueError):
        layers[1](x, return_balance=True, sequence_offsets=off)
