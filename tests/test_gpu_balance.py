"""GPU: balance and z-losses, per-expert counts and the router that gives them, against the 64-bit oracle.

Tolerances, in units u = 2^-24 (half a step of f32):
  * a softmax or sigmoid value: exp to 2 steps (4 u), its argument rounded to |difference| u, at most 40 u here, a sum of at
    most 1024 positive terms in at most 32 + 5 additions (37 u), a reciprocal and a product (3 u): under 90 u; two such
    factors, a dot product of the same length and the last products: 2 * 90 + 37 + 10 < 240 u of the terms' magnitude;
  * the losses add at most 1024 rows a warp-lane in turn plus 8 warps and 592 / 8 + 8 slots and 1024 tiles of sequences here:
    LOSS = 90 + 1200 u of the (positive) sum.  The z-loss squares lse, whose error is 90 u / sum + u |lse|: 3 * 90 u (|lse| + 1)^2;
  * bf16 results: half a step more, 2^-8 of the value.
"""
import numpy as np
import pytest
import torch

from oracle import training_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
GRAD, WEIGHT, LOSS = 240 * U, 180 * U, 1300 * U


def make(dev, T, E, K, *, dtype=torch.float32, S=0, mask=False, seed=0, spread=2.0):
    rng = np.random.default_rng(seed)
    logits = torch.from_numpy((rng.standard_normal((T, E)) * spread + rng.standard_normal(E)).astype(np.float32)).to(dtype)
    where = {}
    if mask:
        where["token_mask"] = torch.from_numpy(rng.random(T) < 0.8)
    if S:
        where["sequence_offsets"] = torch.from_numpy(np.sort(rng.integers(0, T + 1, S + 1)).astype(np.int32))
    return logits, where


def on(dev, where):
    return {k: v.to(dev) for k, v in where.items()}


def plain(where):
    return {k: v.numpy() for k, v in where.items()}


def check(dev, logits, K, where, sigmoid, *, experts=None, load=None, with_weights=True):
    """Forward and backward of one call; `experts` given: finished routes."""
    from mok import ops
    T, E = logits.shape
    rng = np.random.default_rng(7)
    x = logits.to(dev)
    score = dict(sigmoid=sigmoid)
    chosen = O.select(logits.float().numpy(), K) if experts is None else experts
    l64 = logits.double().requires_grad_(True)
    ref = O.losses(l64, chosen, load=load, **plain(where), **score)
    d_losses = torch.tensor([0.9, 0.02], dtype=torch.float32)
    total = (ref * d_losses.double()).sum()
    if experts is None:
        got_e, got_w, got_l, got_c, coef = ops.router_topk_balance(x, K, sigmoid=sigmoid, **on(dev, where))
        assert got_e.dtype == torch.int64 and np.array_equal(got_e.cpu().numpy(), chosen)
        ref_w = O.weights(l64, chosen, sigmoid)
        assert got_w.dtype == torch.float32 and (got_w.cpu().double() - ref_w).abs().max() <= WEIGHT
        routes = ()
        if with_weights:
            d_w = torch.from_numpy(rng.standard_normal((T, K)).astype(np.float32))
            total = total + (ref_w * d_w.double()).sum()
            routes = (got_e, got_w, d_w.to(dev))
    else:
        ids = torch.from_numpy(experts).to(dev)
        got_l, got_c, coef = ops.router_balance(x, ids, load=None if load is None else torch.from_numpy(load).to(dev),
                                                sigmoid=sigmoid, **on(dev, where))
        routes = ()
    assert got_c.dtype == torch.int32 and np.array_equal(got_c.cpu().numpy(), O.expert_counts(chosen, E, **plain(where)))
    rows = np.concatenate(O.counted_rows(T, **plain(where)))
    lse = torch.logsumexp(l64.detach()[torch.from_numpy(rows)], 1)
    lse = lse[lse != -np.inf]
    ref_l = ref.detach()
    got_l = got_l.cpu().double()
    assert abs(float(got_l[0] - ref_l[0])) <= LOSS * float(ref_l[0]) + 1e-30
    assert abs(float(got_l[1] - ref_l[1])) <= LOSS * float(ref_l[1]) + 270 * U * float(((lse.abs() + 1) ** 2).mean() if len(lse) else 0)
    got = ops.router_balance_bwd(d_losses.to(dev), x, coef, None if "token_mask" not in where else where["token_mask"].to(dev),
                                 None if "sequence_offsets" not in where else where["sequence_offsets"].to(dev),
                                 *(routes or (None, None, None)), sigmoid)
    assert got.dtype == logits.dtype
    grad = torch.autograd.grad(total, l64)[0] if total.requires_grad else torch.zeros(T, E, dtype=torch.float64)
    grad = torch.nan_to_num(grad, nan=0.0)              # rows without a finite logit: torch's 0 * (-inf - -inf)
    # magnitude of the terms of each element
    with torch.no_grad():
        scale = torch.zeros(T, E, dtype=torch.float64)
        counts = O.expert_counts(chosen, E, **plain(where)) if load is None else load
        parts = O.counted_rows(T, **plain(where))
        n, live = max(1, sum(map(len, parts))), max(1, sum(len(r) > 0 for r in parts))
        for s, r in enumerate(parts):
            if len(r):
                a = torch.from_numpy(counts[s] * E / max(1, counts[s].sum()) / len(r) / live)
                p, soft = O._scores(l64[r], sigmoid), torch.softmax(l64[r], 1)
                scale[r] += 0.9 * p * (a + (p * a).sum(1, keepdim=True)) + 0.02 * 2 / n * torch.logsumexp(l64[r], 1).abs()[:, None] * soft
                scale[r] += 0.02 * 2 / n * soft     # lse near 0 has an absolute error
        if routes:
            w, dw = ref_w, d_w.double().abs()
            scale.scatter_add_(1, torch.from_numpy(chosen), w * (dw + (w * dw).sum(1, keepdim=True)))
        scale = torch.nan_to_num(scale, nan=0.0)
    bound = GRAD * scale + (grad.abs() * 2.0 ** -8 if logits.dtype == torch.bfloat16 else 0) + 1e-38
    err = (got.cpu().double() - grad).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    return got


SHAPES = [(1, 1, 1), (1, 7, 3), (3, 8, 2), (17, 4, 4), (255, 16, 2), (513, 24, 5), (300, 33, 32), (1000, 64, 6), (777, 100, 7),
          (2049, 128, 8), (640, 255, 8), (511, 256, 9), (300, 500, 6), (130, 512, 31), (200, 1000, 8), (97, 1024, 32), (333, 256, 32),
          (200, 70, 20), (150, 128, 17), (90, 300, 16)]


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,K", SHAPES)
def test_routing_with_losses(cuda_device, T, E, K, dtype, sigmoid):
    logits, where = make(cuda_device, T, E, K, dtype=dtype, seed=T + E)
    check(cuda_device, logits, K, where, sigmoid)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T,E,K,S,mask", [(513, 24, 5, 1, False), (2000, 64, 4, 37, True), (900, 16, 2, 300, True), (40, 8, 2, 90, False),
                                          (5000, 256, 8, 3, False), (1111, 1000, 3, 5, True), (20000, 4, 1, 2, True)])
def test_routing_on_packed_sequences(cuda_device, T, E, K, S, mask, sigmoid):
    """Ragged and empty sequences, rows in front of, and behind them, masked rows."""
    logits, where = make(cuda_device, T, E, K, S=S, mask=mask, seed=S)
    check(cuda_device, logits, K, where, sigmoid)
    check(cuda_device, logits, K, where, sigmoid, with_weights=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,K,S,mask", [(1, 1, 1, 0, False), (600, 33, 5, 0, True), (3000, 128, 200, 7, True), (444, 1024, 2, 11, False)])
def test_losses_of_finished_routes(cuda_device, T, E, K, S, mask, dtype):
    """Ids outside [0, E), the same expert twice, more than 32 routes, and counts that ranks have added up."""
    logits, where = make(cuda_device, T, E, K, dtype=dtype, S=S, mask=mask, seed=K)
    rng = np.random.default_rng(5)
    experts = rng.integers(-2, E + 2, (T, K))
    experts[:, -1] = experts[:, 0]
    experts[0, 0] = 2 ** 40
    check(cuda_device, logits, K, where, False, experts=experts)
    load = rng.integers(0, 1000, (max(1, S), E)).astype(np.int32)
    check(cuda_device, logits, K, where, True, experts=experts, load=load)


@pytest.mark.parametrize("offsets", [[0, 0], [0, 5], [130, 137], [250, 256], [40, 200], [256, 256], [300, 900], [-7, 1 << 30]])
@pytest.mark.parametrize("E,K", [(5, 2), (30, 3), (200, 4), (600, 2)])
def test_one_sequence_inside_a_small_batch(cuda_device, E, K, offsets):
    """Blocks whose rows all lie outside the sequence add nothing; bounds are cut to the batch."""
    logits, _ = make(cuda_device, 256, E, K, seed=E)
    check(cuda_device, logits, K, {"sequence_offsets": torch.tensor(offsets, dtype=torch.int32)}, False)


@pytest.mark.parametrize("E", [8, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 512, 513, 1024])
def test_batches_around_the_sizes_where_the_kernels_change(cuda_device, E):
    at_once = 16 * (8 if E <= 16 else 4 if E <= 32 else 2 if E <= 64 else 1)
    for passes in (1, 2, 3, 6):
        for T in (8 * passes * at_once, 8 * passes * at_once + 1):
            logits, where = make(cuda_device, T, E, 3, seed=T, mask=True)
            check(cuda_device, logits, 3, where, T % 2 == 0)
            check(cuda_device, logits, 3, where, T % 2 == 0, experts=O.select(logits.numpy(), 3))


def test_many_rows_and_few_experts(cuda_device):
    logits, where = make(cuda_device, 70001, 8, 2, S=9, mask=True, seed=4)
    check(cuda_device, logits, 2, where, False)


def test_empty_rows_and_masked_experts(cuda_device):
    """Experts switched off with -inf or the lowest value, rows without a finite logit, equal logits."""
    logits, _ = make(cuda_device, 64, 20, 4, seed=1)
    logits[:, 5:9] = -np.inf
    logits[3] = -np.inf
    logits[4, 1:] = -np.inf                                 # one logit left for four routes
    logits[6] = 0.0                                         # ties: the lower expert first
    logits[7, ::2] = 1.5
    for sigmoid in (False, True):
        got = check(cuda_device, logits, 4, {}, sigmoid)
        assert bool((got[3] == 0).all()) and bool(torch.isfinite(got).all())
    from mok import ops
    low = torch.full((8, 6), torch.finfo(torch.float32).min, device=cuda_device)
    low[:, 2] = 1.0
    experts, weights, losses, _, coef = ops.router_topk_balance(low, 2)
    assert experts.tolist() == [[2, 0]] * 8 and weights.tolist() == [[1.0, 0.0]] * 8 and torch.isfinite(losses).all()
    assert torch.isfinite(ops.router_balance_bwd(torch.ones(2, device=cuda_device), low, coef)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E", [6, 60, 300])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_rows_of_the_lowest_value(cuda_device, E, dtype, sigmoid):
    """A row whose every logit is the type's lowest value is uniform, not empty; lse^2 overflows, so no z-loss is asked for."""
    from mok import ops
    T, K = 40, 4
    logits = make(cuda_device, T, E, K, dtype=dtype, seed=E)[0]
    logits[7:12] = torch.finfo(dtype).min
    logits[20, 3:] = torch.finfo(dtype).min
    x = logits.to(cuda_device)
    experts, weights, losses, counts, coef = ops.router_topk_balance(x, K, sigmoid=sigmoid)
    chosen = O.select(logits.float().numpy(), K)
    assert np.array_equal(experts.cpu().numpy(), chosen) and float(weights[7:12].sub(1 / K).abs().max()) < WEIGHT
    l64 = logits.double().requires_grad_(True)
    uniform = torch.zeros(T, E, dtype=torch.float64)        # the 64-bit oracle on rows shifted to zero: the same probabilities
    uniform[7:12] = -torch.finfo(dtype).min
    ref = O.losses(l64 + uniform if not sigmoid else torch.where(uniform != 0, l64 * 0, l64), chosen, sigmoid=sigmoid)[0]
    assert abs(float(losses[0]) - float(ref)) <= LOSS * float(ref)
    got = ops.router_balance_bwd(torch.tensor([1.0, 0.0], device=cuda_device), x, coef, None, None, experts, weights,
                                 torch.ones_like(weights), sigmoid)
    assert bool(torch.isfinite(got).all())
    if not sigmoid:
        grad, = torch.autograd.grad(ref, l64)
        a = O.expert_counts(chosen, E) * E / counts.sum().item() / T
        scale = 2 * torch.from_numpy(a).max() + 2.0 ** -20       # weights of a row add up to 1 within WEIGHT
        assert float((got.cpu().double() - grad).abs().max()) <= (GRAD + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) * float(scale) + WEIGHT


@pytest.mark.parametrize("E", [70, 128, 256, 600])
def test_many_routes_among_equal_and_missing_logits(cuda_device, E):
    """More than 16 routes with ties across the 16th, with just enough, and with too few logits above -inf."""
    K, T = 30, 24
    logits = make(cuda_device, T, E, K, seed=E)[0]
    logits[0:4] = torch.round(logits[0:4])
    logits[4] = 0.0
    for row, left in ((5, 30), (6, 29), (7, 17), (8, 16), (9, 15), (10, 1), (11, 0)):
        logits[row, torch.randperm(E, generator=torch.Generator().manual_seed(row))[left:]] = -np.inf
    for sigmoid in (False, True):
        check(cuda_device, logits, K, {}, sigmoid)


def test_far_below_zero_sigmoids_do_not_vanish(cuda_device):
    logits = torch.randn(200, 16, generator=torch.Generator().manual_seed(2)) * 3 - 150.0       # sigma underflows in f32
    check(cuda_device, logits, 3, {}, True)
    check(cuda_device, logits + 300.0, 3, {}, True)                                             # and saturates


def test_masked_rows_may_hold_anything(cuda_device):
    """NaN and infinities in rows that do not count reach neither the losses nor a gradient; in a row that counts they do."""
    from mok import ops
    logits, _ = make(cuda_device, 100, 12, 3, seed=9)
    mask = torch.ones(100, dtype=torch.bool)
    mask[10:20] = False
    offsets = torch.tensor([0, 50, 90], dtype=torch.int32)
    dirty = logits.clone()
    dirty[10:15], dirty[15:20], dirty[92] = np.nan, np.inf, -np.inf
    args = lambda l: (l.to(cuda_device), 3, mask.to(cuda_device), offsets.to(cuda_device))       # noqa: E731
    clean_out, dirty_out = ops.router_topk_balance(*args(logits)), ops.router_topk_balance(*args(dirty))
    assert torch.equal(clean_out[2], dirty_out[2]) and torch.equal(clean_out[3], dirty_out[3])
    keep = mask.clone()
    keep[92] = False
    assert torch.equal(clean_out[0][keep], dirty_out[0][keep]) and torch.equal(clean_out[1][keep], dirty_out[1][keep])
    d = torch.ones(2, device=cuda_device)
    grads = [ops.router_balance_bwd(d, a[0], o[4], a[2], a[3]) for a, o in ((args(logits), clean_out), (args(dirty), dirty_out))]
    assert torch.equal(*grads) and bool((grads[0][10:20] == 0).all()) and bool((grads[0][90:] == 0).all())
    dirty[30, 2] = np.nan
    assert bool(torch.isnan(ops.router_topk_balance(*args(dirty))[2]).all())
    none = ops.router_topk_balance(logits.to(cuda_device), 3, torch.zeros(100, dtype=torch.bool, device=cuda_device))
    assert none[2].tolist() == [0.0, 0.0] and int(none[3].sum()) == 0
    assert int(ops.router_balance_bwd(d, logits.to(cuda_device), none[4], torch.zeros(100, dtype=torch.bool, device=cuda_device))
               .count_nonzero()) == 0


def test_routes_are_those_of_the_plain_router(cuda_device):
    from mok import ops
    for T, E, K in ((512, 128, 8), (300, 1000, 32), (64, 5, 5)):
        logits = make(cuda_device, T, E, K, seed=E)[0].to(cuda_device)
        experts, weights = ops.router_topk(logits, K)
        got = ops.router_topk_balance(logits, K)
        assert torch.equal(got[0], experts) and (got[1] - weights).abs().max() < 2e-6


def test_logits_at_any_address(cuda_device):
    """Rows that start on no 16-byte boundary: an odd number of experts, and a view one element into its storage."""
    for dtype in (torch.float32, torch.bfloat16):
        for E in (64, 63, 65):
            base = torch.randn(300 * E + 1, generator=torch.Generator().manual_seed(E)).to(dtype)
            logits = base[1:].view(300, E)
            from mok import ops
            moved = base.to(cuda_device)[1:].view(300, E)
            assert moved.data_ptr() % 16
            a, b = ops.router_topk_balance(moved, 4), ops.router_topk_balance(logits.to(cuda_device).clone(), 4)
            assert all(torch.equal(x, y) for x, y in zip(a, b))
            d = torch.ones(2, device=cuda_device)
            routes = (a[0], a[1], torch.ones_like(a[1]))
            assert torch.equal(ops.router_balance_bwd(d, moved, a[4], None, None, *routes),
                               ops.router_balance_bwd(d, logits.to(cuda_device).clone(), b[4], None, None, *routes))


def test_offsets_beyond_32_bits(cuda_device):
    """More than 2^31 logits: the last rows are routed and get their gradient like any other."""
    from mok import ops
    T, E, K = (1 << 21) + 5, 1024, 2
    logits = torch.zeros(T, E, dtype=torch.bfloat16, device=cuda_device)
    tail = make(cuda_device, 50, E, K, dtype=torch.bfloat16, seed=8)[0]
    logits[-50:] = tail.to(cuda_device)
    offsets = torch.tensor([T - 50, T], dtype=torch.int32, device=cuda_device)
    experts, weights, losses, counts, coef = ops.router_topk_balance(logits, K, None, offsets)
    small = ops.router_topk_balance(tail.to(cuda_device), K)
    assert torch.equal(experts[-50:], small[0]) and torch.equal(weights[-50:], small[1]) and torch.equal(counts, small[3])
    assert experts[0].tolist() == [0, 1] and (losses - small[2]).abs().max() < 1e-4
    d = torch.tensor([1.0, 0.1], device=cuda_device)
    got = ops.router_balance_bwd(d, logits, coef, None, offsets)
    assert int(got[:-50].count_nonzero()) == 0
    want = ops.router_balance_bwd(d, tail.to(cuda_device), small[4])
    assert (got[-50:].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("T,E,K,S,mask", [(1, 1, 1, 0, False), (513, 4, 2, 0, True), (7777, 256, 8, 40, True), (3000, 1024, 3, 700, False),
                                          (100, 60, 255, 3, True), (962, 16, 8, 61, True), (50, 900, 4, 9, False), (40000, 300, 2, 500, True), (9000, 8, 3, 4000, False)])
def test_expert_counts(cuda_device, T, E, K, S, mask, dtype):
    from mok import ops
    _, where = make(cuda_device, T, 4, K, S=S, mask=mask, seed=T)
    experts = np.random.default_rng(1).integers(-3, E + 3, (T, K))
    got = ops.expert_counts(torch.from_numpy(experts).to(cuda_device, dtype), E, **on(cuda_device, where))
    assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), O.expert_counts(experts, E, **plain(where)))


@pytest.mark.parametrize("T,E,K", [(7, 5, 4), (130, 30, 17), (90, 64, 32), (33, 128, 9), (50, 700, 32)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_weight_gradients_of_an_expert_named_twice_add_up(cuda_device, T, E, K, sigmoid):
    """And ids outside [0, E) get none.  Bound: K additions and the terms' own roundings, 240 u of their magnitude."""
    from mok import ops
    rng = np.random.default_rng(K)
    experts = rng.integers(-1, max(2, E // 3), (T, K))
    logits = rng.standard_normal((T, E)).astype(np.float32)
    w, dw = rng.random((T, K)).astype(np.float32), rng.standard_normal((T, K)).astype(np.float32)
    w[0, 0] = 0.0
    d = lambda a: torch.from_numpy(a).to(cuda_device)                                    # noqa: E731
    args = (torch.zeros(2, device=cuda_device), d(logits), torch.zeros(E + 2, device=cuda_device), None, None, d(experts), d(w), d(dw), sigmoid)
    got = ops.router_balance_bwd(*args)
    assert torch.equal(got, ops.router_balance_bwd(*args))
    term = w.astype(np.float64) * (dw - (w.astype(np.float64) * dw).sum(1, keepdims=True))
    size = w.astype(np.float64) * (np.abs(dw) + np.abs(w.astype(np.float64) * dw).sum(1, keepdims=True))
    want, scale = np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        for k in range(K):
            e = experts[t, k]
            if e >= 0:
                f = 1 / (1 + np.exp(float(logits[t, e]))) if sigmoid else 1.0
                want[t, e] += term[t, k] * f
                scale[t, e] += size[t, k] * f
    assert (np.abs(got.cpu().numpy() - want) <= GRAD * scale).all()


def test_no_tokens(cuda_device):
    from mok import functional as F, ops
    logits = torch.zeros(0, 8, device=cuda_device)
    offsets = torch.zeros(4, dtype=torch.int32, device=cuda_device)
    experts, weights, losses, counts, coef = ops.router_topk_balance(logits, 2, None, offsets)
    assert experts.shape == weights.shape == (0, 2) and losses.tolist() == [0, 0] and counts.tolist() == [[0] * 8] * 3
    assert ops.router_balance_bwd(losses, logits, coef, None, offsets).shape == (0, 8)
    assert F.expert_counts(experts, 8).tolist() == [[0] * 8]
    assert F.balance_loss(logits, experts).losses.tolist() == [0, 0]


def test_refusals(cuda_device):
    from mok import ops
    x = torch.zeros(8, 6, device=cuda_device)
    ids = torch.zeros(8, 2, dtype=torch.int64, device=cuda_device)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda_device)              # noqa: E731
    mask = torch.ones(8, dtype=torch.bool, device=cuda_device)
    for bad in (x.half(), x.double()):
        with pytest.raises(TypeError):
            ops.router_topk_balance(bad, 2)
    with pytest.raises(TypeError):
        ops.router_balance(x, ids.int())
    with pytest.raises(TypeError):
        ops.expert_counts(ids.short(), 6)
    for call in (lambda: ops.router_topk_balance(x.t(), 2), lambda: ops.router_topk_balance(x, 0), lambda: ops.router_topk_balance(x, 7),
                 lambda: ops.router_topk_balance(torch.zeros(2, 1025, device=cuda_device), 2), lambda: ops.router_topk_balance(x[0], 1),
                 lambda: ops.router_topk_balance(torch.zeros(8, 64, device=cuda_device), 33),
                 lambda: ops.router_topk_balance(x, 2, mask[:7]), lambda: ops.router_topk_balance(x, 2, mask.int()),
                 lambda: ops.router_topk_balance(x, 2, mask.cpu()), lambda: ops.router_topk_balance(x, 2, None, i32(1)),
                 lambda: ops.router_topk_balance(x, 2, None, i32(2).long()), lambda: ops.router_topk_balance(x, 2, None, i32(2, 2)),
                 lambda: ops.router_balance(x, ids[:7]), lambda: ops.router_balance(x, ids.t()), lambda: ops.router_balance(x, ids.cpu()),
                 lambda: ops.router_balance(x, ids, None, None, i32(6)), lambda: ops.router_balance(x, ids, None, i32(4), i32(1, 6)),
                 lambda: ops.expert_counts(ids, 0), lambda: ops.expert_counts(ids, 1025), lambda: ops.expert_counts(ids[0], 6)):
        with pytest.raises(ValueError):
            call()
    g, coef = torch.ones(2, device=cuda_device), torch.ones(8, device=cuda_device)
    w = torch.ones(8, 2, device=cuda_device)
    for args in ((g[:1], x, coef), (g, x, coef[:7]), (g, x, coef, None, i32(3)), (g, x, coef, None, None, ids, w),
                 (g, x, coef, None, None, ids.repeat(1, 4), w.repeat(1, 4), w.repeat(1, 4)), (g, x, coef, None, None, ids, w, w[:, :1]), (g, x, coef, None, None, ids[:4], w, w), (g.cpu(), x, coef)):
        with pytest.raises(ValueError):
            ops.router_balance_bwd(*args)
    with pytest.raises(TypeError):
        ops.router_balance_bwd(g.double(), x, coef)


def test_gradients_through_the_functional_calls(cuda_device):
    """The autograd functions and the operators' own formulas give the bytes of the explicit calls; unused outputs cost nothing."""
    from mok import functional as F, ops
    logits, where = make(cuda_device, 600, 40, 4, S=5, mask=True, seed=12)
    where = on(cuda_device, where)
    mask, off = where["token_mask"], where["sequence_offsets"]
    x = logits.to(cuda_device).requires_grad_(True)
    d_w = torch.randn(600, 4, device=cuda_device)
    d_l = torch.tensor([0.3, 0.01], device=cuda_device)
    for score in ("softmax", "sigmoid"):
        experts, weights, bal = F.route_balanced(x, 4, score=score, **where)
        e, w, losses, counts, coef = ops.router_topk_balance(x.detach(), 4, mask, off, score == "sigmoid")
        assert torch.equal(experts, e) and torch.equal(weights, w) and torch.equal(bal.losses, losses) and torch.equal(bal.counts, counts)
        want = ops.router_balance_bwd(d_l, x.detach(), coef, mask, off, e, w, d_w, score == "sigmoid")
        got, = torch.autograd.grad([weights, bal.losses], x, [d_w, d_l])
        assert torch.equal(got, want)
        through_op = ops.router_topk_balance(x, 4, mask, off, score == "sigmoid")
        got, = torch.autograd.grad([through_op[1], through_op[2]], x, [d_w, d_l])
        assert torch.equal(got, want)
        experts, weights, bal = F.route_balanced(x, 4, score=score, **where)
        got, = torch.autograd.grad(0.3 * bal.balance + 0.01 * bal.z, x)                 # weights unused
        only = ops.router_balance_bwd(d_l, x.detach(), coef, mask, off, None, None, None, score == "sigmoid")
        assert torch.equal(got, only)
        finished = F.balance_loss(x, e, score=score, **where)
        assert torch.equal(finished.losses, losses)
        assert torch.equal(torch.autograd.grad(finished.losses, x, d_l)[0], only)
        assert torch.equal(torch.autograd.grad(ops.router_balance(x, e, mask, off, None, score == "sigmoid")[0], x, d_l)[0], only)
    experts, weights, _ = F.route_balanced(x, 4)                                         # losses unused
    got, = torch.autograd.grad(weights, x, d_w)
    assert (got - ops.router_topk_bwd(experts, weights.detach(), d_w, 40)).abs().max() < 1e-6
    y = x.detach().clone()
    y[5] = np.nan                                                                        # and then not read for them
    y.requires_grad_(True)
    got, = torch.autograd.grad(F.route_balanced(y, 4)[1][:5], y, d_w[:5])
    assert torch.isfinite(got[:5]).all() and bool((got[6:] == 0).all())


def test_finished_counts_of_two_ranks_give_the_global_loss(cuda_device):
    """Averaged over ranks, the loss with the summed counts is the loss of the whole batch."""
    from mok import ops
    logits = make(cuda_device, 800, 16, 2, seed=3)[0].to(cuda_device)
    experts = ops.router_topk(logits, 2)[0]
    whole, counts, _ = ops.router_balance(logits, experts)
    halves = [(logits[a:a + 400], experts[a:a + 400]) for a in (0, 400)]
    load = sum(ops.expert_counts(e, 16) for _, e in halves)
    assert torch.equal(load, counts)
    parts = [ops.router_balance(l, e, None, None, load)[0] for l, e in halves]
    assert (sum(parts) / 2 - whole).abs().max() <= 2 * LOSS * float(whole.max())


def test_group_of_one_rank(cuda_device, single_rank_group):
    from mok import functional as F
    x = make(cuda_device, 300, 24, 3, seed=3)[0].to(cuda_device).requires_grad_(True)
    a, b = F.route_balanced(x, 3), F.route_balanced(x, 3, group=single_rank_group)
    assert torch.equal(a[2].losses, b[2].losses) and torch.equal(a[2].counts, b[2].counts)
    grads = [torch.autograd.grad([r[1].square().sum(), r[2].balance], x)[0] for r in (a, b)]
    assert (grads[0] - grads[1]).abs().max() <= GRAD * 4


def test_runs_and_streams_give_the_same_bytes(cuda_device):
    from mok import ops
    logits, where = make(cuda_device, 30000, 200, 6, S=11, mask=True, seed=2)
    x, where = logits.to(cuda_device), on(cuda_device, where)
    args = (x, 6, where["token_mask"], where["sequence_offsets"])
    first = ops.router_topk_balance(*args)
    d = torch.ones(2, device=cuda_device)
    grad = ops.router_balance_bwd(d, x, first[4], *args[2:])
    streams = [torch.cuda.Stream(cuda_device) for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:                                       # three calls in flight at once
        with torch.cuda.stream(s):
            for _ in range(4):
                out = ops.router_topk_balance(*args)
                outs.append((out, ops.router_balance_bwd(d, x, out[4], *args[2:])))
    torch.cuda.synchronize()
    for out, g in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, first)) and torch.equal(g, grad)


def test_two_captured_graphs_share_nothing(cuda_device):
    from mok import ops
    x = [make(cuda_device, 2000, 64, 4, seed=s)[0].to(cuda_device) for s in (1, 2)]
    off = torch.tensor([0, 700, 1900], dtype=torch.int32, device=cuda_device)
    d = torch.ones(2, device=cuda_device)

    def step(l):
        out = ops.router_topk_balance(l, 4, None, off)
        return (*out, ops.router_balance_bwd(d, l, out[4], None, off, out[0], out[1], torch.ones_like(out[1])), ops.expert_counts(out[0], 64, None, off))
    want = [[t.clone() for t in step(l)] for l in x]
    side = torch.cuda.Stream(cuda_device)
    with torch.cuda.stream(side):
        step(x[0])
    torch.cuda.synchronize()
    graphs, got = [], []
    for l in x:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(step(l))
        graphs.append(g)
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_compiled_and_threaded_calls(cuda_device):
    """Traced whole by torch.compile, and called by several host threads at once on streams of their own."""
    import threading
    from mok import functional as F, ops
    logits, where = make(cuda_device, 700, 48, 3, S=4, mask=True, seed=21)
    where = on(cuda_device, where)
    x = logits.to(cuda_device)
    off, mask = where["sequence_offsets"], where["token_mask"]

    def step(l, r, seed):
        experts, weights, losses, counts, coef = ops.router_topk_balance(l, 3, mask, off)
        d = ops.router_balance_bwd(losses, l, coef, mask, off, experts, weights, weights)
        return experts, weights, losses, counts, d, ops.expert_counts(experts, 48), ops.dropout_add(r, r, seed, 0.3), ops.dropout_add_bwd(r, seed, 0.3)
    r = torch.randn(100, 64, device=cuda_device)
    seed = torch.tensor([5], device=cuda_device)
    want = step(x, r, seed)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(x, r, seed)
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    leaf = x.clone().requires_grad_(True)

    def loss(l):
        _, weights, bal = F.route_balanced(l, 3, **where)
        return (weights * weights).sum() + bal.losses.sum()
    grad, = torch.autograd.grad(loss(leaf), leaf)
    grad_c, = torch.autograd.grad(torch.compile(loss, backend="aot_eager")(leaf), leaf)
    assert torch.equal(grad, grad_c)

    failed = []

    def work():
        try:
            stream = torch.cuda.Stream(cuda_device)
            with torch.cuda.stream(stream):
                for _ in range(20):
                    if not all(torch.equal(a, b) for a, b in zip(want, step(x, r, seed))):
                        raise AssertionError("other bytes")
        except Exception as e:                              # noqa: BLE001 - reported below
            failed.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed, failed


def test_captured_behind_copies_and_other_streams(cuda_device):
    """In a graph, calls whose neighbours are a memset, a copy, and work of another stream that they wait for."""
    from mok import ops
    source = make(cuda_device, 3000, 96, 5, seed=31)[0].to(cuda_device)
    x, seed = torch.zeros_like(source), torch.tensor([3], device=cuda_device)
    want = ops.router_topk_balance(source, 5)
    want_grad = ops.router_balance_bwd(want[2], source, want[4], None, None, want[0], want[1], want[1])
    want_drop = ops.dropout_add(source, source, seed, 0.25)
    side = torch.cuda.Stream(cuda_device)
    pool = torch.cuda.Stream(cuda_device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=pool):
        x.zero_()
        x.copy_(source)
        out = ops.router_topk_balance(x, 5)
        side.wait_stream(pool)
        with torch.cuda.stream(side):
            drop = ops.dropout_add(x, x, seed, 0.25)
            counts = ops.expert_counts(out[0], 96)
        pool.wait_stream(side)
        grad = ops.router_balance_bwd(out[2], x, out[4], None, None, out[0], out[1], out[1])
        drop2 = drop.clone()
        x.zero_()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)) and torch.equal(grad, want_grad)
        assert torch.equal(drop, want_drop) and torch.equal(drop2, want_drop) and torch.equal(counts[0], want[3][0])
        assert int(x.count_nonzero()) == 0
        for t in (*out, grad, drop, drop2, counts):
            t.zero_()
