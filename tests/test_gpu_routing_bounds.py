"""GPU: routing with its losses where rows hold NaN.  u = 2^-24 is half a step of f32; a bf16 result is off by 2^-8 of the value more."""
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
