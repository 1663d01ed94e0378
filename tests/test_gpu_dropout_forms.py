"""GPU: dropout of activations in other layouts through the functional call."""
import pytest
import torch

from oracle import training_oracle as O

pytestmark = pytest.mark.gpu


def test_other_layouts_drop_what_their_contiguous_copies_drop(cuda_device):
    """Training takes the layouts that evaluation takes: transposed, strided and broadcast activations and residuals."""
    from mok import functional as F
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    t = lambda *s: torch.randn(s, generator=gen, device=cuda_device).bfloat16()           # noqa: E731
    seed = torch.tensor([99], dtype=torch.int64, device=cuda_device)
    for x, r in ((t(40, 30).t(), t(30, 40)), (t(30, 40), t(40, 30).t()), (t(30, 80)[:, ::2], t(1, 40).expand(30, 40)), (t(40, 30).t(), None)):
        x.requires_grad_(True)
        r = None if r is None else r.requires_grad_(True)
        plain = [None if v is None else v.detach().contiguous().requires_grad_(True) for v in (x, r)]
        got, want = F.dropout_add(x, r, p=0.4, seed=seed), F.dropout_add(*plain, p=0.4, seed=seed)
        assert torch.equal(got, want)
        g = t(30, 40)
        ins = [v for v in (x, r) if v is not None]
        for a, b in zip(torch.autograd.grad(got, ins, g), torch.autograd.grad(want, [v for v in plain if v is not None], g)):
            assert torch.equal(a, b)
        keep, _ = O.dropout_keep(99, 0, 1200, 0.4)
        if r is None:
            assert torch.equal((got == 0).cpu().flatten(), torch.from_numpy(~keep))
        assert torch.equal(F.dropout_add(x, r, p=0.4, training=False), x if r is None else x + r)
