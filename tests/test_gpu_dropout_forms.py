"""GPU: dropout written over one of its inputs, and activations in other layouts through the functional call."""
import pytest
import torch

from oracle import training_oracle as O

pytestmark = pytest.mark.gpu


def run(out, x, residual, seed, p):
    from mok import _lib
    _lib.check(_lib.mok_dropout_add(x.data_ptr(), None if residual is None else residual.data_ptr(), seed.data_ptr(), out.data_ptr(),
                                    x.numel(), x.dtype == torch.bfloat16, p, _lib.stream_ptr(x.device)), "dropout_add")
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("count", [1, 8, 1003, 70001])
@pytest.mark.parametrize("p", [0.0, 0.3, 1.0])
def test_the_result_may_take_the_place_of_an_input(cuda_device, dtype, first, count, p):
    """Bit for bit what a result of its own holds; aligned groups of eight, odd addresses, ends that fill no group."""
    gen = torch.Generator(device=cuda_device).manual_seed(count)
    base = [torch.randn(count + 9, generator=gen, device=cuda_device).to(dtype) for _ in range(2)]
    x, r = (b[first:first + count] for b in base)
    seed = torch.tensor([1234567], dtype=torch.int64, device=cuda_device)
    both = run(torch.empty_like(base[0])[first:first + count], x, r, seed, p)
    alone = run(torch.empty_like(base[0])[first:first + count], x, None, seed, p)

    def over(which, residual):
        bufs = [b.clone() for b in base]
        v = [b[first:first + count] for b in bufs]
        got = run(v[which], v[0], v[1] if residual else None, seed, p)
        for b, c in zip(bufs, base):                        # nothing beside the elements
            assert torch.equal(b[:first], c[:first]) and torch.equal(b[first + count:], c[first + count:])
        assert torch.equal(v[1 - which], base[1 - which][first:first + count])
        return got
    assert torch.equal(over(0, True), both) and torch.equal(over(1, True), both) and torch.equal(over(0, False), alone)


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
