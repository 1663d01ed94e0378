"""CPU: the oracle of the routing losses and of dropout against published numbers, torch's autograd and differences; the
refusals of the operators; the host side of the functional calls."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import training_oracle as O


# ---------------------------------------------------------------------------------------------- the oracle
def test_generator_gives_the_published_answers():
    """Known answers that accompany the generator's publication (counter, key -> output)."""
    ones = 0xFFFFFFFF
    for counter, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((ones,) * 4, (ones, ones), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(O.philox4x32(np.array([counter], dtype=np.uint64), key)[0]) == want


def test_dropout_rate_and_pieces():
    keep, factor = O.dropout_keep(12345, 0, 200000, 0.3)
    assert abs(keep.mean() - 0.7) < 5 * (0.21 / 200000) ** 0.5 and abs(factor - 1 / 0.7) < 1e-4
    part, _ = O.dropout_keep(12345, 777, 1003, 0.3)
    assert (part == keep[777:777 + 1003]).all()
    assert O.dropout_keep(1, 0, 64, 0.0)[0].all() and not O.dropout_keep(1, 0, 64, 1.0)[0].any()


def test_even_routing_has_balance_one():
    T, E, K = 64, 8, 2
    experts = np.stack([np.arange(T) % E, (np.arange(T) + 3) % E], 1)
    got = O.losses(torch.zeros(T, E, dtype=torch.float64), experts)
    assert abs(float(got[0]) - 1.0) < 1e-12 and abs(float(got[1]) - np.log(E) ** 2) < 1e-12


@pytest.mark.parametrize("sigmoid", [False, True])
def test_oracle_gradient_is_the_formulas_and_that_of_differences(sigmoid):
    """a_e = f_e / n_s of the row's sequence: d balance = p (a - sum p a) / S' (times 1 - sigma), d z = 2/n lse softmax."""
    rng = np.random.default_rng(3)
    T, E, K = 23, 9, 3
    logits = torch.from_numpy(rng.standard_normal((T, E)) * 2).requires_grad_(True)
    experts = O.select(logits.detach().numpy(), K)
    where = dict(token_mask=rng.random(T) < 0.8, sequence_offsets=[2, 9, 9, 20])
    g = torch.tensor([0.7, -0.3], dtype=torch.float64)
    grad, = torch.autograd.grad(O.losses(logits, experts, sigmoid=sigmoid, **where) @ g, logits)
    want = torch.zeros(T, E, dtype=torch.float64)
    parts = O.counted_rows(T, **where)
    counts = O.expert_counts(experts, E, **where)
    n, live = sum(map(len, parts)), sum(len(r) > 0 for r in parts)
    with torch.no_grad():
        for s, rows in enumerate(parts):
            for r in rows:
                a = torch.from_numpy(counts[s] * E / counts[s].sum() / len(rows))
                soft, sig = torch.softmax(logits[r], 0), torch.sigmoid(logits[r])
                p = sig / sig.sum() if sigmoid else soft
                d = p * (a - (p * a).sum()) / live * ((1 - sig) if sigmoid else 1)
                want[r] = g[0] * d + g[1] * 2 / n * torch.logsumexp(logits[r], 0) * soft
    assert (grad - want).abs().max() < 1e-14
    for r, e in ((3, 1), (10, 0), (0, 0), (22, 4)):
        h = 1e-5
        moved = [logits.detach().clone() for _ in range(2)]
        moved[0][r, e] += h
        moved[1][r, e] -= h
        up, down = (O.losses(m, experts, sigmoid=sigmoid, **where) @ g for m in moved)
        assert abs(float(up - down) / (2 * h) - float(grad[r, e])) < 1e-8


# ---------------------------------------------------------------------------------------------- refusals
def _raises(exc, call, *args, **kwargs):
    with pytest.raises(exc):
        call(*args, **kwargs)


def test_operators_refuse_cpu_tensors_and_wrong_arguments():
    """Every check that does not need a device; the rest are with the GPU tests."""
    from mok import functional as F, nn, ops
    logits, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    _raises(ValueError, ops.router_balance, logits, ids)
    _raises(ValueError, ops.router_topk_balance, logits, 2)
    _raises(ValueError, ops.router_balance_bwd, torch.zeros(2), logits, torch.zeros(10))
    _raises(ValueError, ops.expert_counts, ids, 8)
    _raises(ValueError, ops.dropout_add, logits, None, torch.zeros(1, dtype=torch.int64), 0.1)
    _raises(ValueError, ops.dropout_add_bwd, logits, torch.zeros(1, dtype=torch.int64), 0.1)
    for call in (lambda **k: F.route_balanced(logits, 2, **k), lambda **k: F.balance_loss(logits, ids, **k)):
        _raises(ValueError, call, score="tanh")
    _raises(ValueError, F.balance_loss, logits, ids, sequence_offsets=torch.zeros(2, dtype=torch.int32), group=object())
    for p in (-0.1, 1.5, float("nan"), "0.1"):
        _raises(ValueError, F.dropout_add, logits, p=p)
    _raises(ValueError, F.dropout_add, logits, torch.zeros(4, 7), p=0.0)
    _raises(TypeError, F.route_balanced_and_schedule, None, F.MoKConfig(), logits, num_local_experts=8)
    for kwargs in (dict(score="none"), dict(dropout=1.5), dict(dropout="x")):
        _raises(ValueError, nn.MoKLayer, 256, 256, 4, 2, group=_one_rank(), device="cpu", **kwargs)
    layer = nn.MoKLayer(256, 256, 4, 2, group=_one_rank(), device="cpu")
    x = torch.zeros(512, 256, dtype=torch.bfloat16)
    _raises(ValueError, layer, x, ids, None)
    _raises(ValueError, layer, x, ids, torch.zeros(4, 2), return_balance=True)
    _raises(ValueError, layer, x, token_mask=torch.ones(512, dtype=torch.bool))


def _one_rank():
    import torch.distributed as dist
    if not dist.is_initialized():
        dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    return dist.group.WORLD


def test_c_entries_refuse_bad_arguments():
    from mok import _lib as L
    p = ctypes.c_void_p(4096)
    z = None
    p = 4096
    balance = lambda *, logits=p, T=512, E=8, K=2, S=1, top=p, out=0, w=0, off=0, n=1 << 20, scratch=p: L.mok_router_balance(  # noqa: E731
        L.pack_router_balance(logits, top, out, w, 0, off, 0, p, p, p, scratch, n, 0, T, E, K, S, 0), None)
    assert L.mok_router_balance(None, None) == L.mok_router_balance_bwd(None, None) == -1
    assert balance(logits=0) == balance(T=0) == balance(E=0) == balance(K=0) == balance(K=256) == balance(S=0) == -1
    assert balance(S=2) == balance(top=0) == balance(out=p, w=p) == balance(w=p) == balance(top=0, out=p) == -1
    assert balance(top=0, out=p, w=p, K=9) == balance(top=0, out=p, w=p, E=64, K=33) == -1
    many = dict(T=100000, E=64)
    assert balance(n=64, **many) == balance(scratch=4104, **many) == balance(scratch=0, **many) == -1
    for chooses in (0, 1):
        assert L.mok_router_balance_scratch_bytes(512, 8, 1, chooses) == 0 < L.mok_router_balance_scratch_bytes(100000, 64, 1, chooses)
    assert L.mok_router_balance_scratch_bytes(2816, 24, 1, 0) == 0 < L.mok_router_balance_scratch_bytes(2816, 24, 1, 1)
    assert balance(E=1025) == -3 and balance(T=1 << 24, K=200) == balance(T=0x7fffffff, K=1) == -4
    assert L.mok_router_balance_scratch_bytes(0, 8, 1, 0) == 0
    bwd = lambda *, g=p, T=512, E=8, K=2, S=1, top=0, w=0, dw=0, off=0: L.mok_router_balance_bwd(                              # noqa: E731
        L.pack_router_balance_bwd(g, p, p, 0, off, top, w, dw, p, 0, T, E, K, S, 0), None)
    assert bwd(g=0) == bwd(T=0) == bwd(S=3) == bwd(top=p) == bwd(top=p, w=p) == bwd(top=p, w=p, dw=p, K=33, E=64) == -1
    assert bwd(top=p, w=p, dw=p, K=9) == -1
    assert bwd(E=2000) == -3 and bwd(T=0x7fffffff) == bwd(S=1 << 30, off=p) == -4
    p = ctypes.c_void_p(4096)
    counts = lambda *, ids=p, T=512, E=8, K=2, S=1, off=z: L.mok_expert_counts(ids, 0, T, K, E, S, z, off, p, z)              # noqa: E731
    assert counts(ids=z) == counts(T=-1) == counts(E=0) == counts(S=2) == -1
    assert counts(E=1025) == -3 and counts(T=1 << 30, K=4) == -4
    drop = lambda x=p, seed=p, out=p, n=8, rate=0.5: L.mok_dropout_add(x, z, seed, out, n, 1, rate, z)                         # noqa: E731
    assert drop(x=z) == drop(seed=z) == drop(out=z) == drop(n=0) == drop(n=-1) == drop(rate=1.01) == drop(rate=float("nan")) == -1


def test_packed_arguments_have_the_layout_of_the_structs():
    """Member by member, checked with gcc on the header: every field is set to a number of its own."""
    import os
    import subprocess
    import tempfile
    from mok import _lib as L
    from tests.conftest import ROOT
    text = open(os.path.join(ROOT, "include", "mok_b200.h")).read()
    for name, pack, n in (("mok_router_balance_args", L.pack_router_balance, 18), ("mok_router_balance_bwd_args", L.pack_router_balance_bwd, 15)):
        body = text[text.index("typedef struct " + name):]
        body = body[body.index("{") + 1:body.index("}")]
        fields = [w.split()[-1].strip("*") for line in body.split(";") for w in line.split(",") if w.strip()]
        assert len(fields) == n
        src = '#include <stdio.h>\n#include <string.h>\n#include "mok_b200.h"\nint main(){%s a; if (fread(&a, 1, sizeof a + 1, stdin) != sizeof a) return 1;' % name
        src += "".join('printf("%%lld ", (long long)a.%s);' % f for f in fields) + "return 0;}"
        with tempfile.TemporaryDirectory() as d:
            c, exe = os.path.join(d, "s.c"), os.path.join(d, "s")
            open(c, "w").write(src)
            subprocess.check_call(["gcc", "-w", "-I", os.path.join(ROOT, "include"), c, "-o", exe])
            out = subprocess.run([exe], input=pack(*range(1, n + 1)), capture_output=True, check=True).stdout
        assert [int(v) for v in out.split()] == list(range(1, n + 1)), name


# ---------------------------------------------------------------------------------------------- host side
def test_slots_of_block_and_sequence_are_never_shared():
    """The forward kernel's staircase: block + sequence is unique among the pairs that meet, whatever the lengths."""
    rng = np.random.default_rng(0)
    for _ in range(300):
        T, S, blocks = int(rng.integers(1, 200)), int(rng.integers(1, 40)), int(rng.integers(1, 30))
        cuts = np.sort(rng.integers(0, T + 1, S + 1))
        per = -(-T // blocks)
        pairs = [(b, s) for b in range(blocks) for s in range(S)
                 if max(b * per, cuts[s]) < min(min((b + 1) * per, T), cuts[s + 1])]
        slots = [b + s for b, s in pairs]
        assert len(set(slots)) == len(slots) and all(0 <= v < blocks + S for v in slots)


def test_group_counts_are_summed_before_the_loss(monkeypatch):
    """balance_loss(group=...): expert_counts -> all-reduce -> the loss with the sum as its load."""
    from mok import functional as F, ops
    seen = {}
    monkeypatch.setattr(ops, "expert_counts", lambda ids, E, mask: torch.tensor([[3, 1]], dtype=torch.int32))
    monkeypatch.setattr(F.dist, "all_reduce", lambda t, group: t.add_(torch.tensor([[1, 7]], dtype=torch.int32)))

    def balance(logits, ids, mask, offsets, load, sigmoid):
        seen["load"] = load
        return torch.ones(2), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(4)
    monkeypatch.setattr(ops, "router_balance", balance)
    out = F.balance_loss(torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.int64), group=object())
    assert seen["load"].tolist() == [[4, 8]] and out.losses.tolist() == [1.0, 1.0]
    assert float(out.balance) == float(out.z) == 1.0


def test_dropout_without_anything_to_drop_draws_no_seed(monkeypatch):
    from mok import functional as F
    monkeypatch.setattr(torch, "randint", lambda *a, **k: pytest.fail("seed drawn"))
    x, r = torch.randn(3, 4), torch.randn(3, 4)
    assert F.dropout_add(x, p=0.0) is x and F.dropout_add(x, p=0.4, training=False) is x
    assert torch.equal(F.dropout_add(x, r, p=0.4, training=False), x + r)


def test_launches_run_with_the_tensors_device_current(monkeypatch):
    from mok import _lib
    calls, current = [], [0]

    class Device:
        def __init__(self, device): self.index = device.index
        def __enter__(self): self.before, current[0] = current[0], self.index
        def __exit__(self, *exc): current[0] = self.before
    monkeypatch.setattr(_lib, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 100 + device.index)
    entry = lambda *args: calls.append((current[0], args)) or 0              # noqa: E731
    _lib.launch(torch.device("cuda", 0), "op", entry, 1)
    _lib.launch(torch.device("cuda", 3), "op", entry, 2)
    assert calls == [(0, (1, 100)), (3, (2, 103))] and current == [0]
    with pytest.raises(ValueError):
        _lib.launch(torch.device("cuda", 0), "op", lambda *a: -1)


def test_operators_with_optional_tensors_take_the_short_way():
    import mok
    op = mok.ops.dropout_add
    x, seed = torch.ones(8), torch.zeros(1, dtype=torch.int64)
    assert op._forwards_only((x, None, seed, 0.1)) and op._forwards_only((x, x, seed, 0))
    assert not op._forwards_only((x.requires_grad_(True), None, seed, 0.1))
    y = torch.ones(8, requires_grad=True)
    assert not op._forwards_only((torch.ones(8), y, seed, 0.1))
    assert not op._forwards_only((torch.ones(8), torch.ones(8, device="meta"), seed, 0.1))
    assert mok.ops.router_balance._forwards_only((torch.ones(2, 4), torch.zeros(2, 2, dtype=torch.int64)))


def test_meta_tensors_get_shapes():
    import mok
    m = lambda dtype, *shape: torch.empty(*shape, dtype=dtype, device="meta")         # noqa: E731
    logits, ids, off = m(torch.bfloat16, 700, 12), m(torch.int64, 700, 3), m(torch.int32, 6)
    shapes = lambda ts: [(tuple(t.shape), t.dtype) for t in ts]                        # noqa: E731
    tail = [((2,), torch.float32), ((5, 12), torch.int32), ((62,), torch.float32)]
    assert shapes(mok.ops.router_balance(logits, ids, None, off)) == tail
    assert shapes(mok.ops.router_topk_balance(logits, 3, None, off)) == [((700, 3), torch.int64), ((700, 3), torch.float32)] + tail
    assert shapes([mok.ops.expert_counts(ids, 12, None, off)]) == tail[1:2]
    assert shapes([mok.ops.router_balance_bwd(m(torch.float32, 2), logits, m(torch.float32, 62), None, off),
                   mok.ops.dropout_add(logits, None, m(torch.int64, 1), 0.5),
                   mok.ops.dropout_add_bwd(logits, m(torch.int64, 1), 0.5)]) == [((700, 12), torch.bfloat16)] * 3
