"""Operators around the experts of a training step: the calls a trainer makes of them, over the range of sizes it makes
them with.

  route    the router with its losses: top-K experts and weights, balance loss, z-loss and per-expert counts from one
           set of logits, then the gradient of the logits from all of them
  balance  the same losses for finished routes, and their gradient
  counts   routes per expert, the numbers that ranks add up before a loss over the global batch
  dropout  dropout from a counter-based generator at the layer's exit, with the residual, and its gradient

Where `own` is false everything is computed in plain torch operations, in 32 bits (long sums in 64).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# gradient weights a trainer gives the two losses
_BALANCE_COEF, _Z_COEF = 0.01, 0.001


def _mok():
    # the package's folder has a dash in its name, so it is reached the way the tests reach it
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mixture-of-kittens_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import mok
    return mok


# ------------------------------------------------------------------------------------------------------ cases
def _route(name, T, E, K, dtype="f32", score="softmax", S=0, mask=False):
    return {"name": name, "kind": "route", "T": T, "E": E, "K": K, "dtype": dtype, "score": score, "S": S, "mask": mask}


def _dropout(name, rows, cols, dtype, *, residual=True, backward=True, p=0.1):
    return {"name": name, "kind": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "residual": residual,
            "backward": backward, "p": p}


def listed():
    return [
        # the smallest batch the layer takes, a handful of experts: launches and host time are all there is
        _route("route_smallest", 512, 8, 2),
        # the benchmark's layer (128 experts, top-8) on one rank's batch
        _route("route_train", 16384, 128, 8),
        # fine-tuning on packed sequences: bf16 logits, sigmoid scores, padding rows masked and rows behind the last sequence
        _route("route_packed", 10007, 256, 8, dtype="bf16", score="sigmoid", S=37, mask=True),
        # a long-context step, many experts
        _route("route_large", 131072, 256, 8),
        # losses alone, for a model whose own code chose the experts: the ragged fine-tuning layer
        {**_route("balance_small", 2816, 24, 5), "kind": "balance"},
        # a large expert set, one loss per packed sequence
        {**_route("balance_large", 65536, 500, 6, dtype="bf16", S=61), "kind": "balance"},
        # counts of one layer in a logging step, and of a large batch over one of eight ranks' worth of sequences
        {"name": "counts_small", "kind": "counts", "T": 512, "E": 4, "K": 2, "S": 0, "mask": False},
        {"name": "counts_large", "kind": "counts", "T": 262144, "E": 256, "K": 8, "S": 16, "mask": True},
        # the smallest layer's output, inference-sized
        _dropout("dropout_smallest", 512, 256, "bf16", residual=False, backward=False),
        # the residual of the benchmark's layer
        _dropout("dropout_train", 16384, 2048, "bf16"),
        # odd sizes, 32-bit activations
        _dropout("dropout_odd", 5003, 1021, "f32", p=0.37),
        # the largest layer's residual
        _dropout("dropout_large", 16384, 7168, "bf16", p=0.05),
    ]


def _log_uniform(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    kind = rng.choice(["route", "route", "balance", "counts", "dropout", "dropout"])
    if kind == "dropout":
        cols = _log_uniform(rng, 200, 7168)
        rows = min(_log_uniform(rng, 300, 60000), 16384 * 7168 // cols)
        dtype = rng.choice(["bf16", "bf16", "f32"])
        if dtype == "f32":
            rows = max(1, rows // 2)
        return {"kind": kind, "rows": rows, "cols": cols, "dtype": dtype, "residual": rng.random() < 0.7,
                "backward": rng.random() < 0.7, "p": round(rng.uniform(0.01, 0.6), 4)}
    E = _log_uniform(rng, 4, 1024)
    K = rng.randint(1, min(E, 16))
    T = _log_uniform(rng, 300, 131072)
    if kind == "counts":
        return {"kind": kind, "T": T, "E": E, "K": K, "S": rng.choice([0, rng.randint(1, 64)]), "mask": rng.random() < 0.5}
    T = max(256, min(T, 131072 * 256 // (E * max(1, K // 8))))
    return {"kind": kind, "T": T, "E": E, "K": K, "dtype": rng.choice(["f32", "f32", "bf16"]),
            "score": rng.choice(["softmax", "softmax", "sigmoid"]), "S": rng.choice([0, rng.randint(1, 64)]), "mask": rng.random() < 0.4}


# ------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    if case["kind"] == "dropout":
        dt = _DTYPES[case["dtype"]]
        shape = (case["rows"], case["cols"])
        st["x"] = torch.randn(shape, generator=gen, device="cuda").to(dt)
        st["res"] = torch.randn(shape, generator=gen, device="cuda").to(dt) if case["residual"] else None
        st["d_out"] = torch.randn(shape, generator=gen, device="cuda").to(dt) if case["backward"] else None
        st["seed"] = torch.randint(0, 2 ** 63 - 1, (1,), generator=gen, device="cuda")
    else:
        T, E, K, S = (case[n] for n in "TEKS")
        # experts differ in popularity, tokens in how sure the router is
        logits = torch.randn(T, E, generator=gen, device="cuda") * 1.5 + torch.randn(E, generator=gen, device="cuda") * 0.7
        st["mask"] = torch.rand(T, generator=gen, device="cuda") < 0.9 if case["mask"] else None
        st["offsets"] = None
        if S:                                           # ragged sequences, some empty, and rows behind the last one
            cuts = torch.randint(0, T - T // 64, (S - 1,), generator=gen, device="cuda").sort().values
            ends = torch.tensor([0, T - T // 64], device="cuda")
            st["offsets"] = torch.cat([ends[:1], cuts, ends[1:]]).int()
        if case["kind"] != "route":
            st["experts"] = torch.topk(logits, K, dim=1).indices
        if case["kind"] != "counts":
            st["logits"] = logits.to(_DTYPES[case["dtype"]])
            st["d_losses"] = torch.tensor([_BALANCE_COEF, _Z_COEF], device="cuda")
        if case["kind"] == "route":
            st["d_weights"] = torch.randn(T, K, generator=gen, device="cuda") * 0.1
    if own:
        st["ops"] = _mok().ops
    return st


def work(case):
    if case["kind"] == "dropout":
        n, b = case["rows"] * case["cols"], 2 if case["dtype"] == "bf16" else 4
        return {"bytes": n * b * (2 + case["residual"] + 2 * case["backward"]), "flops": n * (2 + case["backward"])}
    T, E, K, S = case["T"], case["E"], case["K"], max(1, case["S"])
    routes = T * K * 8 + (T if case["mask"] else 0) + S * E * 4
    if case["kind"] == "counts":
        return {"bytes": routes, "flops": T * K}
    b = 2 if case["dtype"] == "bf16" else 4
    more = T * K * 8 if case["kind"] == "route" else 0  # weights out, their gradient in
    return {"bytes": routes + 2 * T * E * b + more, "flops": 20 * T * E}


# ------------------------------------------------------------------------------------------------------ the operators
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    ops, kind = st["ops"], st["kind"]
    if kind == "dropout":
        out = ops.dropout_add(st["x"], st["res"], st["seed"], st["p"])
        return (out, ops.dropout_add_bwd(st["d_out"], st["seed"], st["p"])) if st["backward"] else (out,)
    if kind == "counts":
        return (ops.expert_counts(st["experts"], st["E"], st["mask"], st["offsets"]),)
    sigmoid = st["score"] == "sigmoid"
    if kind == "balance":
        losses, counts, coef = ops.router_balance(st["logits"], st["experts"], st["mask"], st["offsets"], None, sigmoid)
        d_logits = ops.router_balance_bwd(st["d_losses"], st["logits"], coef, st["mask"], st["offsets"], None, None, None, sigmoid)
        return losses, counts, d_logits
    experts, weights, losses, counts, coef = ops.router_topk_balance(st["logits"], st["K"], st["mask"], st["offsets"], sigmoid)
    d_logits = ops.router_balance_bwd(st["d_losses"], st["logits"], coef, st["mask"], st["offsets"], experts, weights,
                                      st["d_weights"], sigmoid)
    return experts, weights, losses, counts, d_logits


def _segments(st):
    """Per token: its sequence, and whether it counts."""
    T, S = st["T"], max(1, st["S"])
    at = torch.arange(T, device="cuda")
    if st["offsets"] is None:
        seq, counted = torch.zeros_like(at), torch.ones(T, dtype=torch.bool, device="cuda")
    else:
        off = st["offsets"].long()
        seq = torch.searchsorted(off, at, right=True) - 1
        counted = (seq >= 0) & (at < off[-1])
        seq = seq.clamp(0, S - 1)
    if st["mask"] is not None:
        counted = counted & st["mask"]
    return seq, counted, S


def _counts(st, experts, seq, counted, S):
    slot = seq[:, None] * st["E"] + experts
    got = torch.zeros(S * st["E"], dtype=torch.int64, device="cuda")
    got.scatter_add_(0, slot.flatten(), counted[:, None].expand_as(slot).flatten().long())
    return got.view(S, st["E"])


def _run_plain(st):
    if st["kind"] == "dropout":
        keep, scale = _keep(st["seed"], st["x"].numel(), st["p"])
        keep = keep.view(st["x"].shape)
        out = torch.where(keep, st["x"].float() * scale, 0.0)
        if st["res"] is not None:
            out = out + st["res"].float()
        out = out.to(st["x"].dtype)
        if not st["backward"]:
            return (out,)
        return out, torch.where(keep, st["d_out"].float() * scale, 0.0).to(st["x"].dtype)
    seq, counted, S = _segments(st)
    if st["kind"] == "counts":
        return (_counts(st, st["experts"], seq, counted, S).int(),)
    E, K = st["E"], st["K"]
    logits, sigmoid = st["logits"].float(), st["score"] == "sigmoid"
    if st["kind"] == "route":
        top, experts = torch.sort(logits, dim=1, descending=True, stable=True)
        top, experts = top[:, :K], experts[:, :K]
        raw = 1.0 / (1.0 + torch.exp(-top)) if sigmoid else torch.exp(top - top[:, :1])
        weights = raw / raw.sum(1, keepdim=True)
    else:
        experts = st["experts"]
    counts = _counts(st, experts, seq, counted, S)
    # probabilities over all experts, log of the sum of exponentials
    m = logits.max(1, keepdim=True).values
    ex = torch.exp(logits - m)
    total = ex.sum(1, keepdim=True)
    q = ex / total
    lse = (m + torch.log(total)).squeeze(1)
    sig = 1.0 / (1.0 + torch.exp(-logits))
    p = sig / sig.sum(1, keepdim=True) if sigmoid else q
    # the losses
    member = torch.zeros(S, st["T"], dtype=torch.float64, device="cuda")
    member.scatter_(0, seq[None], counted[None].double())
    n_seq = member.sum(1)
    n, live = n_seq.sum().clamp(min=1), (n_seq > 0).sum().clamp(min=1)
    mean_p = (member @ p.double()) / n_seq.clamp(min=1)[:, None]
    share = counts.double() * E / counts.sum(1, keepdim=True).clamp(min=1)
    balance = (share * mean_p).sum() / live
    z = torch.where(counted, lse.double() ** 2, 0.0).sum() / n
    losses = torch.stack([balance, z]).float()
    # the gradient
    coef = (share / n_seq.clamp(min=1)[:, None] / live).float()[seq]
    inner = p * (coef - (p * coef).sum(1, keepdim=True))
    if sigmoid:
        inner = inner * (1.0 - sig)
    d_logits = st["d_losses"][0] * inner + st["d_losses"][1] * (2.0 / n.float()) * lse[:, None] * q
    d_logits = torch.where(counted[:, None], d_logits, 0.0)
    if st["kind"] == "balance":
        return losses, counts.int(), d_logits.to(st["logits"].dtype)
    d_w = weights * (st["d_weights"] - (weights * st["d_weights"]).sum(1, keepdim=True))
    if sigmoid:
        d_w = d_w * (1.0 - raw)
    d_logits = d_logits.scatter_add(1, experts, d_w)
    return experts, weights, losses, counts.int(), d_logits.to(st["logits"].dtype)


def _keep(seed, count, p):
    """(which of `count` elements stay, the factor on them) by Philox4x32-10 (Salmon et al., 2011): block i >> 3 of the
    counter gives eight 16-bit numbers, an element stays where its number is at least round(65536 p)."""
    low = 0xFFFFFFFF
    threshold = int(math.floor(p * 65536 + 0.5))
    block = torch.arange((count + 7) // 8, device="cuda")
    c = [block & low, block >> 32, torch.zeros_like(block), torch.zeros_like(block)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        h0, l0 = _product(0xD2511F53, c[0])
        h1, l1 = _product(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    halves = torch.stack([w >> s & 0xFFFF for w in c for s in (0, 16)], dim=1).flatten()[:count]
    return halves >= threshold, 65536.0 / (65536 - threshold) if threshold < 65536 else 0.0


def _product(a, b):
    """High and low 32 bits of a * b; 64-bit signed products of 16-bit halves of b do not overflow."""
    lo, hi = a * (b & 0xFFFF), a * (b >> 16)
    mid = hi + (lo >> 16)
    return mid >> 16, (mid & 0xFFFF) << 16 | (lo & 0xFFFF)


# ------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "dropout":
        return _exact_dropout(st)
    T, E, K, S = case["T"], case["E"], case["K"], max(1, case["S"])
    mask = np.ones(T, bool) if st["mask"] is None else st["mask"].cpu().numpy()
    bounds = [0, T] if st["offsets"] is None else st["offsets"].tolist()
    rows = [np.arange(bounds[s], bounds[s + 1])[mask[bounds[s]:bounds[s + 1]]] for s in range(S)]
    picked = None if case["kind"] == "counts" else st["logits"].double()
    if case["kind"] == "route":
        left, chosen = picked.clone(), []
        for _ in range(K):                              # the largest left, the lowest index among equals
            best = left.max(1, keepdim=True).values
            at = torch.where(left == best, torch.arange(E, device="cuda"), E).min(1, keepdim=True).values
            left.scatter_(1, at, -math.inf)
            chosen.append(at)
        experts = torch.cat(chosen, 1)
        top = picked.gather(1, experts)
        if case["score"] == "sigmoid":
            weights = torch.sigmoid(top)
            slope = 1 - weights
            weights = weights / weights.sum(1, keepdim=True)
        else:
            weights, slope = torch.softmax(top, 1), 1.0
    else:
        experts = st["experts"]
    routes = experts.cpu().numpy()
    counts = np.stack([np.bincount(routes[r].ravel(), minlength=E) for r in rows])
    if case["kind"] == "counts":
        return (torch.from_numpy(counts).int(),)
    grad = torch.zeros(T, E, dtype=torch.float64, device="cuda")
    d_balance, d_z = (float(v) for v in st["d_losses"])
    n, live = max(1, sum(map(len, rows))), max(1, sum(len(r) > 0 for r in rows))
    balance = z = 0.0
    for s, r in enumerate(rows):
        if not len(r):
            continue
        at = torch.from_numpy(r).cuda()
        l = picked[at]
        soft = torch.softmax(l, 1)
        sig = torch.sigmoid(l)
        p = sig / sig.sum(1, keepdim=True) if case["score"] == "sigmoid" else soft
        f = torch.from_numpy(counts[s] * (E / max(1, counts[s].sum()))).cuda()
        lse = torch.logsumexp(l, 1)
        balance += float((p.mean(0) * f).sum()) / live
        z += float((lse * lse).sum()) / n
        g = p * (f - p @ f[:, None]) / (len(r) * live)
        grad[at] = d_balance * (g * (1 - sig) if case["score"] == "sigmoid" else g) + d_z * 2 / n * lse[:, None] * soft
    losses = torch.tensor([balance, z], dtype=torch.float64)
    counts = torch.from_numpy(counts).int()
    if case["kind"] == "balance":
        return losses, counts, grad
    dw = st["d_weights"].double()
    grad.scatter_add_(1, experts, weights * (dw - (weights * dw).sum(1, keepdim=True)) * slope)
    return experts, weights, losses, counts, grad


def _exact_dropout(st):
    n = st["x"].numel()
    seed = int(st["seed"])
    keys = [(seed & 0xFFFFFFFF, seed >> 32)]
    for _ in range(9):
        keys.append(((keys[-1][0] + 0x9E3779B9) % 2 ** 32, (keys[-1][1] + 0xBB67AE85) % 2 ** 32))
    drop = math.floor(st["p"] * 65536 + 0.5)
    factor = 65536.0 / (65536 - drop) if drop < 65536 else 0.0
    kept = np.empty(-(-n // 8) * 8, bool)
    u32, word = np.uint64(32), np.uint64(0xFFFFFFFF)
    for first in range(0, kept.size // 8, 1 << 18):     # a slice of counters at a time stays in the host's cache
        i = np.arange(first, min(first + (1 << 18), kept.size // 8), dtype=np.uint64)
        a, b, c, d = i & word, i >> u32, np.zeros_like(i), np.zeros_like(i)
        for k0, k1 in keys:
            x, y = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
            a, b, c, d = (y >> u32) ^ b ^ np.uint64(k0), y & word, (x >> u32) ^ d ^ np.uint64(k1), x & word
        words = np.stack([a, b, c, d], 1).astype("<u4")
        kept[first * 8:first * 8 + i.size * 8] = (words.view("<u2") >= drop).ravel() if drop < 65536 else False
    keep = torch.from_numpy(kept[:n]).cuda().view(st["x"].shape)
    out = torch.where(keep, st["x"].double() * factor, 0.0)
    if st["res"] is not None:
        out += st["res"].double()
    if not st["backward"]:
        return (out,)
    return out, torch.where(keep, st["d_out"].double() * factor, 0.0)
