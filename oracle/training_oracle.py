"""64-bit restatement, on the CPU, of what surrounds the experts in a training step: the router's balance and z-losses with
the counts behind them and their gradients, and dropout from a counter-based generator."""
from __future__ import annotations

import numpy as np
import torch


# ---------------------------------------------------------------------------------------------- routing losses
def counted_rows(T: int, token_mask=None, sequence_offsets=None) -> list[np.ndarray]:
    """Indices of the rows that count, per sequence."""
    mask = np.ones(T, bool) if token_mask is None else np.asarray(token_mask, bool)
    bounds = [0, T] if sequence_offsets is None else [min(max(int(o), 0), T) for o in sequence_offsets]
    return [np.arange(a, max(a, b))[mask[a:max(a, b)]] for a, b in zip(bounds, bounds[1:])]


def expert_counts(experts: np.ndarray, E: int, token_mask=None, sequence_offsets=None) -> np.ndarray:
    out = []
    for rows in counted_rows(experts.shape[0], token_mask, sequence_offsets):
        ids = experts[rows].ravel()
        out.append(np.bincount(ids[(ids >= 0) & (ids < E)], minlength=E))
    return np.stack(out).astype(np.int32)


def _softmax(row: torch.Tensor) -> torch.Tensor:
    return torch.softmax(row, 0) if bool((row != -np.inf).any()) else torch.zeros_like(row)


def _scores(rows: torch.Tensor, sigmoid: bool) -> torch.Tensor:
    if sigmoid:                                             # log sigma, normalised: no underflow anywhere
        rows = torch.nn.functional.logsigmoid(rows)
    return torch.softmax(rows, 1)


def losses(logits: torch.Tensor, experts: np.ndarray, *, token_mask=None, sequence_offsets=None, load=None, sigmoid=False) -> torch.Tensor:
    """[balance, z] in float64, differentiable with respect to `logits` (float64)."""
    E = logits.shape[1]
    parts = counted_rows(logits.shape[0], token_mask, sequence_offsets)
    counts = expert_counts(experts, E, token_mask, sequence_offsets) if load is None else np.asarray(load)
    n, live = max(1, sum(map(len, parts))), max(1, sum(len(r) > 0 for r in parts))
    balance = z = logits.new_zeros(())
    for s, rows in enumerate(parts):
        if not len(rows):
            continue
        some = rows[[bool((logits[r].detach() != -np.inf).any()) for r in rows]]
        f = torch.from_numpy(counts[s] * (E / max(1, int(counts[s].sum()))))
        if len(some):
            picked = logits[torch.from_numpy(some)]
            balance = balance + (f * _scores(picked, sigmoid).sum(0)).sum() / (len(rows) * live)
            z = z + (torch.logsumexp(picked, 1) ** 2).sum() / n
    return torch.stack([balance, z])


def select(logits: np.ndarray, K: int) -> np.ndarray:
    """The K largest per row, descending, the lower index among equals, NaN like -inf."""
    return np.argsort(-np.where(np.isnan(logits), -np.inf, logits).astype(np.float64), axis=1, kind="stable")[:, :K]


def weights(logits: torch.Tensor, experts: np.ndarray, sigmoid=False) -> torch.Tensor:
    """Weights of the chosen experts in float64, differentiable; 0 where a row has no logit above -inf."""
    top = logits.gather(1, torch.from_numpy(experts))
    empty = (top == -np.inf).all(1, keepdim=True)
    return torch.where(empty, 0.0, _scores(torch.where(empty, 0.0, top), sigmoid))


# ---------------------------------------------------------------------------------------------- dropout
def philox4x32(counter: np.ndarray, key: tuple[int, int]) -> np.ndarray:
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): counter uint64 [n, 4] of 32-bit words -> uint32 [n, 4]."""
    a, b, c, d = (counter[:, i].astype(np.uint64) for i in range(4))
    low, u32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    k0, k1 = key
    for _ in range(10):
        x, y = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (y >> u32) ^ b ^ np.uint64(k0), y & low, (x >> u32) ^ d ^ np.uint64(k1), x & low
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack([a, b, c, d], 1).astype(np.uint32)


def dropout_keep(seed: int, first: int, count: int, p: float) -> tuple[np.ndarray, float]:
    """(which of the elements first .. first + count - 1 stay, the factor on them)."""
    lo, hi = first // 8, (first + count + 7) // 8
    block = np.arange(lo, hi, dtype=np.uint64)
    zero = np.zeros_like(block)
    words = philox4x32(np.stack([block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), zero, zero], 1),
                       (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    u = words.astype("<u4").view("<u2").ravel()[first - lo * 8:][:count].astype(np.int64)
    threshold = int(np.floor(p * 65536 + 0.5))
    return u >= threshold, 65536 / (65536 - threshold) if threshold < 65536 else 0.0


def dropout_add(x: torch.Tensor, residual, seed: int, p: float, first: int = 0) -> torch.Tensor:
    keep, factor = dropout_keep(seed, first, x.numel(), p)
    out = torch.where(torch.from_numpy(keep).view(x.shape), x.double() * factor, 0.0)
    return out if residual is None else out + residual.double()
