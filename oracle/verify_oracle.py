"""The verification of drafted tokens from its formulas, in numpy float64: what include/et_speculative.h
defines, one sequence at a time."""
from __future__ import annotations

import numpy as np

EMPTY_REST = 2.0 ** -30


def probabilities(row: np.ndarray, temperature: float):
    """softmax(row / temperature) or None where the row has no distribution."""
    x = row.astype(np.float64)
    if np.isnan(x).any() or np.isnan(temperature) or x.max() in (np.inf, -np.inf):
        return None
    masked = x == -np.inf
    w = np.exp(np.where(masked, 0.0, x - x.max()) / temperature)
    w[masked] = 0.0
    return w / w.sum()


def argmax(row: np.ndarray) -> int:
    """Lowest index of the largest entry, NaN below everything (0 where all are NaN)."""
    x = row.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    best = x.max()
    hits = np.nonzero((x == best) & ~np.isnan(row.astype(np.float64)))[0]
    return int(hits[0]) if hits.size else 0


def draw(weights: np.ndarray, coin: float) -> int:
    sums = np.cumsum(weights)
    hits = np.nonzero((sums > coin * sums[-1]) & (weights > 0))[0]
    return int(hits[0]) if hits.size else int(np.nonzero(weights > 0)[0][-1])


def verify_one(target, draft, drafted, length, temperature, coins, K):
    """target [K + 1, V], draft [K, V] or None, drafted [K], coins [K + 1]; returns (tokens [K + 1], accepted)."""
    V = target.shape[1]
    length = min(max(int(length), 0), K)
    temperature = max(float(temperature), 0.0) if not np.isnan(temperature) else float("nan")
    tokens = np.full(K + 1, -1, dtype=np.int32)
    n, final = 0, None
    while final is None:
        if temperature == 0.0:
            best = argmax(target[n])
            if n < length and drafted[n] == best:
                tokens[n] = best
                n += 1
            else:
                final = best
            continue
        p = probabilities(target[n], temperature)
        if n == length:
            final = -1 if p is None else draw(p, float(coins[K]))
            continue
        x = int(drafted[n])
        inside = 0 <= x < V
        if draft is not None:
            q = probabilities(draft[n], temperature)
        else:
            q = np.zeros(V)
            if inside:
                q[x] = 1.0
        if p is None or q is None:
            final = -1
        elif inside and float(coins[n]) * q[x] < p[x]:
            tokens[n] = x
            n += 1
        else:
            rest = np.maximum(p - q, 0.0)
            final = draw(rest if rest.sum() > EMPTY_REST else p, float(coins[K]))
    tokens[n] = final
    return tokens, n


def verify(target, draft, drafted, lengths, temperatures, coins):
    """float arrays [S, K + 1, V], [S, K, V] or None, [S, K], [S] or None, [S], [S, K + 1]."""
    S, positions, _ = target.shape
    K = positions - 1
    out = [verify_one(target[b], None if draft is None else draft[b], drafted[b], K if lengths is None else lengths[b],
                      float(temperatures[b]), coins[b], K) for b in range(S)]
    return np.stack([o[0] for o in out]), np.array([o[1] for o in out], dtype=np.int32)
