"""The dense operators around the MoE block in 64 bits, on the CPU: projections with their epilogue, rotary positions,
verification of drafted tokens.  Plain numpy, one row at a time where the definition is one row at a time."""
from __future__ import annotations

import math

import numpy as np

_erf = np.vectorize(math.erf, otypes=[np.float64])


def activation(y, name):
    with np.errstate(over="ignore", invalid="ignore"):
        if name is None:
            return y
        if name == "relu":
            return np.where(y < 0, 0.0, y)
        if name == "silu":
            return y / (1.0 + np.exp(-y))
        if name == "gelu":
            return 0.5 * y * (1.0 + _erf(y / math.sqrt(2.0)))
        if name == "gelu_tanh":
            return 0.5 * y * (1.0 + np.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)))
    raise ValueError(name)


def linear(x, w, bias=None, act=None, residual=None):
    """(the result, the sum of the products' magnitudes, the sum without bias)."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    pre = x @ w.T
    y = activation(pre if bias is None else pre + np.asarray(bias, np.float64), act)
    return (y if residual is None else y + np.asarray(residual, np.float64)), np.abs(x) @ np.abs(w).T, pre


def rotary(x, positions, inv_freq, sections=None, interleaved=False, weight=None, eps=1e-6):
    """x [n, heads, D], positions [n] or [axes, n]: (the result, what bounds each output's error: |x1| + |x2| of its pair)."""
    x = np.array(x, np.float64)
    pos = np.atleast_2d(np.asarray(positions)).astype(np.float64)
    half = len(inv_freq)
    sections = sections or (half,)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    y, size = x.copy(), np.abs(x)
    f = 0
    for axis, count in enumerate(sections):
        for _ in range(count):
            lo, hi = (2 * f, 2 * f + 1) if interleaved else (f, f + half)
            angle = (pos[axis] * inv_freq[f])[:, None]
            c, s = np.cos(angle), np.sin(angle)
            y[..., lo] = x[..., lo] * c - x[..., hi] * s
            y[..., hi] = x[..., hi] * c + x[..., lo] * s
            size[..., lo] = size[..., hi] = np.abs(x[..., lo]) + np.abs(x[..., hi])
            f += 1
    return y, size


def distribution(row, temperature):
    """softmax(row / temperature) in 64 bits; one-hot at the first of the largest for temperature 0.  NaN counts as -inf, a row
    without a number is zero everywhere, +inf takes all."""
    row = np.where(np.isnan(row), -np.inf, np.asarray(row, np.float64))
    top = row.max()
    if top == -np.inf:
        return np.zeros_like(row)
    if not temperature > 0:
        p = np.zeros_like(row)
        p[int(np.argmax(row))] = 1.0
        return p
    if top == np.inf:
        e = (row == np.inf).astype(np.float64)
    else:
        e = np.exp((row - top) / float(temperature))
    return e / e.sum()


def draw(weights, r):
    """The lowest token whose inclusive cumulative weight exceeds r times the total; -1 without any weight."""
    run_up = np.cumsum(weights)
    if not run_up[-1] > 0:
        return -1
    past = np.nonzero(run_up > r * run_up[-1])[0]
    return int(past[0]) if past.size else int(np.nonzero(weights)[0][-1])


def verify(logits, draft_tokens, lens, accept_u, sample_u, draft_logits=None, temperature=1.0, max_query_len=None):
    """(tokens [S, max_query_len], accepted [S], accept probabilities [n_drafts])."""
    S = len(lens)
    width = max_query_len or max(lens, default=0)
    temperature = np.broadcast_to(np.asarray(temperature, np.float64), (S,))
    tokens = np.full((S, width), -1, np.int64)
    accepted = np.zeros(S, np.int32)
    probs = np.zeros(0 if draft_tokens is None else len(draft_tokens), np.float64)
    row = draft = 0
    for s, n in enumerate(lens):
        weights = None
        for j in range(n - 1):
            d = int(draft_tokens[draft + j])
            p = distribution(logits[row + j], temperature[s])
            if draft_logits is not None:
                q = distribution(draft_logits[draft + j], temperature[s])
            else:
                q = np.zeros_like(p)
                if 0 <= d < p.size:
                    q[d] = 1.0
            if 0 <= d < p.size:
                probs[draft + j] = min(1.0, p[d] / q[d]) if q[d] > 0 else float(p[d] > 0)
            if weights is None:
                if float(accept_u[draft + j]) < probs[draft + j]:
                    tokens[s, j] = d
                    accepted[s] += 1
                else:
                    weights = np.maximum(p - q, 0.0)
                    if not weights.sum() > 0:
                        weights = p
        if n > 0:
            if weights is None:
                weights = distribution(logits[row + n - 1], temperature[s])
            tokens[s, accepted[s]] = draw(weights, float(sample_u[s]))
        row, draft = row + n, draft + max(n - 1, 0)
    return tokens, accepted, probs
