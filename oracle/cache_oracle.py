"""The 8-bit cache, the attention over it and the adjustment of logits in 64 bits, on the CPU: plain numpy, one row or one block
at a time where the definition is."""
from __future__ import annotations

import numpy as np


def _e4m3_values():
    """Value of every code: sign, 4 exponent bits with bias 7 (0: steps of 2^-9), 3 fraction bits; 0x7f and 0xff are no numbers."""
    out = np.zeros(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        v = f * 2.0 ** -9 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        out[c] = (-1 if c & 128 else 1) * (np.nan if c & 127 == 127 else v)
    return out


E4M3 = _e4m3_values()
_POSITIVE = E4M3[:127]                       # 0 .. 448, in the order of the codes


def e4m3_codes(y):
    """Codes of the nearest numbers, ties to the even code, clamped to +-448; NaN to 0x7f."""
    y = np.asarray(y, np.float64)
    a = np.minimum(np.abs(np.nan_to_num(y, nan=0.0, posinf=448.0, neginf=-448.0)), 448.0)
    hi = np.clip(np.searchsorted(_POSITIVE, a), 1, 126)
    lo = hi - 1
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo) | np.where(np.signbit(y), 128, 0)
    return np.where(np.isnan(y), 127, code).astype(np.uint8)


def block_scale(amax):
    e = -64
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def store(key, value, k, v, scales, slots, src=None):
    """key, value [n, H, D] (float64), k [nb, H, bs, D] and v [nb, H, D, bs] (uint8 codes), scales [nb, H, 2]: changed in place."""
    nb, H, bs, D = k.shape
    rows = {}                                 # block -> {token: row}; the later of two wins
    for i, slot in enumerate(slots):
        r = i if src is None else src[i]
        if 0 <= slot < nb * bs and 0 <= r < len(key):
            rows.setdefault(slot // bs, {})[slot % bs] = r
    for b, tokens in rows.items():
        at, which = list(tokens), list(tokens.values())
        for x, c, w in ((key, k[b], 0), (value, v[b].transpose(0, 2, 1), 1)):     # c: [H, bs, D], a view
            for h in range(H):
                new = x[which, h]
                finite = np.abs(new[np.isfinite(new)])
                s = block_scale(finite.max() if finite.size else 0.0)
                if 0 not in tokens:
                    old = scales[b, h, w]
                    s = max(s, old)
                    if s != old:
                        c[h] = e4m3_codes(E4M3[c[h]] * (old / s)) if old else 0
                c[h, at] = e4m3_codes(new / s)
                scales[b, h, w] = s


def gathered(k, v, scales, table, L):
    """(K, V) [H, L, D] of a sequence, as the values that the cache stands for."""
    nb, H, bs, D = k.shape
    n = -(-L // bs)
    blocks = [b if 0 <= b < nb else 0 for b in list(table[:n]) + [0] * max(0, n - len(table))]
    s = scales[blocks]                        # [n, H, 2]
    kk = (E4M3[k[blocks]] * s[..., 0][:, :, None, None]).transpose(1, 0, 2, 3).reshape(H, -1, D)[:, :L]
    vv = (E4M3[v[blocks]] * s[..., 1][:, :, None, None]).transpose(1, 0, 3, 2).reshape(H, -1, D)[:, :L]
    return kk, vv


def attend(q, k, v, scales, tables, lens, q_lens, scale):
    """q [n, Hq, D]: (out, sum of p |v|, the largest sum of |q k| scale of a row), the latter two for error bounds."""
    H, D = k.shape[1], k.shape[3]
    G = q.shape[1] // H
    out, mag, top = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    row = 0
    for i, (L, ql) in enumerate(zip(lens, q_lens)):
        kk, vv = gathered(k, v, scales, tables[i], L)
        for j in range(ql):
            seen = L - ql + j + 1
            if seen > 0:
                for h in range(H):
                    x = q[row + j, h * G:(h + 1) * G] @ kk[h, :seen].T * scale
                    p = np.exp(x - x.max(1, keepdims=True))
                    p /= p.sum(1, keepdims=True)
                    out[row + j, h * G:(h + 1) * G] = p @ vv[h, :seen]
                    mag[row + j, h * G:(h + 1) * G] = p @ np.abs(vv[h, :seen])
                    top[row + j, h * G:(h + 1) * G] = (np.abs(q[row + j, h * G:(h + 1) * G]) @ np.abs(kk[h, :seen]).T * scale).max(1)
        row += ql
    return out, mag, top


def adjust(logits, q_lens, tokens=None, token_lens=None, prompt_lens=None, drafts=None, repetition=None, frequency=None, presence=None,
           bias=None, mask=None, mask_rows=None):
    """logits [n, V] (float64); tokens: a list per sequence; repetition, frequency, presence [S]; bias: a list of (token, value) per
    sequence.  (the result, the largest magnitude on the way)."""
    x = np.array(logits, np.float64)
    mag = np.abs(np.where(np.isfinite(x), x, 0.0))
    V, row, draft = x.shape[1], 0, 0
    for s, n in enumerate(q_lens):
        told = [] if tokens is None else list(tokens[s][:None if token_lens is None else token_lens[s]])
        prompt = 0 if prompt_lens is None else min(prompt_lens[s], len(told))
        for j in range(n):
            so_far = told + ([] if drafts is None else list(drafts[draft:draft + j]))
            count, seen = np.zeros(V), np.zeros(V, bool)
            for i, t in enumerate(so_far):
                if 0 <= t < V:
                    seen[t] = True
                    count[t] += i >= prompt
            r, y = repetition[s], x[row + j]
            y = np.where(seen, np.where(y > 0, y / r, y * r), y)
            mag[row + j] = np.maximum(mag[row + j], np.abs(np.where(np.isfinite(y), y, 0)))
            less = frequency[s] * count + presence[s] * (count > 0)
            y = y - less
            add = np.zeros(V)
            for t, b in ([] if bias is None else bias[s]):
                if 0 <= t < V:
                    add[t] = b
            y = y + add
            mag[row + j] += np.abs(less) + np.abs(add)
            m = -1 if mask is None else row + j if mask_rows is None else mask_rows[row + j]
            if mask is not None and 0 <= m < len(mask):
                words = np.asarray(mask[m]).astype(np.int64) & 0xffffffff
                t = np.arange(V)
                y = np.where((words[t // 32] >> (t % 32)) & 1, y, -np.inf)
            x[row + j] = y
        row, draft = row + n, draft + max(n - 1, 0)
    return x, mag
