"""TEST INFRASTRUCTURE: the operators that programs name as custom calls (@b200.*), in 64 bits from their definitions, one sequence and
one head after another. Each attention also gives, beside the result, the sums of absolute values that bound its rounding errors."""
from __future__ import annotations

import numpy as np


def visible(n: int, p: int, window: int, sinks: int) -> np.ndarray:
    """Positions below n that a query at position p sees."""
    j = np.arange(n)
    see = j <= p
    return j[see & ((p - j < window) | (j < sinks))] if window else j[see]


def attend(q, k, v, scale):
    """One query [D] over keys and values [n, D]: the result, sum_j w_j |v_j|, and max_j scale sum_d |q_d k_jd|."""
    if len(k) == 0:
        return np.zeros(q.shape), np.zeros(q.shape), 0.0
    with np.errstate(all="ignore"):
        s = scale * (k @ q)
        m = s.max()
        if m == -np.inf:
            return np.zeros(q.shape), np.zeros(q.shape), 0.0
        w = np.exp(s - m)
        w = w / w.sum()
        return w @ v, w @ np.abs(v), float(scale * (np.abs(k) @ np.abs(q)).max())


def paged_attention(q, cache, table, lengths, new=None, layer=0, scale=None, window=0, sinks=0, bounds=False):
    q, cache = np.asarray(q, np.float64), np.asarray(cache[layer], np.float64)
    B, H, D = q.shape
    pages, size, KH = cache.shape[1], cache.shape[2], cache.shape[3]
    scale = D ** -0.5 if scale is None else scale
    out, mag, top = np.zeros(q.shape), np.zeros(q.shape), np.zeros((B, H, 1))
    for b in range(B):
        n = min(max(int(lengths[b]), 0), table.shape[1] * size)
        p = n if new is not None else n - 1
        js = visible(n, p, window, sinks)
        page = np.asarray(table[b], np.int64)[js // size] if len(js) else js
        js, page = js[(page >= 0) & (page < pages)], page[(page >= 0) & (page < pages)]
        k, v = cache[0][page, js % size], cache[1][page, js % size]                   # [n, KH, D]
        if new is not None:
            k, v = (np.concatenate([t, np.asarray(new[i], np.float64)[b:b + 1]]) for i, t in enumerate((k, v)))
        for h in range(H):
            out[b, h], mag[b, h], top[b, h] = attend(q[b, h], k[:, h // (H // KH)], v[:, h // (H // KH)], scale)
    return (out, mag, top) if bounds else out


def window_attention(q, k, v, lengths=None, scale=None, window=0, sinks=0, bounds=False):
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    B, T, H, D = q.shape
    KH = k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out, mag, top = np.zeros(q.shape), np.zeros(q.shape), np.zeros((B, T, H, 1))
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        for i in range(n):
            js = visible(n, i, window, sinks)
            for h in range(H):
                out[b, i, h], mag[b, i, h], top[b, i, h] = attend(q[b, i, h], k[b, js, h // (H // KH)], v[b, js, h // (H // KH)], scale)
    return (out, mag, top) if bounds else out


def token_log_probs(logits, tokens, top=0):
    """Log probabilities, entropies, normalisers, and with `top` the alternatives' log probabilities and numbers."""
    x = np.asarray(logits, np.float64)
    R, V = x.shape
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        total = np.log(np.exp(x - m).sum(1, keepdims=True))
        norm = np.where(m == -np.inf, -np.inf, m + total)[:, 0]                      # nothing left: the logarithm of zero
        logp = (x - m) - total
        p = np.exp(logp)
        entropy = -np.where(p == 0, 0.0, p * logp).sum(1)
    known = (np.asarray(tokens) >= 0) & (np.asarray(tokens) < V)
    lp = np.where(known, logp[np.arange(R), np.where(known, tokens, 0)], 0.0)
    outs = [lp, entropy, norm]
    if top:
        ids = np.argsort(-np.where(np.isnan(x), -np.inf, x) + 0.0, axis=1, kind="stable")
        ids = np.stack([np.concatenate([r[~np.isnan(x[i, r])], r[np.isnan(x[i, r])]]) for i, r in enumerate(ids)])[:, :top]
        outs += [np.take_along_axis(logp, ids, 1), ids.astype(np.int32)]
    return outs


def token_log_probs_grad(logits, tokens, d_log_prob, d_entropy, d_normalizer):
    x = np.asarray(logits, np.float64)
    R, V = x.shape
    entropy = token_log_probs(x, tokens)[1]
    with np.errstate(all="ignore"):
        logp = x - x.max(1, keepdims=True)
        logp = logp - np.log(np.exp(logp).sum(1, keepdims=True))
        p = np.exp(logp)
    dx = np.asarray(d_normalizer, np.float64)[:, None] * p
    dx -= np.asarray(d_entropy, np.float64)[:, None] * np.where(p == 0, 0.0, p * (logp + entropy[:, None]))
    for r in range(R):
        if 0 <= tokens[r] < V:
            dx[r] -= d_log_prob[r] * p[r]
            dx[r, tokens[r]] += d_log_prob[r]
    return dx


def write_pages(cache, rows, slots):
    cache = np.array(cache)
    size = cache.shape[3]
    for i, s in enumerate(slots):
        if s >= 0:
            cache[:, :, s // size, s % size] = rows[:, :, i]
    return cache


def copy_pages(cache, pairs):
    old, cache = np.array(cache), np.array(cache)
    for src, dst in pairs:
        cache[:, :, dst] = old[:, :, src]
    return cache


def run(target: str, xs, config: dict):
    """A custom call by its target: its results as 64-bit (or whole) arrays."""
    if target == "b200.paged_attention":
        return [paged_attention(*xs, **config)]
    if target == "b200.window_attention":
        return [window_attention(*xs, **config)]
    if target == "b200.token_log_probs":
        outs = token_log_probs(*xs, **config)
        return outs[:3] + [outs[2] - outs[2].astype(np.float32)] + outs[3:]
    if target == "b200.token_log_probs_grad":
        return [token_log_probs_grad(xs[0], xs[1], *xs[5:])]
    raise NotImplementedError(f"oracle: custom_call {target}")
