"""Plain 64-bit restatements of the distillation operators (numpy; test infrastructure).

Written from the definitions: sorting for the top logits, dense distributions for the
loss and its gradient, one sequence at a time for the verification of drafts.
"""

from __future__ import annotations

import numpy as np


def top_logits(logits, k, temperature=1.0):
    """(values, indices, lse) of fp32/fp64 rows; NaN first, then falling, ties by index."""
    z = np.asarray(logits, dtype=np.float64)
    rows, vocab = z.shape
    indices = np.empty((rows, k), dtype=np.int64)
    lse = np.empty(rows)
    for i, row in enumerate(z):
        falling = np.where(np.isnan(row), -np.inf, -row)
        order = np.lexsort((np.arange(vocab), falling, ~np.isnan(row)))
        indices[i] = order[:k]
        top = row[order[0]]
        if np.isnan(top) or np.isinf(top):
            lse[i] = top
        else:
            lse[i] = top / temperature + np.log(np.exp((row - top) / temperature).sum())
    return np.take_along_axis(z, indices, 1), indices, lse


def verify_drafts(target, tokens, uniforms, noise, draft=None, lens=None):
    """Accepted counts and emitted tokens; products, differences and quotients in fp32, as
    the definition has them (they decide comparisons)."""
    target = np.asarray(target, dtype=np.float32)
    batch, places, vocab = target.shape
    drafts = places - 1
    accepted = np.zeros(batch, dtype=np.int64)
    out = np.full((batch, places), -1, dtype=np.int64)
    for b in range(batch):
        length = drafts if lens is None else int(np.clip(lens[b], 0, drafts))
        n = 0
        while n < length:
            x = int(tokens[b, n])
            if not 0 <= x < vocab:
                break
            q = np.float32(1) if draft is None else np.float32(draft[b, n, x])
            if not np.float32(uniforms[b, n]) * q < target[b, n, x]:
                break
            n += 1
        p = target[b, n]
        r = p.copy()
        if n < length:
            if draft is None:
                if 0 <= tokens[b, n] < vocab:
                    r[tokens[b, n]] = 0
            else:
                r = p - np.asarray(draft[b, n], dtype=np.float32)
            if not (r > 0).any():
                r = p
        with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
            score = np.where(r > 0, r / np.asarray(noise[b], dtype=np.float32), np.float32(0))
        score = np.where(np.isnan(score), np.float32(0), score)
        accepted[b] = n
        out[b, :n] = tokens[b, :n]
        if score.max() > 0:
            out[b, n] = int(score.argmax())
    return accepted, out


def distillation(hidden, weight, indices, logits, lse=None, temperature=1.0, upstream=None):
    """(loss, mass, dhidden, spread) of KL(teacher || student) in 64 bits; the last two are
    None without `upstream`.  spread bounds dhidden's terms: sum_v |dz_v| |W_v| |upstream| / tau.

    The teacher's distribution: its listed tokens and, with `lse`, one bucket of all
    others; the student's: softmax(hidden . weight^T / temperature), its unlisted tokens
    in one bucket.  Rows without a listed token give zeros."""
    x = np.asarray(hidden, dtype=np.float64)
    w = np.asarray(weight, dtype=np.float64)
    wa = np.abs(w)
    rows, vocab = x.shape[0], w.shape[0]
    loss, mass = np.zeros(rows), np.zeros(rows)
    grad = None if upstream is None else np.zeros_like(x)
    spread = None if upstream is None else np.zeros_like(x)
    for i in range(rows):
        used = indices[i] >= 0
        cols = indices[i][used]
        t = np.asarray(logits[i], dtype=np.float64)[used] / temperature
        if not len(cols) or (lse is None and not (t > -np.inf).any()) or (lse is not None and lse[i] == -np.inf):
            continue
        if lse is None:
            p = np.exp(t - t.max())
            p /= p.sum()
            rest = 0.0
        else:
            p = np.exp(t - np.float64(lse[i]))
            rest = max(0.0, 1.0 - p.sum()) if len(cols) < vocab else 0.0
        z = w @ x[i] / temperature
        z -= z.max()
        logq = z - np.log(np.exp(z).sum())
        q = np.exp(logq)
        others = np.ones(vocab, dtype=bool)
        others[cols] = False
        loss[i] = (p[p > 0] * (np.log(p[p > 0]) - logq[cols][p > 0])).sum()
        mass[i] = q[cols].sum()
        dz = q.copy()
        np.subtract.at(dz, cols, p)
        if rest > 0:
            m = z[others].max()
            log_rest = m + np.log(np.exp(z[others] - m).sum()) + (logq[0] - z[0])
            loss[i] += rest * (np.log(rest) - log_rest)
            dz[others] -= rest * np.exp(logq[others] - log_rest)
        if upstream is not None:
            grad[i] = (dz @ w) * (upstream[i] / temperature)
            spread[i] = (np.abs(dz) @ wa) * abs(upstream[i] / temperature)
    return loss, mass, grad, spread
