"""Draft verification in numpy and 64 bits: the definitions the CUDA
operators implement, one request and one row at a time."""

from __future__ import annotations

import numpy as np


def row_probs(row, t: float, k: int = 0, p: float = 1.0) -> np.ndarray:
    """Target probabilities (float64) of one logits row: softmax(l / t) over
    what top-k (k <= 0 or >= V: off) and top-p (not < 1: off) keep; t not
    > 0: one-hot at the first largest token; no finite or +inf entry: zeros.
    NaN reads as -inf."""
    x = np.asarray(row, dtype=np.float64).copy()
    x[np.isnan(x)] = -np.inf
    x += 0.0
    v = x.size
    out = np.zeros(v)
    m = x.max()
    if m == -np.inf:
        return out
    if not t > 0:
        out[int(np.argmax(x))] = 1.0
        return out
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x - m) / np.float64(t))
    w[x == -np.inf] = 0.0
    if m == np.inf:
        w[:] = 0.0
    w[x == m] = 1.0
    low = -np.inf
    if 0 < k < v:
        low = np.sort(x)[v - k]
    kept = x >= low
    if p < 1:
        if p > 0:
            need = np.float64(p) * w[kept].sum()
            for val in np.unique(x[kept])[::-1]:
                if w[x >= val].sum() >= need:
                    break
            low = max(low, val)
        else:
            low = m
        kept = x >= low
    w[~kept] = 0.0
    return w / w.sum()


def draw(r, u: float) -> int:
    """Lowest i whose running sum exceeds u * sum(r); the last i with mass
    when none does; -1 without mass."""
    r = np.asarray(r, dtype=np.float64)
    total = r.sum()
    if not total > 0:
        return -1
    over = np.nonzero(np.cumsum(r) > u * total)[0]
    return int(over[0]) if over.size else int(np.nonzero(r)[0][-1])


def verify_rows(probs_of, v: int, draft, num_valid, uniforms,
                draft_probs=None):
    """probs_of(b, j) -> row probabilities (float64, [v]) or None; draft
    [B, K]; num_valid [B] or None; uniforms [B, K + 1]. Returns (sampled
    [B, K + 1], count [B]) int32."""
    draft = np.asarray(draft)
    b, k = draft.shape
    sampled = np.full((b, k + 1), -1, dtype=np.int32)
    count = np.zeros(b, dtype=np.int32)
    for i in range(b):
        n = k if num_valid is None else min(int(num_valid[i]), k)
        if n < 0:
            continue
        s = 0
        while s < n:
            x = int(draft[i, s])
            p = probs_of(i, s)
            q = 1.0
            if p is None or not 0 <= x < v:
                break
            if draft_probs is not None:
                q = float(_clean(draft_probs[i, s])[x])
            if not float(uniforms[i, s]) * q < p[x]:
                break
            s += 1
        p = probs_of(i, s)
        tok = -1
        if p is not None:
            r = p.copy()
            if s < n and draft_probs is not None:
                r = np.maximum(p - _clean(draft_probs[i, s]), 0.0)
            elif s < n and 0 <= int(draft[i, s]) < v:
                r[int(draft[i, s])] = 0.0
            tok = draw(r, float(uniforms[i, k]))
            if tok < 0:
                tok = draw(p, float(uniforms[i, k]))
        sampled[i, :s] = draft[i, :s]
        sampled[i, s] = tok
        count[i] = s + (tok >= 0)
    return sampled, count


def _clean(p) -> np.ndarray:
    p = np.asarray(p, dtype=np.float64)
    return np.where((p > 0) & np.isfinite(p), p, 0.0)


def _row(rows, row_start, i, j):
    if row_start is None:
        return rows[i, j]
    at = int(row_start[i]) + j
    return rows[at] if 0 <= at < len(rows) else None


def verify_sampled(logits, draft, uniforms, num_valid=None, temperature=1.0,
                   top_k=0, top_p=1.0, row_start=None):
    """logits: float array [B, K + 1, V], or [N, V] with row_start. Settings
    are numbers or [B] arrays."""
    b = np.asarray(draft).shape[0]
    t, k, p = (np.broadcast_to(np.asarray(x), (b,))
               for x in (temperature, top_k, top_p))

    def probs_of(i, j):
        row = _row(logits, row_start, i, j)
        return None if row is None else row_probs(row, float(t[i]),
                                                  int(k[i]), float(p[i]))
    return verify_rows(probs_of, logits.shape[-1], draft, num_valid, uniforms)


def verify_greedy(logits, draft, num_valid=None, row_start=None):
    b, k = np.asarray(draft).shape
    return verify_sampled(logits, draft, np.zeros((b, k + 1)), num_valid,
                          0.0, 0, 1.0, row_start)


def verify_probs(probs, draft, uniforms, num_valid=None, draft_probs=None,
                 row_start=None):
    def probs_of(i, j):
        row = _row(probs, row_start, i, j)
        return None if row is None else _clean(row)
    return verify_rows(probs_of, probs.shape[-1], draft, num_valid, uniforms,
                       draft_probs)
