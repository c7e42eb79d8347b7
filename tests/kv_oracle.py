"""numpy fp64 definitions of the KV-cache operators (test infrastructure only): the 8-bit row format
and the attention of new tokens over the last keys of a cache."""

from __future__ import annotations

import numpy as np

MIN_SCALE = 2.0 ** -100


def quantise(x):
    """[..., D] -> (codes, scales [...]) of the 8-bit row format, in fp64. Rows with a non-finite
    value give codes 0 and a NaN scale."""
    x = np.asarray(x, dtype=np.float64)
    finite = np.isfinite(x).all(axis=-1)
    safe = np.where(finite[..., None], x, 0.0)
    scale = np.maximum(np.abs(safe).max(axis=-1) / 127.0, MIN_SCALE)
    codes = np.clip(np.rint(safe / scale[..., None]), -127, 127)
    return codes, np.where(finite, scale, np.nan)


def extend(q, k, v, causal: bool, scale: float):
    """q [n, H, D] are the last n tokens of a sequence with keys k, v [L, H_kv, D]: row i sees keys
    j <= L - n + i (all L when not causal). Returns o [n, H, D], lse [n, H] and what the rounding
    errors of a kernel scale with: a = sum_j p_j |v_j| [n, H, D] and the largest
    scale * sum_d |q_d k_jd| over the keys a row sees [n, H]."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    n, heads, d = q.shape
    length, heads_kv = k.shape[:2]
    group = heads // heads_kv
    qh = q.transpose(1, 0, 2).reshape(heads_kv, group, n, d)
    kh, vh = k.transpose(1, 2, 0)[:, None], v.transpose(1, 0, 2)[:, None]
    s = np.matmul(qh, kh) * scale
    size = np.matmul(np.abs(qh), np.abs(kh)) * scale
    seen = np.arange(length)[None, :] <= (np.arange(n)[:, None] + (length - n))
    if not causal:
        seen = np.ones_like(seen)
    with np.errstate(invalid="ignore", divide="ignore"):
        s = np.where(seen, s, -np.inf)
        size = np.where(seen, size, 0.0).max(axis=-1, initial=0.0)
        top = s.max(axis=-1, keepdims=True, initial=-np.inf)
        p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
        total = p.sum(axis=-1, keepdims=True)
        lse = np.where(total > 0, top + np.log(total), -np.inf)[..., 0]
        p = np.where(total > 0, p / np.where(total > 0, total, 1.0), 0.0)
    o, a = np.matmul(p, vh), np.matmul(p, np.abs(vh))

    def ragged(x):
        return x.reshape(heads, n, -1).transpose(1, 0, 2)

    return ragged(o), ragged(lse)[..., 0], ragged(a), ragged(size)[..., 0]
