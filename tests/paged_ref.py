"""Plain 64-bit forms of the per-head norm with rotation and of attention over a paged cache, from
their definitions (include/beacon_cuda.h), for the tests."""
from __future__ import annotations

import numpy as np


def table64(positions, rot, theta=10000.0):
    i = np.arange(rot // 2)
    a = np.arange(positions)[:, None] * theta ** (-2.0 * i / rot)
    return np.concatenate([np.cos(a), np.sin(a)], axis=1)


def pair_index(rot, interleaved):
    i = np.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def norm_rope(x, gain, table, pos, interleaved, eps=1e-5):
    """x [T, heads, D], pos [T] -> y [T, heads, D] (all float64); gain / table may be None."""
    z = np.array(x, dtype=np.float64)
    if gain is not None:
        z = z / np.sqrt((z * z).mean(-1, keepdims=True) + eps) * gain
    if table is None:
        return z
    rot = table.shape[1]
    a, b = pair_index(rot, interleaved)
    c, s = table[pos][:, None, :rot // 2], table[pos][:, None, rot // 2:]
    y = z.copy()
    y[..., a] = z[..., a] * c - z[..., b] * s
    y[..., b] = z[..., b] * c + z[..., a] * s
    return y


def norm_rope_bwd(dy, x, gain, table, pos, interleaved, eps=1e-5):
    """(dx, dgain) for dy, x [T, heads, D]; dgain None without a gain."""
    dz = np.array(dy, dtype=np.float64)
    if table is not None:
        rot = table.shape[1]
        a, b = pair_index(rot, interleaved)
        c, s = table[pos][:, None, :rot // 2], table[pos][:, None, rot // 2:]
        da, db = dz[..., a] * c + dz[..., b] * s, dz[..., b] * c - dz[..., a] * s
        dz[..., a], dz[..., b] = da, db
    if gain is None:
        return dz, None
    x = np.asarray(x, dtype=np.float64)
    r = np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    e = dz * gain
    dx = e / r - x * (e * x).sum(-1, keepdims=True) / (x.shape[-1] * r ** 3)
    return dx, (dz * x / r).sum((0, 1))


def paged_attention(q, k_cache, v_cache, page_table, q_lens, kv_lens, causal=True):
    """q [T, H, D]; caches [pages, Hkv, page, D]; -> out [T, H, D], lse [T, H] in float64.  Rows that no
    sequence owns stay NaN."""
    T, H, D = q.shape
    page, Hkv = k_cache.shape[2], k_cache.shape[1]
    g = H // Hkv
    out, lse = np.full((T, H, D), np.nan), np.full((T, H), np.nan)
    t0 = 0
    for s, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        pages = page_table[s, :-(-kv // page)]
        for h in range(H):
            k = k_cache[pages, h // g].reshape(-1, D)[:kv].astype(np.float64)
            v = v_cache[pages, h // g].reshape(-1, D)[:kv].astype(np.float64)
            for i in range(n):
                seen = max(0, min(kv, kv - n + i + 1)) if causal else kv
                if seen == 0:
                    out[t0 + i, h], lse[t0 + i, h] = 0.0, -np.inf
                    continue
                z = k[:seen] @ q[t0 + i, h].astype(np.float64) / np.sqrt(D)
                m = z.max()
                e = np.exp(z - m)
                out[t0 + i, h] = e @ v[:seen] / e.sum()
                lse[t0 + i, h] = m + np.log(e.sum())
        t0 += n
    return out, lse
