"""The embedding-table operators in 64-bit numpy, from their definitions (vectordb_amd/rows.py)."""
import numpy as np


def bf16_round(x):
    """float64 -> the nearest bfloat16 value (halves to even), through float32: exact here, since a float32 quotient by 7
    never lands on the middle of two bfloat16 values unless the true quotient does."""
    u = np.asarray(x, dtype=np.float64).astype(np.float32).view(np.uint32)
    return (((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)


def encode(x, group):
    """(codes int [n, dim], scales float32 [n, groups] holding bfloat16 values, values float64 [n, dim], sqnorm float64 [n])."""
    x = np.asarray(x, dtype=np.float64)
    n, dim = x.shape
    groups = -(-dim // group)
    codes, scales = np.zeros((n, dim), dtype=np.int64), np.zeros((n, groups), dtype=np.float32)
    values, sq = np.zeros((n, dim)), np.zeros(n)
    for g in range(groups):
        part = x[:, g * group:(g + 1) * group]
        bad = ~np.isfinite(part).all(axis=1)
        s = bf16_round(np.where(bad, 0.0, np.abs(np.where(np.isfinite(part), part, 0.0)).max(axis=1)) / 7.0)
        sd = s.astype(np.float64)[:, None]
        with np.errstate(divide="ignore", invalid="ignore"):
            c = np.where((sd > 0) & ~bad[:, None], np.clip(np.rint(part / sd), -7, 7), 0.0)  # np.rint: halves to even
        s = np.where(bad, np.float32(np.nan), s)
        codes[:, g * group:(g + 1) * group] = c.astype(np.int64)
        scales[:, g] = s
        values[:, g * group:(g + 1) * group] = c * s.astype(np.float64)[:, None]
        sq += (s.astype(np.float64) ** 2) * (c * c).sum(1)
    return codes, scales, values, sq


def distances(values, q, metric):
    """float64 [nq, n]."""
    v, q = np.asarray(values, dtype=np.float64), np.asarray(q, dtype=np.float64)
    p = q @ v.T
    if metric == "dot":
        return -p
    vv, qq = (v * v).sum(1), (q * q).sum(1)
    if metric == "cosine":
        with np.errstate(divide="ignore", invalid="ignore"):
            return 1.0 - p / np.sqrt(qq[:, None] * vv[None, :])
    return np.maximum(qq[:, None] + vv[None, :] - 2.0 * p, 0.0)


def distance_tolerance(values, q, d, metric):
    """How far a returned float32 may be from float64 `d`. Rounding once: half a unit in the last place, 2^-24 |d|. The
    query's fixed point: each component off by at most half of 2^(e - 30) with max|q| >= 2^(e - 1), so by 2^-30 max|q|,
    which moves the product by 2^-30 max|q| sum|v|. The float64 sums (here and there) have fewer than 4096 terms each:
    4096 * 2^-53 of the terms' magnitudes, twice."""
    v, q = np.asarray(values, dtype=np.float64), np.asarray(q, dtype=np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        fixed = 2.0 ** -30 * np.abs(q).max(axis=1)[:, None] * np.abs(v).sum(1)[None, :]
        mag = np.abs(q) @ np.abs(v).T
        vv, qq = (v * v).sum(1)[None, :], (q * q).sum(1)[:, None]
        if metric == "cosine":
            scale = 1.0 / np.sqrt(vv * qq)
            extra = 1.0 + mag * scale
        elif metric == "l2":
            scale, extra = 2.0, vv + qq + 2 * mag
        else:
            scale, extra = 1.0, mag
        return 2.0 ** -24 * np.abs(d) + fixed * scale + 2 * 4096 * 2.0 ** -53 * extra + 2.0 ** -149


def lookup(values, ids, scale):
    n = values.shape[0]
    ok = (ids >= 0) & (ids < n)
    return np.where(ok[..., None], np.asarray(values, dtype=np.float64)[np.where(ok, ids, 0)], 0.0) * scale


def grad(g, ids, n, scale):
    """(gradient float64 [n, dim], sum of magnitudes, ids per row)."""
    g = np.asarray(g, dtype=np.float64).reshape(-1, g.shape[-1])
    ids = np.asarray(ids).reshape(-1)
    ok = (ids >= 0) & (ids < n)
    out, mag = np.zeros((n, g.shape[1])), np.zeros((n, g.shape[1]))
    np.add.at(out, ids[ok], g[ok])
    np.add.at(mag, ids[ok], np.abs(g[ok]))
    return out * scale, mag * abs(scale), np.bincount(ids[ok], minlength=n)
