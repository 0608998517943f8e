"""Plain definitions of the rotary positions and of the rows that leave the paged cache, in 64 bits, row by row."""
import math

import numpy as np
import torch

E32 = 2.0 ** -24  # half a step of f32, relative


def freqs(rd, theta, scaling="plain", factor=1.0, length=0.0, low=0.0, high=0.0):
    out = []
    for j in range(rd // 2):
        f = (theta * factor ** (rd / (rd - 2)) if scaling == "base" else theta) ** (-2 * j / rd)
        if scaling == "linear":
            f /= factor
        if scaling == "parts":
            k = min(1.0, max(0.0, (length * f / (2 * math.pi) - low) / (high - low)))
            f = k * f + (1 - k) * f / factor
        out.append(f)
    return np.array(out)


def rope(x, pos, f, magnitude, layout, inverse):
    """x [rows][heads][hd] f64 (CPU) -> the turned rows, and the sum of the magnitudes that each element is made of."""
    rd = 2 * len(f)
    a = torch.from_numpy(np.outer(np.asarray(pos, np.float64), f))[:, None] * (-1 if inverse else 1)
    c, s = magnitude * a.cos(), magnitude * a.sin()
    j = torch.arange(rd // 2)
    i0, i1 = (j, j + rd // 2) if layout == "half" else (2 * j, 2 * j + 1)
    y, mag = x.clone(), x.abs()
    u, v = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = u * c - v * s, v * c + u * s
    mag[..., i0], mag[..., i1] = (u * c).abs() + (v * s).abs(), (v * c).abs() + (u * s).abs()
    return y, mag


def weights(q, k, kv_len, scale, window=0, observers=0, holes=(), decay=0.0, old=None):
    """q [n][hq][hd], k [>= kv_len][hk][hd] (f64, CPU) of one request, the last n of its kv_len rows the queries' own.
    -> [hk][kv_len] the weight that every key receives, NaN where a row that sees it has one, and the largest sum of
    magnitudes of a score.  Each row sees its keys alone: others' values never enter."""
    n, hq, hd = q.shape
    hk, g, top = k.shape[1], hq // k.shape[1], 0.0
    out = torch.zeros(hk, kv_len, dtype=torch.float64)
    hole = torch.zeros(kv_len, dtype=torch.bool)
    for a, b in holes:
        hole[a:b] = True
    for i in range(max(0, n - observers) if observers else 0, n):
        p = kv_len - n + i
        lo = max(0, p - window + 1) if window else 0
        j = torch.arange(lo, p + 1)
        j = j[~hole[lo:p + 1]]
        if not len(j):
            continue
        for h in range(hk):
            x, kk = q[i, h * g:(h + 1) * g], k[j, h]
            s = x @ kk.T * scale
            w = torch.softmax(s, -1)
            w[(s == -math.inf).all(-1)] = 0
            out[h, j] += w.sum(0)
            xf, kf = (t.nan_to_num(0.0, 0.0, 0.0).abs() for t in (x, kk))
            top = max(top, float((xf @ kf.T).max()) * scale)
    if decay:
        out[:, :kv_len - n] += decay * old[:, :kv_len - n]
    return out, top


def weights_bound(want, top, hd, kv, rows):
    """How far a right result may be off.  A score is a sum of hd products in f32 (at most hd E32 of the sum of magnitudes
    `top`, which moves a weight and the sum that divides it by that much each), is turned into base 2 and has its maximum
    taken off (two roundings of at most 2 top each in numerator and sum), goes through an exponential within 2 E32; sums over kv
    keys and then over the rows are in f32, at most E32 per addend; division, the joins of splits, decay and rounding are a few
    E32 more (16)."""
    rel = (2 * hd * top + 8 * top + 2 * kv + rows + 16) * E32
    return rel * want.abs() + 2.0 ** -126


def evict(scores, kpos, n, budget, sink, recent, hole=None):
    """One head: scores [n], kpos [n] -> moves [(place, row)], by a sort."""
    m = budget
    key = []
    there = [not (hole is not None and hole[j]) for j in range(n)]
    newest = max([int(kpos[j]) for j in range(n) if there[j]], default=-(2 ** 31))
    for j in range(n):
        s = float(scores[j])
        if not there[j]:
            key.append((0, 0.0, j))
        elif kpos[j] < sink or kpos[j] > newest - recent:
            key.append((-2, 0.0, j))
        else:
            key.append((0, 0.0, j) if math.isnan(s) else (-2, 0.0, j) if s == math.inf else (-1, -s, j))
    stay = sorted(x[2] for x in sorted(key)[:m])
    kept = set(stay)
    return list(zip([j for j in range(m) if j not in kept], [j for j in stay if j >= m]))


def release(kv, new, dropped, table, ps, n_pages, free, n_free):
    free, left, out = list(free), min(max(n_free, 0), n_pages), []
    for b, (n, m) in enumerate(zip(kv, new)):
        cut = 0 <= m < n
        out.append(dropped[b] + (n - m if cut else 0))
        if cut:
            for i in range(-(-m // ps), min(-(-n // ps), len(table[b]))):
                if 0 <= table[b][i] < n_pages and left < n_pages:
                    free[left] = table[b][i]
                    left += 1
    return out, free, left
