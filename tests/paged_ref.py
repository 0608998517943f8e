"""A plain model of the paged cache for its tests: pages laid out from rows, and the definitions of the plan, the norm,
rotation and cache write, and the attention, row by row in 64 bits."""
import math

import numpy as np
import torch

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def half_step(kind):
    """The most that a rounding to the type is off, relative to the value."""
    return torch.finfo(DT[kind]).eps / 2


def dev(a, dtype=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(a)).to(dtype).cuda()


def plan(lens, news, T, ps, n_pages, free, n_free, table):
    """The definition of sd_op_page_plan, request by request."""
    B, table, left = len(lens), table.copy(), min(max(n_free, 0), n_pages)
    start, cu, kv, slots, pos, open_, admitted = left, [0], [], [], [], True, 0
    for b in range(B):
        o, n = int(lens[b]), int(news[b])
        have, want = (-(-o // ps), -(-(o + n) // ps)) if o >= 0 and n >= 0 else (0, 0)
        open_ = open_ and o >= 0 and n >= 0 and cu[-1] + n <= T and want - have <= left and want <= table.shape[1]
        if open_:
            admitted += 1
            for j in range(have, want):
                left -= 1
                table[b, j] = free[left]
            for p in range(o, o + n):
                page = int(table[b, p // ps])
                slots.append(page * ps + p % ps if 0 <= page < n_pages else -1)
                pos.append(p)
        cu.append(cu[-1] + (n if open_ else 0))
        kv.append(o + (n if open_ else 0))
    pad = T - len(slots)
    return dict(table=table, cu=cu, kv=kv, slots=slots + [-1] * pad, pos=pos + [0] * pad,
                status=[admitted, cu[-1], start - left, left])


class Cache:
    """K and V pages on the GPU: every element `fill` until rows are put in."""

    def __init__(self, kind, hk, hd, ps, n_pages, pstride=0, fill=math.nan):
        self.hk, self.hd, self.ps, self.n_pages = hk, hd, ps, n_pages
        self.page = hk * ps * hd
        self.pstride = pstride or self.page
        self.k, self.v = (torch.full((n_pages * self.pstride,), fill, dtype=DT[kind], device="cuda") for _ in range(2))

    def views(self):
        k = torch.as_strided(self.k, (self.n_pages, self.hk, self.ps // 32, self.hd // 32, 32, 32),
                             (self.pstride, self.ps * self.hd, 32 * self.hd, 1024, 32, 1))
        v = torch.as_strided(self.v, (self.n_pages, self.hk, self.ps // 32, self.hd, 32),
                             (self.pstride, self.ps * self.hd, 32 * self.hd, 32, 1))
        return k, v

    def put(self, slots, k, v):
        """k, v [rows][hk][hd] into the slots."""
        s = torch.as_tensor(slots, device="cuda").long()
        kv, vv = self.views()
        kv[s // self.ps, :, s % self.ps // 32, :, s % 32] = k.view(len(s), self.hk, self.hd // 32, 32)
        vv[s // self.ps, :, s % self.ps // 32, :, s % 32] = v

    def rows(self, slots):
        s = torch.as_tensor(slots, device="cuda").long()
        kv, vv = self.views()
        return (kv[s // self.ps, :, s % self.ps // 32, :, s % 32].reshape(len(s), self.hk, self.hd),
                vv[s // self.ps, :, s % self.ps // 32, :, s % 32])


def tables(rng, kv, ps, spare=2, width=None):
    """Random pages for requests of kv rows: (table, n_pages), entries behind a request's pages out of range."""
    need = [-(-n // ps) for n in kv]
    pages = rng.permutation(sum(need) + spare)
    table = np.full((len(kv), width or max(max(need), 1)), -7, np.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pages[at:at + n]
        at += n
    return table, sum(need) + spare


def slots_of(table, b, ps, first, last):
    p = np.arange(first, last)
    return table[b, p // ps] * ps + p % ps


def norm_rotate(x, w, rope, rd, pos, axis):
    """[rows][heads][hd] f64: the result, and the sum of the magnitudes that it is made of."""
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    if rd == 0:
        return x, x.abs()
    j = torch.arange(rd // 2, device=x.device)
    at = pos[axis.long()[j]].T.clamp(0, rope.shape[0] - 1)  # [rows][rd / 2]
    cs = rope[at.long(), j].double()[:, None]
    c, s = cs[..., 0], cs[..., 1]
    lo, hi = x[..., :rd // 2], x[..., rd // 2:rd]
    y = torch.cat([lo * c - hi * s, hi * c + lo * s, x[..., rd:]], -1)
    return y, torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs(), x[..., rd:].abs()], -1)


def attend(q, k, v, kv_len, scale, window=0, gate=None, holes=()):
    """q [n][hq][hd], k, v [kv][hk][hd] (f64) of one request, the last n of the kv_len rows the queries' own (k and v
    may be shorter or longer than kv_len: rows past them are not there).  Each row sees its keys alone: others' values
    never enter.  -> out, the mean magnitude of the values by the same weights, the largest sum of magnitudes of a score."""
    n, hq, hd = q.shape
    g = hq // k.shape[1]
    out, mag, top = torch.zeros_like(q), torch.zeros_like(q), 0.0
    hole = torch.zeros(len(k), dtype=torch.bool, device=q.device)
    for a, b in holes:
        hole[a:b] = True
    for i in range(n):
        p = kv_len - n + i
        lo, hi = max(0, p - window + 1) if window else 0, min(p + 1, len(k))
        if hi <= lo:
            continue
        keep = ~hole[lo:hi]
        if not keep.any():
            continue
        ki, vi = k[lo:hi][keep], v[lo:hi][keep]
        for kh in range(k.shape[1]):
            x, kk, vv = q[i, kh * g:(kh + 1) * g], ki[:, kh], vi[:, kh]
            s = x @ kk.T * scale
            w = torch.softmax(s, -1)
            w[(s == -math.inf).all(-1)] = 0
            out[i, kh * g:(kh + 1) * g] = w @ vv
            mag[i, kh * g:(kh + 1) * g] = w @ vv.abs()
            xf, kf = (t.nan_to_num(0.0, 0.0, 0.0).abs() for t in (x, kk))
            top = max(top, float((xf @ kf.T).max()) * scale)
    if gate is not None:
        out, mag = out * torch.sigmoid(gate), mag * torch.sigmoid(gate)
    return out, mag, top


def attend_fast(q, k, v, kv_len, scale, window=0, gate=None):
    """attend() for finite values and many rows: masked products, 256 rows at a time."""
    n, hq, hd = q.shape
    hk, g = k.shape[1], hq // k.shape[1]
    out, mag, top = torch.zeros_like(q), torch.zeros_like(q), 0.0
    j = torch.arange(len(k), device=q.device)
    for kh in range(hk):
        for a in range(0, n, 256):
            b = min(n, a + 256)
            p = torch.arange(kv_len - n + a, kv_len - n + b, device=q.device)[:, None]
            see = (j <= p) & (j > p - window) if window else j <= p
            x = q[a:b, kh * g:(kh + 1) * g].reshape(-1, hd)
            s = (x @ k[:, kh].T * scale).view(b - a, g, -1).masked_fill(~see[:, None], -math.inf)
            w = torch.softmax(s, -1).nan_to_num(0.0).view(-1, len(k))
            out[a:b, kh * g:(kh + 1) * g] = (w @ v[:, kh]).view(b - a, g, hd)
            mag[a:b, kh * g:(kh + 1) * g] = (w @ v[:, kh].abs()).view(b - a, g, hd)
            top = max(top, float((x.abs() @ k[:, kh].abs().T).max()) * scale)
    if gate is not None:
        out, mag = out * torch.sigmoid(gate), mag * torch.sigmoid(gate)
    return out, mag, top


def attend_bound(kind, want, mag, top, hd, kv):
    """How far a right result may be off, element by element.  u: half a step of the type, e: of f32.  The result is
    rounded to the type (u |out|), the weights are (u of the weighted magnitudes); a score is a sum of hd products in
    f32 (at most hd e of the sum of magnitudes `top`, which moves weights and their sum by that much each), its
    exponential's argument is rounded where its magnitude is at most 2 top (2 e top log2(e) ln(2), twice), the
    exponential is within 2 e, and sums over the keys are in f32 (kv e each for the weights and the products).  The
    factors of splits, gate and division are a few e more (16)."""
    u, e = half_step(kind), 2.0 ** -24
    rel = u + 2 * hd * e * top + 4 * e * top + 2 * kv * e + 16 * e
    return u * want.abs() + rel * mag * (1 + u) + 2.0 ** -25
