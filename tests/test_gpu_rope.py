"""Rotary positions against their definition in 64 bits: tables at any position, both layouts, parts of heads, in place and
into other rows, at strides and orders, and the positions of requests that have dropped cached rows."""
import math

import numpy as np
import pytest
import torch

import evict_ref as er
import paged_ref as pr

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
KIND = {"f16": 0, "bf16": 1, "f32": 2}


def freqs_on(f):
    return torch.from_numpy(np.ascontiguousarray(f)).cuda()


def angle_slack(f, pos):
    """p f / 2 pi in f64: four roundings (2^-53 each of the angle), the definition's own one; the two series to 2^-36."""
    return np.abs(np.outer(np.asarray(pos, np.float64), f)) * 5 * 2.0 ** -53 + 2.0 ** -36


POS = [0, 1, -1, 2, 7, 100, 4095, 16384, 65535, -70000, 1000003, 3000000, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31]


@pytest.mark.parametrize("rd,theta,kw,magnitude", [
    (64, 1e7, {}, 1.0), (2, 1e4, {}, 1.0), (256, 1e6, dict(scaling="linear", factor=8.0), 0.5), (24, 1e4, dict(scaling="base", factor=4.0), 1.0),
    (128, 5e5, dict(scaling="parts", factor=8.0, length=8192.0, low=1.0, high=4.0), 1.2079), (6, 1.0, {}, -1.0)])
def test_table(sdamd, rd, theta, kw, magnitude):
    f = sdamd.rope_freqs(rd, theta, **{**kw, "scaling": dict(plain=0, linear=1, base=2, parts=3)[kw.get("scaling", "plain")]})
    fd = freqs_on(f)
    for pos in (POS, None, [5]):
        n = 777 if pos is None else len(pos)
        out = torch.full((n * rd // 2 + 1, 2), 7.0, device="cuda")
        pd = pr.dev(pos or [0])
        sdamd.op_rope_table(fd.data_ptr(), rd // 2, None if pos is None else pd.data_ptr(), n, out.data_ptr(), magnitude=magnitude)
        p = np.arange(n) if pos is None else np.array(pos)
        a = np.outer(p.astype(np.float64), f)
        want = np.stack([magnitude * np.cos(a), magnitude * np.sin(a)], -1)
        got = out[:-1].cpu().double().numpy().reshape(want.shape)
        bound = er.E32 * np.abs(want) + abs(magnitude) * angle_slack(f, p)[..., None]
        assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) - bound)
        assert (out[-1] == 7).all()


def check_rows(got, want, mag, f, pos, kind, magnitude):
    """The table's rounding (E32 of each product), two roundings of products and sum in f32, the angle's own, one to the type."""
    rd2 = len(f)
    slack = torch.from_numpy(angle_slack(f, pos)).max(-1).values[:, None, None] * abs(magnitude)
    u = torch.finfo(DT[kind]).eps / 2
    bound = u * want.abs() * (1 + u) + (4 * er.E32 + slack / max(abs(magnitude), 1e-3) * 2) * mag * (1 + u) + 2.0 ** -25
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    assert (err <= bound).all(), float((err - bound).max())


CASES = [  # t, hq, hk, hd, rd, layout, type
    (1, 1, 0, 8, 2, "half", "f16"), (1, 8, 2, 256, 64, "half", "f16"), (3, 32, 8, 128, 128, "pairs", "bf16"), (64, 32, 8, 128, 128, "half", "bf16"),
    (5, 4, 1, 64, 24, "half", "f32"), (7, 4, 1, 64, 24, "pairs", "f16"), (6, 3, 3, 64, 20, "pairs", "bf16"), (6, 3, 3, 64, 20, "half", "f16"),
    (300, 28, 4, 128, 64, "half", "f32"), (257, 12, 1, 64, 64, "pairs", "f32"), (2, 2, 2, 1024, 256, "half", "bf16"), (1, 1024, 1, 8, 8, "pairs", "f16"),
    (2049, 8, 2, 256, 64, "pairs", "f16"), (1500, 32, 8, 128, 128, "half", "f16"), (4, 2, 0, 80, 80, "half", "bf16"), (9, 5, 1, 40, 34, "half", "f32"),
    (9, 5, 1, 40, 34, "pairs", "f32"), (3000, 4, 4, 64, 40, "half", "bf16")]


@pytest.mark.parametrize("where", ["out", "in place", "heads outside", "gated"])
@pytest.mark.parametrize("t,hq,hk,hd,rd,layout,kind", CASES)
def test_rows(sdamd, t, hq, hk, hd, rd, layout, kind, where):
    rng = np.random.default_rng(t * 31 + hd + rd)
    f = er.freqs(rd, 1e4)
    pos = rng.integers(-1000, 200000, t)
    magnitude, inverse = (1.0, False) if t % 2 else (1.25, True)
    g = torch.Generator().manual_seed(t + hd)
    dt = DT[kind]
    per = 2 if where == "gated" else 1
    if where == "heads outside":  # [heads][rows][hd]
        q, k = torch.randn(hq, t, hd, generator=g).to(dt), torch.randn(max(hk, 1), t, hd, generator=g).to(dt)
        buf = torch.cat([q.reshape(-1), k.reshape(-1)]).cuda()
        qs, qt, ks, kt, ko = hd, t * hd, hd, t * hd, hq * t * hd
        q64, k64 = q.double().transpose(0, 1), k.double().transpose(0, 1)
    else:
        width = hq * per * hd + max(hk, 1) * hd + 8
        big = torch.randn(t, width, generator=g).to(dt)
        buf = big.cuda().reshape(-1)
        qs, qt, ks, kt, ko = width, per * hd, width, hd, hq * per * hd
        q64 = big[:, :hq * per * hd].reshape(t, hq, per * hd)[..., :hd].double()
        k64 = big[:, hq * per * hd:-8].reshape(t, -1, hd).double()
    before = buf.clone()
    size = buf.element_size()
    fd, pd = freqs_on(f), pr.dev(pos)
    inplace = where == "in place"
    qo, kk = (torch.full((t * n * hd + 8,), 3.0, dtype=dt, device="cuda") for n in (hq, max(hk, 1)))
    args = dict(magnitude=magnitude, inverse=inverse)
    if not inplace:
        args.update(Qo=qo.data_ptr(), Ko=kk.data_ptr() if hk else None)
    sdamd.op_rope(fd.data_ptr(), rd, 0 if layout == "half" else 1, pd.data_ptr(), t, hd, buf.data_ptr(), qs, qt, hq,
                  buf.data_ptr() + ko * size if hk else None, ks, kt, hk, KIND[kind], **args)
    if inplace:
        q2 = torch.as_strided(buf, (t, hq, hd), (qs, qt, 1)).cpu()
        k2 = torch.as_strided(buf, (t, max(hk, 1), hd), (ks, kt, 1), ko).cpu()
        assert torch.equal(buf.view(t, -1)[:, -8:], before.view(t, -1)[:, -8:])
    else:
        assert torch.equal(buf, before) and (qo[t * hq * hd:] == 3).all() and (kk[t * max(hk, 1) * hd:] == 3).all()
        q2, k2 = qo[:t * hq * hd].view(t, hq, hd).cpu(), kk[:t * max(hk, 1) * hd].view(t, -1, hd).cpu()
    for x, y in ((q64, q2), (k64, k2))[:2 if hk else 1]:
        want, mag = er.rope(x, pos, f, magnitude, layout, inverse)
        check_rows(y, want, mag, f, pos, kind, magnitude)
        assert torch.equal(y[..., rd:].double(), x[..., rd:])  # dims that do not turn: as they were


def test_null_positions_are_row_numbers_and_other_dims_keep_any_value(sdamd):
    t, hd, rd = 33, 64, 20
    x = torch.randn(t, 1, hd).half()
    x[:, :, rd] = math.inf
    x[:, :, rd + 1] = math.nan
    y = x.cuda()
    f = er.freqs(rd, 1e4)
    fd = freqs_on(f)
    for layout in (0, 1):
        z = y.clone()
        sdamd.op_rope(fd.data_ptr(), rd, layout, None, t, hd, z.data_ptr(), hd, hd, 1, None, 0, 0, 0, 0)
        want, _ = er.rope(x.double()[..., :rd], np.arange(t), f, 1.0, ["half", "pairs"][layout], False)
        assert (z.cpu()[..., :rd].double() - want).abs().max() < 2.0 ** -9 * 4
        assert torch.isinf(z[:, :, rd]).all() and torch.isnan(z[:, :, rd + 1]).all() and torch.equal(z[..., rd + 2:], y[..., rd + 2:])


def test_gradient(sdamd):
    """The gradient of sum(w * rope(x)) is rope of w turned back: against the definition's by differences (it is linear in x,
    so a difference of any size is exact up to rounding)."""
    t, h, hd, rd = 11, 3, 64, 48
    f = er.freqs(rd, 1e4)
    g = torch.Generator().manual_seed(4)
    pos = np.arange(t) * 37
    x, w = (torch.randn(t, h, hd, generator=g) for _ in range(2))
    fd, pd, wd = freqs_on(f), pr.dev(pos), w.cuda()
    for layout in ("half", "pairs"):
        grad = torch.zeros_like(wd)
        sdamd.op_rope(fd.data_ptr(), rd, 0 if layout == "half" else 1, pd.data_ptr(), t, hd, wd.data_ptr(), h * hd, hd, h, None, 0, 0, 0, 2,
                      magnitude=1.5, inverse=True, Qo=grad.data_ptr())
        loss = lambda x: float((w.double() * er.rope(x, pos, f, 1.5, layout, False)[0]).sum())
        for i in range(0, t * h * hd, 97):
            e = torch.zeros(t * h * hd, dtype=torch.float64)
            e[i] = 0.5
            d = loss(x.double() + e.view_as(x)) - loss(x.double() - e.view_as(x))
            assert abs(d - float(grad.view(-1)[i])) <= 8 * er.E32 * 1.5 * float(w.abs().max()) * 2 + 1e-9


def test_inverse_turns_back(sdamd):
    t, h, hd = 100, 2, 128
    f = er.freqs(hd, 1e6)
    x = torch.randn(t, h, hd, device="cuda")
    fd, pd = freqs_on(f), pr.dev(np.arange(t) * 30011)
    y = x.clone()
    for inv in (False, True):
        sdamd.op_rope(fd.data_ptr(), hd, 1, pd.data_ptr(), t, hd, y.data_ptr(), h * hd, hd, h, None, 0, 0, 0, 2, inverse=inv)
    assert float((x - y).abs().max()) <= 16 * er.E32 * 2 * float(x.abs().max())


def test_a_step_rotates_by_its_table(sdamd):
    """positions -> table -> sd_op_paged_prep with the rows' own numbers: what sd_op_rope gives for the same positions."""
    B, hq, hk, hd, rd, ps = 5, 8, 2, 128, 64, 32
    rng = np.random.default_rng(3)
    news = [1, 7, 0, 1, 30]
    T = sum(news)
    cu = np.concatenate([[0], np.cumsum(news)])
    at = np.concatenate([np.arange(n) + 100 * b for b, n in enumerate(news)])
    dropped = rng.integers(0, 10 ** 6, B)
    f = sdamd.rope_freqs(rd, 1e7, 3, 8.0, 4096.0, 1.0, 32.0)
    fd, pos = freqs_on(f), torch.zeros(T, dtype=torch.int32, device="cuda")
    d = [pr.dev(v) for v in (cu, dropped, at)]
    sdamd.op_page_positions(d[0].data_ptr(), d[1].data_ptr(), B, T, d[2].data_ptr(), pos.data_ptr())
    true = at + np.repeat(dropped, news)
    assert pos.tolist() == true.tolist()
    table = torch.zeros(T, rd // 2, 2, device="cuda")
    sdamd.op_rope_table(fd.data_ptr(), rd // 2, pos.data_ptr(), T, table.data_ptr(), magnitude=1.2)
    big = torch.randn(T, (hq + 2 * hk) * hd, device="cuda").half()
    q1, k1 = torch.zeros(T, hq, hd, device="cuda", dtype=torch.half), torch.zeros(T, hk, hd, device="cuda", dtype=torch.half)
    sdamd.op_rope(fd.data_ptr(), rd, 0, pos.data_ptr(), T, hd, big.data_ptr(), big.shape[1], hd, hq, big.data_ptr() + 2 * hq * hd, big.shape[1], hd,
                  hk, 0, magnitude=1.2, Qo=q1.data_ptr(), Ko=k1.data_ptr())
    c = pr.Cache("f16", hk, hd, ps, 4)
    slots = pr.dev(rng.permutation(4 * ps)[:T])
    q2 = torch.zeros_like(q1)
    rows = torch.arange(T, dtype=torch.int32, device="cuda")
    sdamd.op_paged_prep(big.data_ptr(), big.shape[1], False, None, None, table.data_ptr(), T, rows.data_ptr(), 1, None, slots.data_ptr(), T, hq, hk,
                        hd, rd, ps, 4, q2.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), 0)
    k2, v2 = c.rows(slots)
    x = big.cpu().double().view(T, -1, hd)
    for got, src in ((q1, x[:, :hq]), (q2, x[:, :hq]), (k1, x[:, hq:hq + hk]), (k2, x[:, hq:hq + hk])):
        want, mag = er.rope(src, true, f, 1.2, "half", False)
        check_rows(got.cpu(), want, mag, f, true, "f16", 1.2)


@pytest.mark.parametrize("B,T", [(1, 1), (3, 10), (300, 5000), (8192, 20000), (8192, 200000)])
def test_positions(sdamd, B, T):
    rng = np.random.default_rng(B + T)
    cu = np.sort(rng.integers(0, T + 1, B + 1))
    pos, dropped = rng.integers(0, 1 << 20, T), rng.integers(0, 1 << 30, B)
    want = pos.copy()
    for b in range(B):
        want[cu[b]:cu[b + 1]] += dropped[b]
    args = [pr.dev(cu), pr.dev(dropped), pr.dev(pos)]
    out = torch.full((T + 1,), -5, dtype=torch.int32, device="cuda")
    sdamd.op_page_positions(args[0].data_ptr(), args[1].data_ptr(), B, T, args[2].data_ptr(), out.data_ptr())
    assert out.tolist() == want.tolist() + [-5]
    sdamd.op_page_positions(args[0].data_ptr(), args[1].data_ptr(), B, T, args[2].data_ptr(), args[2].data_ptr())
    assert args[2].tolist() == want.tolist()


def test_replayed(sdamd):
    """A captured step whose positions change between the replays."""
    T, B, rd = 9, 3, 64
    cu, dropped, at = pr.dev([0, 2, 2, 9]), pr.dev([5, 6, 7]), pr.dev(np.arange(T))
    fd = freqs_on(er.freqs(rd, 1e5))
    pos, table, x = torch.zeros(T, dtype=torch.int32, device="cuda"), torch.zeros(T, rd, device="cuda"), torch.randn(T, rd, device="cuda")
    y = torch.zeros_like(x)

    def step(s):
        sdamd.op_page_positions(cu.data_ptr(), dropped.data_ptr(), B, T, at.data_ptr(), pos.data_ptr(), stream=s)
        sdamd.op_rope_table(fd.data_ptr(), rd // 2, pos.data_ptr(), T, table.data_ptr(), stream=s)
        sdamd.op_rope(fd.data_ptr(), rd, 0, pos.data_ptr(), T, rd, x.data_ptr(), rd, rd, 1, None, 0, 0, 0, 2, Qo=y.data_ptr(), stream=s)

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        step(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        dropped.copy_(pr.dev([i, 100 * i, 1000 * i]))
        at.add_(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (pos, table, y)]
        step(None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (pos, table, y)))


@pytest.mark.parametrize("t,kind", [(1, "f16"), (37, "bf16"), (700, "f32")])
@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_rows_of_one_buffer(sdamd, layout, t, kind):
    """q's and k's heads in turn in one buffer, in place by name, and one side in place while the other goes elsewhere: the same
    rows as into buffers of their own."""
    hd, rd, heads = 64, 40, 3
    f = freqs_on(er.freqs(rd, 1e5))
    pos = pr.dev(np.arange(t) * 11 + 5)
    size = torch.finfo(DT[kind]).bits // 8
    for shape, strides in (((t, heads, 2, hd), lambda b: (2 * heads * hd, 2 * hd)), ((heads, 2, t, hd), lambda b: (hd, 2 * t * hd)),
                           ((t, 2, heads, hd), lambda b: (2 * heads * hd, hd))):
        x = torch.randn(shape, device="cuda").to(DT[kind])
        rs, hs = strides(x)
        second = {3: hd, 2: t * hd, 1: heads * hd}[2 if shape[0] == heads and shape[1] == 2 and shape[2] == t else 1 if shape[1] == 2 else 3]

        def call(buf, **kw):
            q, k = buf.data_ptr(), buf.data_ptr() + second * size
            sdamd.op_rope(f.data_ptr(), rd, 0 if layout == "half" else 1, pos.data_ptr(), t, hd, q, rs, hs, heads, k, rs, hs, heads, KIND[kind], **kw)

        q1, k1 = (torch.full((t, heads, hd), 3.0, device="cuda").to(DT[kind]) for _ in range(2))
        call(x, Qo=q1.data_ptr(), Ko=k1.data_ptr())
        here, named, half, out = x.clone(), x.clone(), x.clone(), torch.zeros_like(x)
        call(here)
        own = dict(qo_stride=rs, qo_step=hs, ko_stride=rs, ko_step=hs)
        call(named, Qo=named.data_ptr(), Ko=named.data_ptr() + second * size, **own)
        call(x, Qo=out.data_ptr(), Ko=out.data_ptr() + second * size, **own)
        k2 = torch.zeros_like(k1)
        call(half, **{**own, "Qo": half.data_ptr(), "Ko": k2.data_ptr(), "ko_stride": None, "ko_step": None})
        rows = lambda b, at: torch.as_strided(b, (t, heads, hd), (rs, hs, 1), at)
        for b in (here, named, out):
            assert torch.equal(rows(b, 0), q1) and torch.equal(rows(b, second), k1)
        assert torch.equal(rows(half, 0), q1) and torch.equal(k2, k1) and torch.equal(rows(half, second), rows(x, second))


def test_heads_between_other_rows_heads(sdamd):
    """Heads two steps apart and rows three: every row's later heads lie between the next row's."""
    t, heads, hd, rd = 4, 6, 16, 16
    f, x = freqs_on(er.freqs(rd, 1e4)), torch.randn(2 * hd * (heads - 1) + 3 * hd * (t - 1) + hd, device="cuda")
    rows = torch.as_strided(x, (2, heads, hd), (3 * hd, 2 * hd, 1)).clone()
    y, z = torch.zeros(2, heads, hd, device="cuda"), x.clone()
    sdamd.op_rope(f.data_ptr(), rd, 0, None, 2, hd, x.data_ptr(), 3 * hd, 2 * hd, heads, None, 0, 0, 0, 2, Qo=y.data_ptr())
    sdamd.op_rope(f.data_ptr(), rd, 0, None, 2, hd, z.data_ptr(), 3 * hd, 2 * hd, heads, None, 0, 0, 0, 2)
    want, mag = er.rope(rows.cpu().double(), np.arange(2), er.freqs(rd, 1e4), 1.0, "half", False)
    check_rows(y.cpu(), want, mag, er.freqs(rd, 1e4), np.arange(2), "f32", 1.0)
    assert torch.equal(torch.as_strided(z, (2, heads, hd), (3 * hd, 2 * hd, 1)), y)
    with pytest.raises(sdamd.EngineError, match="two heads overlap"):  # (row 2's first head is row 0's fourth)
        sdamd.op_rope(f.data_ptr(), rd, 0, None, t, hd, x.data_ptr(), 3 * hd, 2 * hd, heads, None, 0, 0, 0, 2)


@pytest.mark.parametrize("t", [1, 50])
def test_outputs_between_the_inputs_rows(sdamd, t):
    """q, k and both outputs side by side in every row of one buffer."""
    hq, hk, hd, rd = 3, 2, 64, 64
    f = freqs_on(er.freqs(rd, 1e4))
    x = torch.randn(t, 2, hq + hk, hd, device="cuda").half()
    x[:, 1] = 7.0
    q, k = (torch.zeros(t, n, hd, device="cuda").half() for n in (hq, hk))
    first = x[:, 0].clone()
    row, at = 2 * (hq + hk) * hd, x.data_ptr()
    args = (f.data_ptr(), rd, 0, None, t, hd, at, row, hd, hq, at + hq * hd * 2, row, hd, hk, 0)
    sdamd.op_rope(*args, Qo=q.data_ptr(), Ko=k.data_ptr())
    out = at + (hq + hk) * hd * 2
    sdamd.op_rope(*args, Qo=out, Ko=out + hq * hd * 2, qo_stride=row, qo_step=hd, ko_stride=row, ko_step=hd)
    assert torch.equal(x[:, 0], first) and torch.equal(x[:, 1], torch.cat([q, k], 1))
