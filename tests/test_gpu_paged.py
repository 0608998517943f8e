"""The paged cache's operators on the GPU against their definitions in 64 bits: the page plan (whole numbers, equal),
the norm, rotation and cache write, the attention, and steps of all three together."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from paged_ref import DT, Cache, dev, half_step, slots_of, tables  # noqa: E402


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- the page plan --------------------------------------------------------------------------------

def plan_on_gpu(sdamd, lens, news, T, ps, n_pages, free, n_free, table):
    B = len(lens)
    a = dict(lens=dev(lens), news=dev(news), free=dev(free), n_free=dev([n_free]), table=dev(table),
             cu=dev(np.full(B + 1, 99)), kv=dev(np.full(B, 99)), slots=dev(np.full(T, 99)), pos=dev(np.full(T, 99)),
             status=dev(np.full(4, 99)))
    sdamd.op_page_plan(a["lens"].data_ptr(), a["news"].data_ptr(), B, T, ps, n_pages, a["free"].data_ptr(),
                       a["n_free"].data_ptr(), a["table"].data_ptr(), table.shape[1], a["cu"].data_ptr(),
                       a["kv"].data_ptr(), a["slots"].data_ptr(), a["pos"].data_ptr(), a["status"].data_ptr(), stream())
    torch.cuda.synchronize()
    return a


def check_plan(sdamd, lens, news, T, ps, n_pages, free, n_free, table):
    a = plan_on_gpu(sdamd, lens, news, T, ps, n_pages, free, n_free, table)
    want = ref.plan(lens, news, T, ps, n_pages, free, n_free, table)
    for k, w in want.items():
        got = a[k].cpu().numpy()
        assert np.array_equal(got, np.asarray(w)), f"{k}: {int((got != np.asarray(w)).sum())} entries differ"
    for k, w in (("lens", lens), ("news", news), ("free", free)):
        assert np.array_equal(a[k].cpu().numpy(), np.asarray(w)), f"{k} changed"


def plan_case(seed, B, ps, hi, new):
    rng = np.random.default_rng(seed)
    lens, news = rng.integers(0, hi, B), rng.integers(0, new + 1, B)
    table, used = tables(rng, lens, ps, 0, width=(hi + new) // ps + 1)
    need = int((-(-(lens + news) // ps) - -(-lens // ps)).sum())
    n_pages = used + need + 3
    free = np.full(n_pages, -9)
    free[:need + 3] = rng.permutation(np.arange(used, n_pages))
    return rng, lens, news, table, need, n_pages, free


@pytest.mark.parametrize("B,ps,hi,new", [(1, 32, 1, 0), (1, 32, 100, 1), (7, 32, 200, 40), (64, 64, 3000, 1),
                                         (1000, 32, 300, 3), (1024, 128, 900, 9), (1025, 32, 64, 20), (8192, 32, 70, 2),
                                         (3, 1024, 9000, 5000)])
def test_plan(sdamd, B, ps, hi, new):
    rng, lens, news, table, need, n_pages, free = plan_case(B + ps, B, ps, hi, new)
    rows = int(news.sum())
    for T, n_free in [(rows + 5, need + 3), (max(rows, 1), need), (max(rows // 2, 1), need + 3), (rows + 1, need // 2),
                      (rows + 1, 0), (rows + 1, -4), (rows + 1, n_pages + 50)]:
        check_plan(sdamd, lens, news, T, ps, n_pages, free, n_free, table)


def test_plan_stops_at_a_request_that_cannot_be(sdamd):
    """Negative counts, more pages than a table row has, counts near the type's end."""
    big = 2 ** 31 - 1
    for lens, news in [([3, -1, 4], [1, 1, 1]), ([3, 2, 4], [1, -1, 1]), ([3, 250, 4], [1, 7, 1]), ([3, big, 4], [1, big, 1]),
                       ([big, 3], [1, 1]), ([-2 ** 31, 3], [-2 ** 31, 1])]:
        table = np.full((len(lens), 8), 5)
        check_plan(sdamd, np.array(lens), np.array(news), 100, 32, 40, np.arange(40), 30, table)


def test_plan_over_holes(sdamd):
    """A page number out of range in the table, or in the free list: its rows have no slot."""
    table = np.array([[3, -1, 0], [2, 77, 0]])
    free = np.array([5, 40, -3, 4, 0, 0])
    check_plan(sdamd, np.array([40, 60]), np.array([60, 10]), 90, 32, 6, free, 4, table)
    check_plan(sdamd, np.array([40, 60]), np.array([60, 10]), 90, 32, 6, free, 3, table)


# ---- norm, rotation, cache write ------------------------------------------------------------------

def rope_table(rd, n=5000, theta=1e4):
    a = torch.arange(n, dtype=torch.float64)[:, None] / theta ** (torch.arange(0, rd, 2, dtype=torch.float64) / max(rd, 1))
    return torch.stack([a.cos(), a.sin()], -1).float().cuda().contiguous()


def prep_case(sdamd, kind, hq, hk, hd, rd, slots, ps, n_pages, axes=1, gated=False, norm=True, pad=0, pstride=0, seed=0,
              poke=None):
    rng = torch.Generator("cuda").manual_seed(seed)
    T, dt = len(slots), DT[kind]
    width = ((2 if gated else 1) * hq + 2 * hk) * hd
    big = torch.randn(T, width + pad, generator=rng, device="cuda").to(dt)
    if poke:
        poke(big)
    qw, kw = (1 + 0.2 * torch.randn(hd, generator=rng, device="cuda") for _ in range(2))
    rope = rope_table(rd)
    pos = torch.randint(0, 5000, (axes, T), generator=rng, device="cuda", dtype=torch.int32)
    pos[:, 0] = 9000  # past the table: its last row
    pos[:, T // 2] = -3
    axis = torch.randint(0, axes + (axes > 1), (max(rd // 2, 1),), generator=rng, device="cuda").to(torch.uint8)
    c = Cache(kind, hk, hd, ps, n_pages, pstride)
    before = c.k.clone(), c.v.clone()
    Q = torch.full((T, hq, hd), math.nan, dtype=dt, device="cuda")
    sl = dev(slots)
    sdamd.op_paged_prep(big.data_ptr(), big.shape[1], gated, qw.data_ptr() if norm else None, kw.data_ptr() if norm else None,
                        rope.data_ptr(), 5000, pos.data_ptr(), axes, axis.data_ptr() if axes > 1 else None, sl.data_ptr(), T,
                        hq, hk, hd, rd, ps, n_pages, Q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(),
                        sdamd.F16 if kind == "f16" else sdamd.BF16, pstride, stream())
    torch.cuda.synchronize()
    x = big[:, :width].double()
    q = x[:, :hq * hd * (2 if gated else 1)].view(T, hq, -1)[..., :hd]
    k, v = x[:, -2 * hk * hd:].view(T, 2, hk, hd).unbind(1)
    ax = axis.clamp(max=axes - 1) if axes > 1 else torch.zeros(max(rd // 2, 1), dtype=torch.uint8, device="cuda")
    q, qm = ref.norm_rotate(q, qw if norm else None, rope, rd, pos, ax)
    k, km = ref.norm_rotate(k, kw if norm else None, rope, rd, pos, ax)
    return Q, c, before, q, qm, k, km, v


def close(kind, got, want, mag, what):
    """The result is rounded once (half a step of the type; 2^-25 where f16 is subnormal); before that the norm's mean
    (8 sums per thread, at most 5 more), root and quotient, two products and one sum are in f32: at most 32 half steps
    of f32, relative to the magnitudes that the result is made of.  Values that are not finite are equal."""
    tol = half_step(kind) * want.abs() + 32 * 2.0 ** -24 * mag * 1.01 + 2.0 ** -25
    g = got.double()
    same = torch.where(want.isfinite(), (g - want).abs() <= tol, (g == want) | (g.isnan() & want.isnan()))
    assert same.all(), f"{what}: {int((~same).sum())} of {same.numel()} off"


def check_prep(sdamd, kind, hq, hk, hd, rd, slots, ps, n_pages, **kw):
    Q, c, before, q, qm, k, km, v = prep_case(sdamd, kind, hq, hk, hd, rd, slots, ps, n_pages, **kw)
    s = np.asarray(slots)
    live = np.nonzero((s >= 0) & (s < n_pages * ps))[0]
    dead = np.setdiff1d(np.arange(len(s)), live)
    at = torch.as_tensor(live, device="cuda")
    gk, gv = c.rows(s[live])
    close(kind, Q[at], q[at], qm[at], "q")
    close(kind, gk, k[at], km[at], "k")
    assert torch.equal(gv.view(torch.int16), v[at].to(gv.dtype).view(torch.int16)), "v"
    assert Q[torch.as_tensor(dead, device="cuda")].isnan().all(), "a row without a slot was written"
    # everything else in the cache is as it was
    c.put(s[live], *Cache_rows(before, c, s[live]))
    assert torch.equal(c.k.view(torch.int16), before[0].view(torch.int16)), "K outside the slots"
    assert torch.equal(c.v.view(torch.int16), before[1].view(torch.int16)), "V outside the slots"


def Cache_rows(before, c, slots):
    old = Cache.__new__(Cache)
    old.__dict__.update(c.__dict__)
    old.k, old.v = before
    return old.rows(slots)


def run_of_slots(rng, T, ps, n_pages, first):
    """Consecutive rows of random pages, from `first` rows into the first page."""
    pages = rng.permutation(n_pages)
    p = np.arange(first, first + T)
    return pages[p // ps] * ps + p % ps


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hk,hd,rd", [(8, 2, 256, 64), (3, 1, 64, 64), (4, 4, 128, 24), (28, 4, 128, 128), (2, 2, 256, 0),
                                         (1, 1, 64, 2), (5, 5, 256, 256), (16, 2, 128, 16)])
def test_prep(sdamd, kind, hq, hk, hd, rd):
    rng = np.random.default_rng(hq * hd + rd)
    for i, (T, first, axes, gated, norm, pad) in enumerate([(1, 0, 1, True, True, 0), (3, 31, 3, False, True, 8),
                                                            (64, 0, 1, False, False, 0), (70, 5, 2, True, True, 24),
                                                            (131, 59, 4, False, True, 0)]):
        check_prep(sdamd, kind, hq, hk, hd, rd, run_of_slots(rng, T, 64, 5, first), 64, 5, axes=axes, gated=gated,
                   norm=norm, pad=pad, seed=i)


def test_prep_of_many_rows(sdamd):
    """Several heads per thread, every page size's blocks, pages further apart than they are long."""
    rng = np.random.default_rng(3)
    check_prep(sdamd, "bf16", 32, 8, 128, 128, run_of_slots(rng, 1500, 32, 60, 3), 32, 60, axes=3)
    check_prep(sdamd, "f16", 8, 2, 256, 64, run_of_slots(rng, 900, 256, 6, 200), 256, 6, gated=True,
               pstride=2 * 256 * 256 + 64)
    check_prep(sdamd, "bf16", 12, 1, 64, 64, run_of_slots(rng, 700, 1024, 2, 0), 1024, 2)


def test_prep_of_mixed_requests_and_rows_without_a_slot(sdamd):
    """Single rows of many requests, slots in any order, negative and too large ones among them."""
    rng = np.random.default_rng(4)
    s = rng.permutation(40 * 32)[:200].astype(np.int64)
    s[[0, 7, 63, 64, 100]] = [-1, 40 * 32, 2 ** 31 - 1, -2 ** 31, -5]
    check_prep(sdamd, "f16", 4, 2, 128, 64, s, 32, 40)
    check_prep(sdamd, "bf16", 4, 2, 128, 64, np.full(3, -1), 32, 40)
    # runs that start anywhere, several in a tile of rows
    runs = np.concatenate([np.arange(a, b) for a, b in [(37, 50), (64, 72), (103, 140), (1000, 1009), (8, 30), (512, 555)]])
    check_prep(sdamd, "bf16", 2, 2, 256, 64, runs, 32, 40)


def test_prep_keeps_what_is_not_finite_to_its_row_and_pair(sdamd):
    def poke(big):
        big[3, 10], big[5, 128 + 100], big[9, -1], big[9, -7] = math.inf, math.nan, math.inf, -math.inf
    check_prep(sdamd, "f16", 2, 1, 128, 32, np.arange(40), 32, 4, norm=False, poke=poke)
    check_prep(sdamd, "bf16", 2, 1, 128, 24, np.arange(40), 32, 4, norm=True, poke=poke)
    check_prep(sdamd, "bf16", 2, 1, 128, 24, np.arange(40), 32, 4, norm=False, poke=poke)


def test_prep_of_weights_and_tables_at_the_alignment_that_is_asked(sdamd):
    """Norm weights 4 bytes, the table 8 bytes past a 16-byte boundary: the same results."""
    for hq, hk, hd, rd in [(4, 2, 128, 64), (2, 1, 64, 24)]:
        T, g = 70, torch.Generator("cuda").manual_seed(hd)
        big = torch.randn(T, (hq + 2 * hk) * hd, generator=g, device="cuda").half()
        w = [1 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)]
        rope, pos, slots = rope_table(rd, 100), dev(np.arange(T)), dev(np.arange(T) + 9)
        got = []
        for off in (0, 1):
            ww = [torch.cat([torch.zeros(off, device="cuda"), x]) for x in w]
            rr = torch.cat([torch.zeros(2 * off, device="cuda"), rope.flatten()])
            c = Cache("f16", hk, hd, 32, 4)
            Q = torch.zeros(T, hq, hd, dtype=torch.float16, device="cuda")
            sdamd.op_paged_prep(big.data_ptr(), big.shape[1], False, ww[0].data_ptr() + 4 * off, ww[1].data_ptr() + 4 * off,
                                rr.data_ptr() + 8 * off, 100, pos.data_ptr(), 1, None, slots.data_ptr(), T, hq, hk, hd, rd, 32,
                                4, Q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), sdamd.F16, 0, stream())
            torch.cuda.synchronize()
            got.append([x.view(torch.int16) for x in (Q, c.k, c.v)])
        assert all(torch.equal(a, b) for a, b in zip(*got))


# ---- attention ------------------------------------------------------------------------------------

def attn_case(sdamd, kind, hq, hk, hd, ps, reqs, window=0, gated=False, scale=None, seed=0, gain=1.0, pstride=0, more_new=0,
              more_kv=0, fill=math.nan, poke=None, holes=None, extra_rows=3):
    """reqs: [(kv_len, new)].  -> everything a call needs, with K and V [kv][hk][hd] per request."""
    rng, g = np.random.default_rng(seed), torch.Generator("cuda").manual_seed(seed)
    kv, new = [r[0] for r in reqs], [r[1] for r in reqs]
    T, dt = sum(new) + extra_rows, DT[kind]
    width = max(-(-(max(kv) + more_kv) // ps), 1)
    table, n_pages = tables(rng, kv, ps, width=width)
    c = Cache(kind, hk, hd, ps, n_pages, pstride, fill)
    q = (gain * torch.randn(T, hq, hd, generator=g, device="cuda")).to(dt)
    big = torch.randn(T, (2 * hq + 2 * hk) * hd + 8, generator=g, device="cuda").to(dt) if gated else None
    ks, vs = [], []
    for b, n in enumerate(kv):
        k, v = (torch.randn(n, hk, hd, generator=g, device="cuda").to(dt) for _ in range(2))
        if poke:
            poke(b, k, v)
        if n:
            c.put(slots_of(table, b, ps, 0, n), k, v)
        ks.append(k)
        vs.append(v)
    for b, blk in holes or ():
        table[b, blk] = (-1, n_pages, 2 ** 31 - 1, -2 ** 31)[blk % 4]
    cu = np.concatenate([[0], np.cumsum(new)])
    out = torch.full((T, hq * hd), 7.0, dtype=dt, device="cuda")
    max_new, max_kv = max(max(new) + more_new, 1), max(max(kv) + more_kv, 1)
    ws = torch.full((max(sdamd.paged_attention_ws(len(reqs), T, max_new, max_kv, hq, hk, hd), 1),), 255, dtype=torch.uint8,
                    device="cuda")
    d = dict(q=q, big=big, c=c, table=dev(table), cu=dev(cu), kvl=dev(kv), out=out, ws=ws, T=T, B=len(reqs), max_new=max_new,
             max_kv=max_kv, ks=ks, vs=vs, kv=kv, new=new, window=window, scale=scale or hd ** -0.5, kind=kind, hq=hq, hk=hk,
             hd=hd, ps=ps, pstride=pstride, n_pages=n_pages, at=cu, holes=holes or ())
    return d


def call(sdamd, d, s=None):
    sdamd.op_paged_attention(d["q"].data_ptr(), d["big"].data_ptr() if d["big"] is not None else None,
                             d["big"].shape[1] if d["big"] is not None else 0, d["c"].k.data_ptr(), d["c"].v.data_ptr(),
                             d["table"].data_ptr(), d["table"].shape[1], d["cu"].data_ptr(), d["kvl"].data_ptr(), d["B"],
                             d["T"], d["max_new"], d["max_kv"], d["hq"], d["hk"], d["hd"], d["ps"], d["n_pages"],
                             d["out"].data_ptr(), d["ws"].data_ptr(), d["ws"].numel(),
                             sdamd.F16 if d["kind"] == "f16" else sdamd.BF16, d["window"], d["scale"], d["pstride"],
                             stream() if s is None else s)


def compare(d, fast=True):
    hq, hd = d["hq"], d["hd"]
    got = d["out"].view(d["T"], hq, hd)
    gates = d["big"][:, :2 * hq * hd].reshape(-1, hq, 2, hd)[:, :, 1].double() if d["big"] is not None else None
    for b, (kv, n) in enumerate(zip(d["kv"], d["new"])):
        if not n:
            continue
        a = int(d["at"][b])
        args = (d["q"][a:a + n].double(), d["ks"][b].double(), d["vs"][b].double(), kv, d["scale"], d["window"],
                gates[a:a + n] if gates is not None else None)
        if fast:
            want, mag, top = ref.attend_fast(*args)
        else:
            want, mag, top = ref.attend(*args, holes=[(blk * d["ps"], (blk + 1) * d["ps"]) for bb, blk in d["holes"] if bb == b])
        tol = ref.attend_bound(d["kind"], want, mag, top, hd, kv)
        g = got[a:a + n].double()
        ok = torch.where(want.isfinite(), (g - want).abs() <= tol, (g == want) | (g.isnan() & want.isnan()))
        assert ok.all(), (f"request {b} (kv {kv}, new {n}): {int((~ok).sum())} of {ok.numel()} off, rows "
                          f"{sorted(set((~ok).nonzero()[:, 0].tolist()))[:8]}, most {(g - want).abs()[want.isfinite()].max():.3g}")
    end = int(d["at"][-1])
    assert (got[end:] == 7.0).all(), "rows behind the last request were written"


def check_attn(sdamd, *a, fast=True, **kw):
    d = attn_case(sdamd, *a, **kw)
    call(sdamd, d)
    torch.cuda.synchronize()
    compare(d, fast)
    return d


HEADS = [(8, 2, 256), (4, 4, 256), (32, 8, 128), (6, 2, 128), (1, 1, 128), (24, 8, 64), (12, 1, 64), (64, 1, 128), (7, 7, 64)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hk,hd", HEADS)
def test_attention_of_single_tokens(sdamd, kind, hq, hk, hd):
    """One new token per request: lengths of one, around the blocks, the pages and the splits."""
    kv = [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 1023, 1024, 1500]
    check_attn(sdamd, kind, hq, hk, hd, 32, [(n, 1) for n in kv], gated=hd == 256, seed=hq)
    check_attn(sdamd, kind, hq, hk, hd, 256, [(n, 1) for n in kv[::-1]], seed=hq + 1)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hk,hd", HEADS)
def test_attention_of_chunks(sdamd, kind, hq, hk, hd):
    """Chunks of 2 to 300 rows on 0 to 700 old ones, single tokens and idle requests among them."""
    reqs = [(2, 2), (0, 0), (5, 4), (40, 40), (45, 0), (100, 7), (33, 32), (160, 129), (1000, 300), (77, 1), (612, 65)]
    check_attn(sdamd, kind, hq, hk, hd, 32, reqs, gated=hd != 128, seed=hq + 2)
    check_attn(sdamd, kind, hq, hk, hd, 128, [(300, 300)], seed=hq + 3)
    check_attn(sdamd, kind, hq, hk, hd, 64, [(900, 3), (17, 3), (3, 3)], seed=hq + 4)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1000])
@pytest.mark.parametrize("hq,hk,hd", [(8, 2, 256), (8, 2, 128), (24, 8, 64)])
def test_attention_in_a_window(sdamd, window, hq, hk, hd):
    reqs = [(1, 1), (700, 1), (40, 40), (900, 200), (33, 5), (5000, 1), (5000, 3)]
    check_attn(sdamd, "bf16", hq, hk, hd, 32, reqs, window=window, seed=window)
    check_attn(sdamd, "f16", hq, hk, hd, 128, reqs[::-1], window=window, gated=True, seed=window + 1)


@pytest.mark.parametrize("hq,hk,hd", [(8, 2, 256), (32, 8, 128), (24, 8, 64)])
def test_attention_over_long_caches(sdamd, hq, hk, hd):
    """Work split over the keys: one request, a few, with and without a chunk."""
    check_attn(sdamd, "bf16", hq, hk, hd, 64, [(20001, 1)], seed=1)
    check_attn(sdamd, "f16", hq, hk, hd, 64, [(9000, 1), (130, 1), (16000, 1)], gated=True, seed=2)
    check_attn(sdamd, "bf16", hq, hk, hd, 32, [(7000, 40)], seed=3)
    check_attn(sdamd, "f16", hq, hk, hd, 32, [(7000, 200), (6000, 1), (300, 2)], seed=4)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_with_sharp_and_rising_scores(sdamd, kind):
    """Scores of a standard deviation of 12: the running maximum rises again and again, most weights vanish."""
    check_attn(sdamd, kind, 8, 2, 256, 32, [(3000, 1), (700, 150)], gain=12.0, seed=5)
    check_attn(sdamd, kind, 8, 8, 64, 32, [(3000, 1), (700, 150)], gain=12.0, seed=6)

    def climb(b, k, v):  # keys that match every query better the later they come
        k[:] = (torch.arange(len(k), device="cuda").view(-1, 1, 1) / 60).to(k.dtype)

    d = attn_case(sdamd, kind, 4, 2, 128, 32, [(900, 1), (900, 260)], poke=climb, seed=7)
    d["q"].abs_()
    call(sdamd, d)
    torch.cuda.synchronize()
    compare(d)


def test_small_weights_count(sdamd):
    """One key whose weight is 1 and 30000 of 2^-22 each (values of one sign): together 0.7 % of the result, which is
    lost where a weight below the type's normal range is rounded away."""
    for kind in ("f16", "bf16"):
        def flat(b, k, v):
            k.zero_()
            k[17] = 1.0
            v.fill_(1.0)
            v[17] = 0.0
        d = attn_case(sdamd, kind, 2, 1, 128, 64, [(30001, 1)], poke=flat, seed=1)
        d["q"].zero_()
        d["q"][:, :, :4] = 22 * math.log(2) / (4 * d["scale"])
        call(sdamd, d)
        torch.cuda.synchronize()
        want = 30000 * 2.0 ** -22 / (1 + 30000 * 2.0 ** -22)
        # q is rounded to the type: the exponent of 2^-22 moves by 22 half steps, its weight by 22 ln 2 of them; the
        # weights are rounded once more, the result too
        tol = want * (22 * math.log(2) + 3) * half_step(kind)
        got = d["out"][0].double()
        assert ((got - want).abs() <= tol).all(), (kind, float(got.min()), float(got.max()), want)


@pytest.mark.parametrize("hq,hk,hd", [(20, 1, 64), (20, 1, 128), (40, 2, 256), (8, 2, 128)])
def test_attention_of_a_prompt_among_longer_caches(sdamd, hq, hk, hd):
    """A fresh prompt and single tokens or drafts on much longer caches, up to 20 heads per kv head."""
    for i, reqs in enumerate([[(300, 300), (5000, 1)], [(2300, 1), (150, 150), (0, 0), (2050, 1)], [(2048, 200), (900, 150)]]):
        check_attn(sdamd, "bf16", hq, hk, hd, 64, reqs, seed=20 + i)
        check_attn(sdamd, "f16", hq, hk, hd, 32, reqs, gated=True, window=700, seed=30 + i)


@pytest.mark.parametrize("B", [65, 150, 5000, 8192])
def test_attention_of_many_requests(sdamd, B):
    """Chunks, drafts and single tokens anywhere among many requests, most of them idle; and all of them in tiles."""
    rng = np.random.default_rng(B)
    busy = set(rng.permutation(B)[:60].tolist()) | {0, 63, 64, B - 1}
    for hq, hk, hd, hi, most in [(8, 2, 64, 900, 70), (3, 1, 128, 60, 40), (8, 1, 256, 300, 9)]:
        reqs = [(0, 0)] * B
        for i, b in enumerate(sorted(busy)):
            new = 1 if i % 3 == 0 else int(rng.integers(1, most))
            reqs[b] = (int(rng.integers(0, hi)) + new, new)
        check_attn(sdamd, "bf16", hq, hk, hd, 32, reqs, seed=B)
        check_attn(sdamd, "f16", hq, hk, hd, 32, reqs, seed=B, more_kv=1500, window=100)
    if B == 150:
        check_attn(sdamd, "f16", 4, 1, 64, 32, [(40 + b % 7, 5 + b % 3) for b in range(B)], seed=3)


@pytest.mark.parametrize("hq,hk,hd", [(8, 2, 256), (6, 2, 128), (24, 8, 64)])
def test_a_window_past_every_key_is_none(sdamd, hq, hk, hd):
    """The largest windows there are, rows before position 0 among the requests': bit for bit the call without one."""
    for reqs in ([(3, 7), (60, 1), (500, 90), (0, 2)], [(5, 6), (200, 1)], [(3000, 1)]):
        d = attn_case(sdamd, "bf16", hq, hk, hd, 32, reqs, seed=21)
        outs = []
        for w in (0, 2 ** 31 - 1, 2 ** 30):
            d["window"] = w
            d["out"].fill_(7.0)
            call(sdamd, d)
            torch.cuda.synchronize()
            outs.append(d["out"].clone())
        d["window"] = 0
        compare(d, fast=False)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_scores_that_are_not_finite(sdamd, kind):
    """Infinities and NaN in seen keys and in queries give what the definition gives, to their rows alone."""
    def poke(b, k, v):
        if b < 2:
            k[20, 0, 3], k[45, -1, 7] = math.inf, math.nan

    for hq, hk, hd in [(8, 2, 256), (4, 2, 128), (3, 1, 64)]:
        d = attn_case(sdamd, kind, hq, hk, hd, 32, [(90, 80), (70, 1), (100, 1), (2500, 2), (64, 40)], poke=poke, seed=22)
        at = d["at"]
        d["q"][at[0] + 5, 0, 2] = math.nan
        d["q"][at[2], -1, 0] = math.inf
        d["q"][at[3] + 1, 0, 9] = -math.inf
        d["q"][at[4] + 33, :, 1] = math.inf
        call(sdamd, d)
        torch.cuda.synchronize()
        compare(d, fast=False)


def test_rows_that_see_nothing(sdamd):
    """More new rows than rows in all: those before position 0 see nothing and give zeros."""
    for hq, hk, hd in [(8, 2, 256), (4, 2, 64)]:
        for reqs in ([(3, 7)], [(0, 5), (60, 1)], [(20, 90), (0, 1)], [(0, 1)]):
            d = check_attn(sdamd, "f16", hq, hk, hd, 32, reqs, gated=True, fast=False, seed=2)
            kv, n = reqs[0]
            assert (d["out"][:n - kv] == 0).all()


def test_holes(sdamd):
    """Pages that are gone: their rows are not seen, by a row that sees nothing else either."""
    for hq, hk, hd in [(8, 2, 256), (8, 2, 128), (3, 1, 64)]:
        holes = [(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (1, 3), (2, 1)]
        check_attn(sdamd, "bf16", hq, hk, hd, 32, [(200, 1), (100, 1), (90, 60)], holes=holes, fast=False, seed=3)
        check_attn(sdamd, "f16", hq, hk, hd, 32, [(200, 2), (100, 33), (90, 90)], holes=holes, window=40, fast=False, seed=4)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hk,hd", [(8, 2, 256), (4, 1, 128), (2, 2, 64)])
def test_what_is_not_seen_changes_nothing(sdamd, kind, hq, hk, hd):
    """NaN and infinities in the values and keys of rows that come later (the cache's unused rows are NaN in every
    test); rows that see them get what the definition gives."""
    def poke(b, k, v):
        if b == 0:
            v[70, 0, 3], v[71, -1, 40], v[72, 0, 5], v[100, 0, 3] = math.inf, math.nan, -math.inf, -math.inf
        if b == 1:
            k[50, 0, 9], v[60, 0], k[61] = math.inf, math.nan, math.nan
        if b == 2:
            v[0, 0, 1] = math.inf

    reqs = [(110, 60), (64, 20), (50, 3), (130, 130), (9, 1)]
    check_attn(sdamd, kind, hq, hk, hd, 32, reqs, poke=poke, fast=False, seed=6)
    check_attn(sdamd, kind, hq, hk, hd, 64, reqs, window=30, poke=poke, fast=False, gated=True, seed=7)
    check_attn(sdamd, kind, hq, hk, hd, 64, [(110, 6), (64, 4), (50, 3)], window=9, poke=poke, fast=False, seed=8)


def test_scores_of_minus_infinity(sdamd):
    """Keys of -inf in one dim: their weights are 0; where every seen key has one the row gives zeros."""
    def poke(b, k, v):
        k[:30, :, 0] = -math.inf
        k[40:41, :, 0] = -math.inf

    for hd in (64, 256):
        d = attn_case(sdamd, "bf16", 4, 2, hd, 32, [(60, 60), (30, 2), (60, 1)], poke=poke, seed=9)
        d["q"].abs_()
        call(sdamd, d)
        torch.cuda.synchronize()
        compare(d, fast=False)
        assert (d["out"][:30] == 0).all() and (d["out"][60:62] == 0).all()


def test_bounds_above_the_actual_sizes(sdamd):
    """max_new and max_kv are upper bounds (a captured graph's): larger ones change splits, not results."""
    reqs = [(1, 1), (300, 1), (64, 1), (40, 2)]
    for more_new, more_kv in [(0, 5000), (60, 0), (300, 40000)]:
        check_attn(sdamd, "bf16", 32, 8, 128, 64, reqs, more_new=more_new, more_kv=more_kv, seed=10)
        check_attn(sdamd, "f16", 8, 2, 256, 32, reqs, more_new=more_new, more_kv=more_kv, gated=True, seed=11)


def test_pages_further_apart(sdamd):
    check_attn(sdamd, "f16", 8, 2, 256, 32, [(100, 1), (200, 100)], pstride=2 * 32 * 256 + 8, seed=12)
    check_attn(sdamd, "bf16", 4, 4, 64, 64, [(100, 1), (200, 100)], pstride=2 * 4 * 64 * 64, seed=13)


def test_offsets_past_32_bits(sdamd):
    """Pages 2^28 elements apart, 20 of them: the last ones start past 2^32 elements (and bytes)."""
    hq, hk, hd, ps, n_pages, far = 4, 2, 128, 32, 20, 2 ** 28
    d = attn_case(sdamd, "bf16", hq, hk, hd, ps, [(150, 1), (300, 40)], seed=14)
    k, v = (torch.empty(n_pages * far, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    small = d["c"]
    page = small.page
    assert d["n_pages"] <= n_pages
    for p in range(d["n_pages"]):  # page p of the case's cache becomes page 19 - p
        k[(19 - p) * far:(19 - p) * far + page] = small.k[p * page:(p + 1) * page]
        v[(19 - p) * far:(19 - p) * far + page] = small.v[p * page:(p + 1) * page]
    d["table"] = torch.where(d["table"] >= 0, 19 - d["table"], d["table"]).int().contiguous()
    small.k, small.v, d["pstride"], d["n_pages"] = k, v, far, n_pages
    call(sdamd, d)
    torch.cuda.synchronize()
    compare(d)
    # and the write of rows there
    big = torch.randn(2, (hq + 2 * hk) * hd, device="cuda").bfloat16()
    Q = torch.zeros(2, hq, hd, dtype=torch.bfloat16, device="cuda")
    slots = dev([19 * ps + 31, 18 * ps])
    sdamd.op_paged_prep(big.data_ptr(), big.shape[1], False, None, None, None, 0, None, 1, None, slots.data_ptr(), 2, hq, hk,
                        hd, 0, ps, n_pages, Q.data_ptr(), k.data_ptr(), v.data_ptr(), sdamd.BF16, far, stream())
    torch.cuda.synchronize()
    rows = big[:, hq * hd:].view(2, 2, hk, hd)
    for i, (p, r) in enumerate([(19, 31), (18, 0)]):
        kk = k[p * far:p * far + page].view(hk, hd // 32, 32, 32)[:, :, r].reshape(hk, hd)
        vv = v[p * far:p * far + page].view(hk, hd, 32)[:, :, r]
        assert torch.equal(kk, rows[i, 0]) and torch.equal(vv, rows[i, 1])


def test_counts_that_do_not_fit_stay_in_bounds(sdamd):
    """Row starts and lengths past the given bounds are cut: whatever they are, only rows of out are written."""
    d = attn_case(sdamd, "bf16", 8, 2, 128, 32, [(100, 1), (100, 30), (64, 2)], seed=15)
    for cu, kv in [([0, 1, 31, 2 ** 31 - 1], [100, 100, 64]), ([-5, 1, 31, 33], [2 ** 31 - 1, 100, -64]),
                   ([40, 3, -7, 33], [100, 100, 2 ** 31 - 1]), ([0, 1, 31, 33], [-2 ** 31, 2 ** 31 - 1, 0])]:
        d["cu"], d["kvl"] = dev(cu), dev(kv)
        call(sdamd, d)
        torch.cuda.synchronize()


def test_two_streams_and_repeats_are_equal(sdamd):
    """The same call again, and calls on two streams at once with a workspace each: bit for bit the same."""
    ds = [attn_case(sdamd, "bf16", 32, 8, 128, 64, [(5000, 1), (300, 1), (900, 80)], seed=16 + i) for i in range(2)]
    first = []
    for d in ds:
        call(sdamd, d)
        torch.cuda.synchronize()
        first.append(d["out"].clone())
        d["out"].fill_(7.0)
    torch.cuda.synchronize()
    ss = [torch.cuda.Stream() for _ in ds]
    for _ in range(5):
        for d, s in zip(ds, ss):
            call(sdamd, d, s.cuda_stream)
    torch.cuda.synchronize()
    for d, f in zip(ds, first):
        assert torch.equal(d["out"].view(torch.int16), f.view(torch.int16))
        compare(d)


# ---- steps of all three ---------------------------------------------------------------------------

class Server:
    """A layer's paged cache and the buffers of its steps, as a serving program keeps them."""

    def __init__(self, sdamd, kind, hq, hk, hd, rd, ps, n_pages, B, T, max_new, max_kv, gated):
        self.__dict__.update(sdamd=sdamd, kind=kind, hq=hq, hk=hk, hd=hd, rd=rd, ps=ps, B=B, T=T, max_new=max_new,
                             max_kv=max_kv, gated=gated)
        self.c = Cache(kind, hk, hd, ps, n_pages)
        self.free = dev(np.random.default_rng(0).permutation(n_pages))
        self.table = dev(np.full((B, -(-max_kv // ps)), -1))
        self.lens, self.news, self.kvl = dev(np.zeros(B)), dev(np.zeros(B)), dev(np.zeros(B))
        self.cu, self.slots, self.pos = dev(np.zeros(B + 1)), dev(np.zeros(T)), dev(np.zeros(T))
        self.n_free, self.status = dev([n_pages]), dev(np.zeros(4))
        self.width = ((2 if gated else 1) * hq + 2 * hk) * hd
        self.big = torch.zeros(T, self.width, dtype=DT[kind], device="cuda")
        self.q = torch.zeros(T, hq, hd, dtype=DT[kind], device="cuda")
        self.out = torch.zeros(T, hq * hd, dtype=DT[kind], device="cuda")
        self.qw = 1 + 0.1 * torch.randn(hd, device="cuda")
        self.kw = 1 + 0.1 * torch.randn(hd, device="cuda")
        self.rope = rope_table(rd, max_kv)
        self.ws = torch.empty(max(sdamd.paged_attention_ws(B, T, max_new, max_kv, hq, hk, hd), 16), dtype=torch.uint8,
                              device="cuda")

    def step(self):
        sd, s = self.sdamd, stream()
        ty = sd.F16 if self.kind == "f16" else sd.BF16
        sd.op_page_plan(self.lens.data_ptr(), self.news.data_ptr(), self.B, self.T, self.ps, self.c.n_pages,
                        self.free.data_ptr(), self.n_free.data_ptr(), self.table.data_ptr(), self.table.shape[1],
                        self.cu.data_ptr(), self.kvl.data_ptr(), self.slots.data_ptr(), self.pos.data_ptr(),
                        self.status.data_ptr(), s)
        sd.op_paged_prep(self.big.data_ptr(), self.width, self.gated, self.qw.data_ptr(), self.kw.data_ptr(),
                         self.rope.data_ptr(), self.rope.shape[0], self.pos.data_ptr(), 1, None, self.slots.data_ptr(),
                         self.T, self.hq, self.hk, self.hd, self.rd, self.ps, self.c.n_pages, self.q.data_ptr(),
                         self.c.k.data_ptr(), self.c.v.data_ptr(), ty, 0, s)
        sd.op_paged_attention(self.q.data_ptr(), self.big.data_ptr() if self.gated else None, self.width if self.gated else 0,
                              self.c.k.data_ptr(), self.c.v.data_ptr(), self.table.data_ptr(), self.table.shape[1],
                              self.cu.data_ptr(), self.kvl.data_ptr(), self.B, self.T, self.max_new, self.max_kv, self.hq,
                              self.hk, self.hd, self.ps, self.c.n_pages, self.out.data_ptr(), self.ws.data_ptr(),
                              self.ws.numel(), ty, stream=s)
        # the step's ends are the next one's starts
        self.lens.copy_(self.kvl)
        self.n_free.copy_(self.status[3:])


def serve(sv, steps, replay=None, seed=0):
    """Runs the steps ([new tokens per request]) and checks each against the requests' whole histories in 64 bits,
    computed from the rounded queries and keys' definition."""
    g = torch.Generator("cuda").manual_seed(seed)
    hist = [[] for _ in range(sv.B)]
    u, e = half_step(sv.kind), 2.0 ** -24
    for news in steps:
        n = sum(news)
        sv.news.copy_(dev(news))
        sv.big.copy_(torch.randn(sv.T, sv.width, generator=g, device="cuda"))
        sv.out.fill_(7.0)
        sv.step() if replay is None else replay()
        torch.cuda.synchronize()
        assert sv.status.tolist()[:2] == [sv.B, n]
        at = 0
        for b, m in enumerate(news):
            if not m:
                continue
            x = sv.big[at:at + m].double()
            kv = x[:, -2 * sv.hk * sv.hd:].view(m, 2, sv.hk, sv.hd)
            p = torch.arange(len(hist[b]), len(hist[b]) + m, device="cuda")[None]
            ax = torch.zeros(sv.rd // 2, dtype=torch.uint8, device="cuda")
            k, _ = ref.norm_rotate(kv[:, 0], sv.kw, sv.rope, sv.rd, p, ax)
            hist[b] += list(zip(k, kv[:, 1]))
            q = x[:, :sv.hq * sv.hd * (2 if sv.gated else 1)].view(m, sv.hq, -1)
            gate = q[..., sv.hd:] if sv.gated else None
            q, _ = ref.norm_rotate(q[..., :sv.hd], sv.qw, sv.rope, sv.rd, p, ax)
            ks, vs = (torch.stack([h[i] for h in hist[b]]) for i in range(2))
            want, mag, top = ref.attend_fast(q, ks, vs, len(ks), sv.hd ** -0.5, 0, gate)
            # the call's own bound, and q and k rounded to the type on the way (and f32 before that): a score moves by
            # at most (2 u + 64 e) of its magnitudes, weights and their sum by that much each
            tol = ref.attend_bound(sv.kind, want, mag, top, sv.hd, len(ks)) + 2 * (2 * u + 64 * e) * top * 1.01 * mag
            got = sv.out[at:at + m].view(m, sv.hq, sv.hd).double()
            bad = (got - want).abs() > tol
            assert not bad.any(), f"step {news}, request {b}: {int(bad.sum())} off"
            at += m
        assert (sv.out[n:] == 7.0).all()


STEPS = [[40, 0, 7, 0], [1, 33, 1, 0], [1, 1, 1, 90], [3, 1, 0, 1], [1, 1, 64, 1], [1, 1, 1, 1]]


@pytest.mark.parametrize("kind,hq,hk,hd,rd,gated", [("f16", 8, 2, 256, 64, True), ("bf16", 8, 2, 128, 128, False),
                                                    ("f16", 6, 2, 64, 24, False)])
def test_serving_steps(sdamd, kind, hq, hk, hd, rd, gated):
    serve(Server(sdamd, kind, hq, hk, hd, rd, 32, 40, 4, 128, 100, 512, gated), STEPS)


def test_serving_steps_replayed_from_a_graph(sdamd):
    """One captured step, replayed with other lengths, news and rows: the counts are read on the device.  Eager work
    runs between the replays."""
    sv = Server(sdamd, "bf16", 8, 2, 128, 64, 32, 40, 4, 128, 100, 512, False)
    sv.step()  # (no new tokens: nothing changes)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sv.step()
    serve(sv, STEPS, graph.replay)


def test_two_graphs_with_a_workspace_each(sdamd):
    """Two captured calls whose work is split, replayed at once on two streams, eager calls between: bit for bit the
    eager results, every time."""
    reqs = [(6000, 1), (300, 1), (900, 120)]
    ds = [attn_case(sdamd, "f16", 8, 2, 256, 64, reqs, gated=True, seed=40 + i) for i in range(2)]
    assert all(d["ws"].numel() > 1 for d in ds)
    first, graphs, ss = [], [], [torch.cuda.Stream() for _ in ds]
    for d in ds:
        call(sdamd, d)
        torch.cuda.synchronize()
        compare(d)
        first.append(d["out"].clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(sdamd, d)
        graphs.append(graph)
    for i in range(4):
        for d in ds:
            d["out"].fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, s in zip(graphs, ss):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for d, f in zip(ds, first):
            assert torch.equal(d["out"].view(torch.int16), f.view(torch.int16))
            d["out"].fill_(7.0)
        torch.cuda.synchronize()
        for d, f in zip(ds, first):
            call(sdamd, d)
            torch.cuda.synchronize()
            assert torch.equal(d["out"].view(torch.int16), f.view(torch.int16))


def test_one_sequence_is_the_contiguous_attention(sdamd):
    """A single f16 request of the engine's heads against sd_op_attention on the same rows."""
    hq, hk, hd, rd, P, L = 8, 2, 256, 64, 200, 45
    sv = Server(sdamd, "f16", hq, hk, hd, rd, 32, 40, 1, 256, 256, 4096, True)
    g = torch.Generator("cuda").manual_seed(1)
    rows = torch.randn(P + L, sv.width, generator=g, device="cuda").half()
    ctx = 4096
    K, V = (torch.zeros(hk * ctx * hd, dtype=torch.float16, device="cuda") for _ in range(2))
    for first, n in ((0, P), (P, L)):
        sv.news.copy_(dev([n]))
        sv.big[:n] = rows[first:first + n]
        sv.step()
        big = rows[first:first + n].contiguous()
        Q = torch.zeros(hq * n * hd, dtype=torch.float16, device="cuda")
        out = torch.zeros(n, hq * hd, dtype=torch.float16, device="cuda")
        sdamd.op_attention(big.data_ptr(), sv.width, sv.qw.data_ptr(), sv.kw.data_ptr(), sv.rope.data_ptr(), n, first, hq, hk,
                           hd, rd, Q.data_ptr(), K.data_ptr(), V.data_ptr(), ctx, out.data_ptr(), stream())
        torch.cuda.synchronize()
        # the keys and values of both caches are the same rows, in the same blocks
        k, v = sv.c.rows(slots_of(sv.table.cpu().numpy().astype(np.int64), 0, 32, 0, first + n))
        k2 = K.view(hk, ctx // 32, hd // 32, 32, 32).permute(1, 3, 0, 2, 4).reshape(ctx, hk, hd)[:first + n]
        v2 = V.view(hk, ctx // 32, hd, 32).permute(1, 3, 0, 2).reshape(ctx, hk, hd)[:first + n]
        u = half_step("f16")
        assert torch.equal(v, v2)
        assert ((k.float() - k2.float()).abs() <= 2 * u * k2.float().abs() + 2.0 ** -24).all()
        # both are within their roundings of the same result: q rounded again after its scale there, weights here;
        # scores reach 6 here, so 4 u of 6 in a weight's exponent, twice, and 3 u of roundings, of values up to 5
        assert ((sv.out[:n].float() - out.float()).abs() <= (2 * 4 * 6 + 3) * u * 5).all()
