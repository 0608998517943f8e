"""Rows that leave the paged cache, against their definitions in 64 bits: the weight that every cached key receives, the rows
that go, their moves, their pages, and a run of them all beside the cache's other operators."""
import math

import numpy as np
import pytest
import torch

import evict_ref as er
import paged_ref as pr
from launches import launches

pytestmark = pytest.mark.gpu
KIND = {"f16": 0, "bf16": 1}


# ---- the weight that every cached key receives ----------------------------------------------------

class Step:
    """Requests with old and new rows in pages, as a step's weights find them."""

    def __init__(self, seed, old, new, hq, hk, hd, ps, kind, window=0, observers=0, decay=1.0, scale=None, pstride=0, fill=math.nan, loud=1.5):
        rng = np.random.default_rng(seed)
        g = torch.Generator("cuda").manual_seed(seed)
        self.old, self.new, self.kv = old, new, [o + n for o, n in zip(old, new)]
        self.hq, self.hk, self.hd, self.ps, self.kind = hq, hk, hd, ps, kind
        self.window, self.observers, self.decay, self.scale = window, observers, decay, hd ** -0.5 if scale is None else scale
        self.table, self.n_pages = pr.tables(rng, self.kv, ps)
        self.cache = pr.Cache(kind, hk, hd, ps, self.n_pages, pstride, fill)
        self.k = []
        for b, n in enumerate(self.kv):
            k = torch.randn(n, hk, hd, generator=g, device="cuda").to(pr.DT[kind])
            self.k.append(k)
            if n:
                self.cache.put(pr.slots_of(self.table, b, ps, 0, n), k, torch.zeros_like(k))
        self.T = sum(new)
        self.q = (loud * torch.randn(max(self.T, 1), hq, hd, generator=g, device="cuda")).to(pr.DT[kind])
        self.scores = torch.rand(self.n_pages, hk, ps, generator=g, device="cuda") * 3
        self.pos = pr.dev(rng.integers(0, 1 << 30, max(self.T, 1)))
        self.holes = {}
        self.extra = 0  # rows of Q behind the last request's

    def run(self, sdamd, out=None, kpos=None, scores=True, max_new=None, max_kv=None, stream=None, ws=None):
        B = len(self.old)
        self.out = torch.full_like(self.scores, -7.0) if out is None else out
        self.kpos = torch.full(self.scores.shape, -9, dtype=torch.int32, device="cuda") if kpos is None else kpos
        max_new, max_kv = max_new or max(max(self.new), 1), max_kv or max(max(self.kv), 1)
        T = max(self.T, 1)
        table = np.full((B, max(self.table.shape[1], -(-max_kv // self.ps))), -7)
        table[:, :self.table.shape[1]] = self.table
        self.dtable, self.cu, self.lens = pr.dev(table), pr.dev(np.concatenate([[0], np.cumsum(self.new)])), pr.dev(self.kv)
        if ws is None:
            self.ws = torch.full((sdamd.paged_weights_ws(B, T, max_new, max_kv, self.hq, self.hk, self.hd, self.observers) + 64,), 0xFF, dtype=torch.uint8,
                                 device="cuda")
        else:
            self.ws = ws
        sdamd.op_paged_weights(self.q.data_ptr(), self.cache.k.data_ptr(), self.dtable.data_ptr(), table.shape[1], self.cu.data_ptr(),
                               self.lens.data_ptr(), B, T, max_new, max_kv, self.hq, self.hk, self.hd, self.ps, self.n_pages,
                               self.scores.data_ptr() if scores else None, self.out.data_ptr(), self.ws.data_ptr(), self.ws.numel() - 64,
                               KIND[self.kind], decay=self.decay, observers=self.observers, window=self.window, scale=self.scale,
                               pos=self.pos.data_ptr(), kpos=self.kpos.data_ptr(), page_stride=self.cache.pstride, stream=stream)
        return self.out

    def check(self, old_scores=None):
        old_scores = self.scores if old_scores is None else old_scores
        assert (self.ws[-64:] == 0xFF).all()
        seen = torch.zeros(self.out.shape, dtype=torch.bool)
        fresh = seen.clone()
        out, kpos, at = self.out.cpu(), self.kpos.cpu(), 0
        for b, (o, n, kv) in enumerate(zip(self.old, self.new, self.kv)):
            if n == 0:
                continue
            s = torch.as_tensor(pr.slots_of(self.table, b, self.ps, 0, kv))
            page, row = s // self.ps, s % self.ps
            there = torch.tensor([not any(x <= j < y for x, y in self.holes.get(b, ())) for j in range(kv)])
            prior = old_scores.cpu()[page.clamp(0, self.n_pages - 1), :, row].double().T  # [hk][kv]
            want, top = er.weights(self.q[at:at + n].cpu().double(), self.k[b].cpu().double(), kv, self.scale, self.window, self.observers,
                                   self.holes.get(b, ()), self.decay, prior)
            got = out[page[there], :, row[there]].double().T
            want = want[:, there]
            rows = n * self.hq // self.hk
            bound = er.weights_bound(want, top, self.hd, kv, rows)
            assert torch.equal(torch.isnan(got), torch.isnan(want)), b
            ok = ((got - want).abs() <= bound) | torch.isnan(want)
            assert ok.all(), (b, float((got - want).abs().nan_to_num(0).max()), float(((got - want).abs() / bound).nan_to_num(0).max()))
            seen[page[there], :, row[there]] = True
            late = there & (torch.arange(kv) >= o)
            fresh[page[late], :, row[late]] = True
            p = self.pos[at:at + n].cpu()[torch.arange(kv)[late] - o]
            assert (kpos[page[late], :, row[late]] == p[:, None]).all()
            at += n
        assert (out[~seen] == -7).all() and (kpos[~fresh] == -9).all()


SHAPES = [  # old, new
    ([0], [1]), ([700], [1]), ([31], [1]), ([32], [1]), ([1000, 0, 5, 64, 1], [1, 1, 1, 0, 1]), ([0], [33]), ([0, 100], [130, 64]),
    ([300, 90, 4000], [4, 5, 6]), ([517, 33, 1200, 8], [1, 200, 1, 0]), ([2500], [40]),
]
HEADS = [(8, 2, 256, "f16"), (8, 2, 128, "bf16"), (3, 1, 64, "f16"), (4, 4, 128, "f16"), (16, 1, 64, "bf16")]


@pytest.mark.parametrize("hq,hk,hd,kind", HEADS)
@pytest.mark.parametrize("old,new", SHAPES)
def test_weights(sdamd, old, new, hq, hk, hd, kind):
    s = Step(len(old) * 7 + hd, old, new, hq, hk, hd, 32 if hd != 64 else 128, kind)
    s.run(sdamd)
    s.check()


@pytest.mark.parametrize("observers", [1, 3, 32, 50, 1000])
@pytest.mark.parametrize("window", [0, 1, 70])
def test_observers_and_windows(sdamd, observers, window):
    for hq, hk, hd, kind in ((8, 2, 256, "f16"), (24, 8, 64, "bf16"), (5, 1, 128, "f16")):
        s = Step(observers + window, [250, 0, 3, 900], [40, 65, 1, 7], hq, hk, hd, 64, kind, window=window, observers=observers, decay=0.5)
        s.run(sdamd)
        s.check()


@pytest.mark.parametrize("hq,hk,hd", [(64, 1, 64), (40, 1, 128), (20, 1, 256), (17, 1, 64), (33, 1, 128)])
def test_many_query_heads(sdamd, hq, hk, hd):
    s = Step(hq, [300, 40], [1, 3], hq, hk, hd, 32, "bf16")
    s.run(sdamd)
    s.check()


def test_long_cache(sdamd):
    for new, obs in (([1, 1], 0), ([40, 1], 16)):
        s = Step(5, [30011, 9000], new, 8, 2, 128, 128, "f16", observers=obs, decay=0.0)
        s.run(sdamd, scores=False)
        s.check()


def test_prompt(sdamd):
    s = Step(6, [0, 700], [1100, 515], 8, 2, 64, 64, "bf16", decay=0.9)
    s.run(sdamd)
    s.check()


def test_decay_zero_reads_nothing_and_out_may_be_scores(sdamd):
    for old, new in (([300, 40], [1, 1]), ([300, 40], [60, 1])):
        s = Step(9, old, new, 8, 2, 128, 32, "f16", decay=0.0)
        s.scores.fill_(math.nan)
        s.run(sdamd)
        s.check()
        s = Step(10, old, new, 8, 2, 128, 32, "f16", decay=1.0)
        prior = s.scores.clone()
        mask = s.run(sdamd).clone() == -7
        s.run(sdamd, out=s.scores)
        assert torch.equal(s.scores[mask], prior[mask])
        s.out = torch.where(mask, torch.full_like(s.scores, -7.0), s.scores)
        s.check(prior)


def test_bounds_above_the_sizes(sdamd):
    for old, new in (([300, 40], [1, 1]), ([300, 40], [60, 2])):
        s = Step(11, old, new, 8, 2, 128, 32, "f16")
        s.run(sdamd, max_new=500, max_kv=9000)
        s.check()
        s.run(sdamd, max_new=70, max_kv=131072)
        s.check()


def test_bounds_below_the_sizes_leave_rows_and_keys_out(sdamd):
    """No key past max_kv is touched."""
    s = Step(12, [500], [1], 8, 2, 128, 32, "f16")
    out = s.run(sdamd, max_kv=100)
    slots = pr.slots_of(s.table, 0, 32, 100, 501)
    assert (out[slots // 32, :, slots % 32] == -7).all()


def test_page_stride_and_holes(sdamd):
    for new in ([1, 1], [50, 1]):
        s = Step(13, [400, 100], new, 8, 2, 128, 32, "bf16", pstride=2 * 32 * 128 + 72)
        s.table[0, 3] = -1
        s.table[0, 5] = s.n_pages + 2
        s.holes = {0: [(96, 128), (160, 192)]}
        s.run(sdamd)
        s.check()


def test_a_request_of_holes_alone(sdamd):
    for new in ([1, 2], [40, 70]):
        s = Step(14, [60, 30], new, 4, 1, 64, 32, "f16")
        s.table[0, :] = -1
        s.holes = {0: [(0, 1 << 20)]}
        s.run(sdamd)
        s.check()


@pytest.mark.parametrize("new", [1, 5, 70])
@pytest.mark.parametrize("old", [200, 3001])
def test_non_finite_keys_and_queries(sdamd, old, new):
    """A NaN or infinite score makes the rows that see it NaN, and no others."""
    for bad in (math.nan, math.inf):
        s = Step(15, [old], [new], 8, 2, 128, 32, "f16")
        late = old + new - 1  # seen by the last row alone
        s.k[0][late, 1, 3] = bad
        s.cache.put(pr.slots_of(s.table, 0, 32, 0, old + new), s.k[0], torch.zeros_like(s.k[0]))
        s.q[:, :, 3] = s.q[:, :, 3].abs() + 0.5
        s.run(sdamd)
        s.check()
        s = Step(16, [old], [new], 8, 2, 128, 32, "f16")
        s.q[new // 2, 6, 0] = bad
        s.run(sdamd)
        s.check()


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("old,window", [(90, 3), (90, 0), (5000, 0)])
def test_every_score_minus_infinity(sdamd, old, window, new):
    s = Step(17, [old], [new], 4, 1, 64, 32, "bf16", window=window)
    s.k[0][:, 0, 0] = -math.inf
    s.cache.put(pr.slots_of(s.table, 0, 32, 0, old + new), s.k[0], torch.zeros_like(s.k[0]))
    s.q[:, :, 0] = 1.0
    s.run(sdamd)
    s.check()


@pytest.mark.parametrize("loud,scale", [(0.0, None), (30.0, None), (1.5, 1e-30), (1.5, 0.5)])
def test_ranges_of_scores(sdamd, loud, scale):
    for old, new in (([500], [1]), ([500], [64]), ([3000], [1])):
        s = Step(18, old, new, 8, 2, 128, 32, "bf16", loud=loud, scale=scale)
        s.run(sdamd)
        s.check()


@pytest.mark.parametrize("old,new", [(100, 1), (100, 70), (3000, 1)])
def test_scores_without_fractions(sdamd, old, new):
    """Scores of 2^30 and more: each row's largest key takes all of its weight."""
    s = Step(19, [old], [new], 8, 2, 128, 32, "f16", loud=4.0, scale=1e9)
    s.run(sdamd)
    q, k = s.q.cpu().double(), s.k[0].cpu().double()
    n = old + new
    slots = pr.slots_of(s.table, 0, 32, 0, n)
    got, prior = (x.cpu()[slots // 32, :, slots % 32].double() for x in (s.out, s.scores))
    got -= prior * (torch.arange(n) < old)[:, None]
    for h in range(2):
        want = torch.zeros(n, dtype=torch.float64)
        for i in range(new):
            x = q[i, 4 * h:4 * h + 4] @ k[:old + i + 1, h].T
            for y in x:
                v, j = y.topk(2)
                assert v[0] - v[1] > 1e-5 * v[0].abs()
                want[j[0]] += 1
        # (3 + 70 x 4 rounded twice, and what is taken off again: half a step of 2^9 each)
        assert (got[:, h] - want).abs().max() <= 1e-4


def test_same_bits_every_time(sdamd):
    for new in ([1, 1, 1], [300, 1, 40]):
        s = Step(20, [3000, 100, 40], new, 8, 2, 128, 64, "f16")
        a = s.run(sdamd).clone()
        for _ in range(3):
            assert torch.equal(a, s.run(sdamd))


@pytest.mark.parametrize("hq,hk,hd,kind,most", [(16, 8, 64, "f16", 8100), (8, 8, 128, "bf16", 3000), (32, 8, 256, "f16", 700)])
def test_many_requests(sdamd, hq, hk, hd, kind, most):
    """A head per workgroup, its scores in LDS up to the most that it takes."""
    rng = np.random.default_rng(hd)
    old = [most - 1] + [int(x) for x in rng.integers(0, 400, 39)]
    for new in ([1] * 40, [2] + [1] * 30 + [0] * 9):
        s = Step(40, old, new, hq, hk, hd, 32, kind, window=0 if sum(new) == 40 else 300)
        s.run(sdamd, max_new=2)
        s.check()


@pytest.mark.parametrize("requests,long", [(128, 2000), (129, 2000), (700, 300), (4500, 40)])
def test_requests_with_chunks(sdamd, requests, long):
    """Both sides of the number from which on the tiles have an index; its steps beyond 64 requests; parts and splits of some."""
    rng = np.random.default_rng(requests)
    old, new = rng.integers(0, long // 8, requests), rng.choice([0, 1, 1, 9, 40], requests)
    old[[0, 70, requests - 2]], new[[0, 3, 70, requests - 1]] = (0, long, long), (0, long, 90, 33)
    s = Step(requests, old.tolist(), new.tolist(), 8, 2, 64, 32, "f16", observers=0 if requests < 500 else 20)
    s.run(sdamd)
    s.check()


def few_launches(sdamd, B, T, max_new, max_kv, hq, hk, hd, observers=0):
    """Workgroup sizes of a call's launches, on lengths of zero."""
    i32 = dict(dtype=torch.int32, device="cuda")
    q, kp = torch.zeros(T * hq * hd, device="cuda").half(), torch.zeros(hk * 32 * hd, device="cuda").half()
    table, cu, kv, out = torch.zeros(B * (max_kv // 32 + 1), **i32), torch.zeros(B + 1, **i32), torch.zeros(B, **i32), torch.zeros(hk * 32, device="cuda")
    ws = torch.empty(sdamd.paged_weights_ws(B, T, max_new, max_kv, hq, hk, hd, observers) + 16, dtype=torch.uint8, device="cuda")
    return [b for _, b in launches(sdamd, lambda st: sdamd.op_paged_weights(
        q.data_ptr(), kp.data_ptr(), table.data_ptr(), max_kv // 32 + 1, cu.data_ptr(), kv.data_ptr(), B, T, max_new, max_kv, hq, hk, hd, 32, 1, None,
        out.data_ptr(), ws.data_ptr(), ws.numel(), 0, decay=0.0, observers=observers, stream=st))]


def test_which_kernels(sdamd):
    """Both sides of each rule's line: a head per workgroup (512 threads), splits (128, and their sum 256), many rows (256 ...)."""
    one, splits = [512], [128, 256]
    assert few_launches(sdamd, 1, 1, 1, 512, 8, 2, 256) == one and few_launches(sdamd, 1, 1, 1, 513, 8, 2, 256) == splits
    assert few_launches(sdamd, 16, 16, 1, 4096, 32, 8, 128) == one and few_launches(sdamd, 16, 16, 1, 4097, 32, 8, 128) == splits
    assert few_launches(sdamd, 32, 32, 1, 8192, 32, 8, 128) == one and few_launches(sdamd, 32, 32, 1, 8193, 32, 8, 128) == splits
    assert few_launches(sdamd, 32, 32, 1, 8192, 40, 8, 128) == splits  # (5 rows of 8192 scores are more than LDS takes)
    assert few_launches(sdamd, 4, 32, 8, 300, 8, 2, 128) == one and len(few_launches(sdamd, 4, 36, 9, 300, 8, 2, 128)) >= 2
    assert few_launches(sdamd, 4, 400, 100, 300, 8, 2, 128, observers=8) == one
    assert few_launches(sdamd, 4, 101, 100, 300, 8, 2, 128)[-1] == 512  # (single tokens among chunks)


def test_replayed_with_other_lengths(sdamd):
    """One captured call under bounds, the lengths changed between the replays."""
    B, hq, hk, hd, ps, blocks = 3, 8, 2, 128, 32, 20
    n_pages = B * blocks
    table = pr.dev(np.random.default_rng(1).permutation(n_pages).reshape(B, blocks))
    kp = torch.randn(n_pages * hk * ps * hd, device="cuda").half()
    T, max_new, max_kv = 60, 50, blocks * ps
    q = torch.randn(T, hq, hd, device="cuda").half()
    cu, kv, pos = pr.dev([0, 0, 0, 0]), pr.dev([0, 0, 0]), pr.dev(np.arange(T))
    scores, kpos = torch.rand(n_pages, hk, ps, device="cuda"), torch.zeros(n_pages, hk, ps, dtype=torch.int32, device="cuda")
    ws = torch.empty(sdamd.paged_weights_ws(B, T, max_new, max_kv, hq, hk, hd, 8), dtype=torch.uint8, device="cuda")

    def call(s, out):
        sdamd.op_paged_weights(q.data_ptr(), kp.data_ptr(), table.data_ptr(), blocks, cu.data_ptr(), kv.data_ptr(), B, T, max_new, max_kv, hq, hk, hd,
                               ps, n_pages, scores.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(), 0, observers=8, pos=pos.data_ptr(),
                               kpos=kpos.data_ptr(), stream=s)

    out = torch.zeros_like(scores)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        call(torch.cuda.current_stream().cuda_stream, out)
    for news, old in (([1, 1, 1], [5, 600, 33]), ([50, 1, 3], [100, 1, 0]), ([0, 9, 0], [0, 631, 7]), ([20, 20, 20], [620, 0, 64])):
        cu.copy_(pr.dev(np.concatenate([[0], np.cumsum(news)])))
        kv.copy_(pr.dev([o + n for o, n in zip(old, news)]))
        want = torch.zeros_like(out)
        call(None, want)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("requests,most,hk", [(64, 4000, 8), (33, 8192, 8), (300, 4900, 1)])
def test_longest_first(sdamd, requests, most, hk):
    """More heads than run at once, of many lengths, some of them equal, some of none: each request is done once."""
    rng = np.random.default_rng(requests)
    old = rng.integers(0, 300, requests)
    old[rng.integers(0, requests, requests // 3)] = 100
    old[[2, requests - 1]] = most - 1, most // 2
    new = rng.choice([0, 1, 1, 1], requests)
    new[[2, requests - 1]] = 1
    s = Step(requests, old.tolist(), new.tolist(), 2 * hk, hk, 64 if hk == 1 else 128, 32, "bf16")
    s.run(sdamd)
    s.check()


def test_two_streams(sdamd):
    """Two calls at once, a workspace each."""
    steps = [Step(30 + i, [4000, 900], [1 + 30 * i, 1], 8, 2, 128, 64, "f16") for i in range(2)]
    want = [s.run(sdamd).clone() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for s, st in zip(steps, streams):
            s.run(sdamd, stream=st.cuda_stream, ws=s.ws, out=s.out.fill_(-7.0), kpos=s.kpos)
            st.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    for s, w in zip(steps, want):
        s2 = s.run(sdamd)
        assert torch.equal(s2, w)


# ---- the rows that go -----------------------------------------------------------------------------

def run_evict(sdamd, scores, kpos, table, lens, budgets, hk, ps, n_pages, sink=0, recent=0, max_kv=None, stream=None):
    B, max_kv = len(lens), max_kv or max(max(lens), 1)
    width = max(max_kv // 2, 1)
    table = np.concatenate([table, np.full((B, max(0, -(-max_kv // ps) - table.shape[1])), -3)], 1)
    out = [torch.full((B,), -4, dtype=torch.int32, device="cuda"), torch.full((B * hk * width + 1, 2), -4, dtype=torch.int32, device="cuda"),
           torch.full((B * hk + 1,), -4, dtype=torch.int32, device="cuda")]
    need = sdamd.page_evict_ws(B, max_kv, hk)
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    args = [scores, kpos, pr.dev(table), pr.dev(lens), pr.dev(budgets)]
    sdamd.op_page_evict(scores.data_ptr(), None if kpos is None else kpos.data_ptr(), args[2].data_ptr(), table.shape[1], args[3].data_ptr(),
                        args[4].data_ptr(), B, max_kv, hk, ps, n_pages, sink, recent, out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(),
                        ws.data_ptr(), need, stream=stream)
    torch.cuda.synchronize()
    assert (ws[need:] == 0xFF).all()
    assert (out[1][-1] == -4).all() and int(out[2][-1]) == -4
    return out[0].tolist(), out[1][:-1].view(B, hk, width, 2).cpu().numpy(), out[2][:-1].view(B, hk).cpu().numpy()


def check_evict(sdamd, seed, lens, budgets, hk, ps, sink=0, recent=0, values="normal", max_kv=None, with_kpos=True, holes=()):
    rng = np.random.default_rng(seed)
    table, n_pages = pr.tables(rng, lens, ps)
    for b, i in holes:
        table[b, i] = -1
    shape = (n_pages, hk, ps)
    s = {"normal": lambda: rng.standard_normal(shape), "few": lambda: rng.integers(0, 3, shape), "equal": lambda: np.ones(shape),
         "zeros": lambda: np.where(rng.random(shape) < 0.5, 0.0, -0.0), "wide": lambda: np.exp(rng.standard_normal(shape) * 15),
         "odd": lambda: rng.choice([math.nan, -math.inf, math.inf, 0.0, -0.0, 1.0, -1e-45, 1e-45, 3e38, -3e38], shape),
         "close": lambda: (np.float32(1.0).view(np.int32) + rng.integers(0, 300, shape)).astype(np.int32).view(np.float32)}[values]().astype(np.float32)
    kpos = rng.integers(0, max(4 * max(lens), 1), shape).astype(np.int32) if with_kpos else None
    max_kv_ = max_kv or max(max(lens), 1)
    new, moves, counts = run_evict(sdamd, torch.from_numpy(s).cuda(), None if kpos is None else torch.from_numpy(kpos).cuda(), table, lens, budgets, hk,
                                   ps, n_pages, sink, recent, max_kv)
    for b, (n, m) in enumerate(zip(lens, budgets)):
        goes = 0 <= m < n <= max_kv_
        assert new[b] == (m if goes else n)
        j = np.arange(n)
        page = table[b, j // ps] if n else j
        hole = (page < 0) | (page >= n_pages)
        for h in range(hk):
            want = []
            if goes:
                x, p = s[page, h, j % ps], kpos[page, h, j % ps] if with_kpos else j
                want = er.evict(x, p, n, m, sink, recent, hole)
            assert counts[b, h] == len(want), (b, h)
            assert [tuple(v) for v in moves[b, h, :len(want)]] == want, (b, h)
            assert (moves[b, h, len(want):] == -4).all()


@pytest.mark.parametrize("values", ["normal", "few", "equal", "zeros", "wide", "odd", "close"])
@pytest.mark.parametrize("sink,recent", [(0, 0), (4, 32), (100, 0), (0, 1000)])
def test_evict(sdamd, values, sink, recent):
    check_evict(sdamd, 1, [1, 2, 33, 64, 257, 1000, 0, 1500, 300], [0, 1, 32, 63, 100, 999, 0, -1, 300], 2, 32, sink, recent, values)


@pytest.mark.parametrize("n,m", [(1, 0), (2, 1), (1023, 512), (1024, 1), (1025, 1024), (2049, 0), (4097, 4096), (8192, 4095), (16385, 8000), (33000, 100), (70001, 65536)])
def test_evict_lengths(sdamd, n, m):
    check_evict(sdamd, n, [n, max(1, n // 3)], [m, m], 1 if n > 20000 else 3, 64, 3, min(m // 2, 100))
    check_evict(sdamd, n + 1, [n], [m], 1, 256, values="few", with_kpos=False)


def test_evict_many_long(sdamd):
    """More heads than leave CUs idle, of more rows than one workgroup takes: larger chunks."""
    check_evict(sdamd, 9, [33001, 5, 40000, 16385, 8192, 0, 32769, 700, 24577], [100, 2, 39999, 8192, 8192, 0, 30000, 699, 0], 2, 128, 3, 500, "few")


@pytest.mark.parametrize("requests,hk,long,bound", [(66, 2, 45001, 131072), (300, 2, 36000, 40000), (8, 2, 300001, 300001)])
@pytest.mark.parametrize("values", ["normal", "few"])
def test_evict_far_bound(sdamd, requests, hk, long, bound, values):
    """Fewer workgroups for a head than chunks that a request may have."""
    rng = np.random.default_rng(10)
    lens = rng.integers(0, 500, requests)
    lens[[1, requests - 2]] = long, long // 3
    check_evict(sdamd, 11, lens.tolist(), (lens * 2 // 3).tolist(), hk, 128, 4, 20, values, max_kv=bound)


def test_evict_all_protected(sdamd):
    check_evict(sdamd, 3, [100, 500], [10, 20], 2, 32, sink=1 << 20)
    check_evict(sdamd, 4, [100, 500], [10, 20], 2, 32, recent=2 ** 31 - 1)


def test_evict_bound_below_a_request(sdamd):
    """A request of more rows than max_kv is left as it is."""
    check_evict(sdamd, 5, [100, 500], [10, 20], 2, 32, max_kv=499)
    check_evict(sdamd, 5, [100, 500], [10, 20], 2, 32, max_kv=40000)


def test_evict_holes(sdamd):
    check_evict(sdamd, 6, [300, 500], [100, 200], 2, 32, holes=[(0, 0), (0, 5), (1, 3), (1, 15)])
    check_evict(sdamd, 7, [64], [10], 1, 32, recent=5, holes=[(0, 0), (0, 1)])


def test_evict_many_requests(sdamd):
    rng = np.random.default_rng(8)
    lens = rng.integers(0, 90, 700).tolist()
    check_evict(sdamd, 8, lens, [int(x) for x in rng.integers(-1, 90, 700)], 2, 32, 2, 8, values="few")


@pytest.mark.parametrize("max_kv", [512, 40000])
def test_evict_replayed_with_other_lengths(sdamd, max_kv):
    """Eviction, moves and release in one captured graph: lengths, budgets and scores change between the replays."""
    B, hk, hd, ps = 3, 2, 64, 64
    blocks = -(-max_kv // ps)
    n_pages = B * blocks
    rng = np.random.default_rng(21)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = pr.dev(rng.permutation(n_pages).reshape(B, blocks))
    kv, budgets, dropped, n_free = torch.zeros(B, **i32), torch.zeros(B, **i32), pr.dev([1, 2, 3]), torch.zeros(1, **i32)
    state = [torch.zeros(n_pages * hk * ps * hd, device="cuda").half() for _ in range(2)] + [torch.zeros(n_pages, hk, ps, device="cuda"),
                                                                                             torch.zeros(n_pages, hk, ps, **i32)]
    out = [torch.zeros(B, **i32), torch.zeros(B, hk, max_kv // 2, 2, **i32), torch.zeros(B, hk, **i32), torch.zeros(B, **i32), torch.zeros(1, **i32),
           torch.zeros(n_pages, **i32)]
    ws = torch.full((max(sdamd.page_evict_ws(B, max_kv, hk), 16),), 0xFF, dtype=torch.uint8, device="cuda")
    p = lambda x: x.data_ptr()

    def call(stream, state, out):
        k, v, scores, kpos = state
        new, moves, counts, gone, left, free = out
        sdamd.op_page_evict(p(scores), p(kpos), p(table), blocks, p(kv), p(budgets), B, max_kv, hk, ps, n_pages, 2, 5, p(new), p(moves), p(counts), p(ws),
                            ws.numel(), stream=stream)
        sdamd.op_paged_move(p(moves), p(counts), p(table), blocks, B, max_kv, hk, hd, ps, n_pages, p(k), p(v), p(scores), p(kpos), 0, stream=stream)
        sdamd.op_page_release(p(kv), p(new), p(dropped), p(table), blocks, B, ps, n_pages, p(free), p(n_free), p(gone), p(left), stream=stream)

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        call(torch.cuda.current_stream().cuda_stream, state, out)
    for lens, keep in (([max_kv, 300, 0], [max_kv // 3, 299, 4]), ([40, max_kv - 1, 512], [41, max_kv - 70, -1]), ([max_kv, max_kv, max_kv], [0, 1, 450])):
        kv.copy_(pr.dev(lens))
        budgets.copy_(pr.dev(keep))
        for t in state[:3]:
            t.normal_()
        state[3].random_(0, 1 << 20)
        for t in out:
            t.fill_(-4)
        here, want = [t.clone() for t in state], [t.clone() for t in out]
        call(None, here, want)
        torch.cuda.synchronize()
        assert want[0].tolist() == [m if 0 <= m < n else n for n, m in zip(lens, keep)] and int(want[2].sum()) > 0
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(state + out, here + want):
            assert torch.equal(a, b)


# ---- their moves and pages ------------------------------------------------------------------------

@pytest.mark.parametrize("hk,hd,ps,kind,pstride", [(2, 256, 32, "f16", 0), (3, 128, 64, "bf16", 3 * 64 * 128 + 40), (1, 64, 256, "f16", 0)])
@pytest.mark.parametrize("marks", [True, False])
def test_move(sdamd, hk, hd, ps, kind, pstride, marks):
    rng = np.random.default_rng(hd)
    lens = [1000, 3, 70, 0, 700]
    keep = [400, 2, 69, 0, 350]
    table, n_pages = pr.tables(rng, lens, ps)
    c = pr.Cache(kind, hk, hd, ps, n_pages, pstride)
    for x in (c.k, c.v):
        x.copy_(torch.randn(x.shape, device="cuda"))
    scores, kpos = torch.rand(n_pages, hk, ps, device="cuda"), torch.randint(0, 1 << 30, (n_pages, hk, ps), dtype=torch.int32, device="cuda")
    width = 500
    moves, counts = np.full((5, hk, width, 2), 5), np.zeros((5, hk), np.int64)
    for b, (n, m) in enumerate(zip(lens, keep)):
        for h in range(hk):
            k = counts[b, h] = int(rng.integers(0, min(m, n - m) + 1)) if b else min(m, n - m) - h
            moves[b, h, :k, 0] = np.sort(rng.choice(m, k, replace=False)) if k else 0
            moves[b, h, :k, 1] = m + np.sort(rng.choice(n - m, k, replace=False)) if k else 0
    wk, wv, wsc, wp = c.k.clone(), c.v.clone(), scores.clone(), kpos.clone()
    ref = pr.Cache.__new__(pr.Cache)
    ref.__dict__.update(c.__dict__, k=wk, v=wv)
    kk, vv = ref.views()
    for b in range(5):
        for h in range(hk):
            for to, fr in moves[b, h, :counts[b, h]]:
                p, q = int(table[b, to // ps]), int(table[b, fr // ps])
                kk[p, h, to % ps // 32, :, to % 32] = kk[q, h, fr % ps // 32, :, fr % 32]
                vv[p, h, to % ps // 32, :, to % 32] = vv[q, h, fr % ps // 32, :, fr % 32]
                if marks:
                    wsc[p, h, to % ps], wp[p, h, to % ps] = wsc[q, h, fr % ps], wp[q, h, fr % ps]
    args = [pr.dev(moves), pr.dev(counts), pr.dev(table)]
    for _ in range(2):  # (the second time over changes nothing: what is read lies behind what is written)
        sdamd.op_paged_move(args[0].data_ptr(), args[1].data_ptr(), args[2].data_ptr(), table.shape[1], 5, 1000, hk, hd, ps, n_pages, c.k.data_ptr(),
                            c.v.data_ptr(), scores.data_ptr() if marks else None, kpos.data_ptr() if marks else None, KIND[kind], page_stride=pstride)
        for a, w in ((c.k, wk), (c.v, wv), (scores, wsc), (kpos, wp)):
            assert torch.equal(a, w)


def test_move_passes_over_what_is_not_there(sdamd):
    ps, hk, hd = 32, 1, 64
    c = pr.Cache("f16", hk, hd, ps, 4)
    c.k.normal_(), c.v.normal_()
    wk, wv = c.k.clone(), c.v.clone()
    table = pr.dev([[0, -1, 9, 2]])
    moves = torch.full((1, 1, 64, 2), 77, dtype=torch.int32, device="cuda")
    bad = [(-1, 100), (0, 128), (3, -5), (40, 100), (1, 70), (64, 100), (2 ** 31 - 1, 3), (-2 ** 31, 2)]
    moves[0, 0, :len(bad)] = pr.dev(bad)
    counts = pr.dev([[len(bad)]])
    call = lambda: sdamd.op_paged_move(moves.data_ptr(), counts.data_ptr(), table.data_ptr(), 4, 1, 128, hk, hd, ps, 4, c.k.data_ptr(), c.v.data_ptr(),
                                       None, None, 0)
    call()
    assert torch.equal(c.k, wk) and torch.equal(c.v, wv)
    counts.fill_(-3)
    call()
    assert torch.equal(c.k, wk) and torch.equal(c.v, wv)
    counts.fill_(2 ** 31 - 1)  # more than the array holds: its own are looked at
    moves.fill_(-1)
    call()
    assert torch.equal(c.k, wk) and torch.equal(c.v, wv)


@pytest.mark.parametrize("B,ps,most", [(1, 32, 40), (9, 64, 3000), (300, 32, 500), (8192, 32, 100), (3, 32, 100000)])
def test_release(sdamd, B, ps, most):
    rng = np.random.default_rng(B)
    kv = rng.integers(0, most, B)
    new = np.where(rng.random(B) < 0.3, kv, rng.integers(-1, most, B) % (kv + 1))
    new[rng.random(B) < 0.05] = -1
    if B > 1:
        new[0], new[1] = 0, kv[1] + 5
    table, n_pages = pr.tables(rng, kv.tolist(), ps)
    if B > 5:
        table[3, 0], table[4, table.shape[1] - 1] = -1, n_pages
    dropped = rng.integers(0, 1 << 30, B)
    free = np.full(n_pages, -6)
    n_free = int(rng.integers(0, 3))
    want = er.release(kv.tolist(), new.tolist(), dropped.tolist(), table.tolist(), ps, n_pages, free.tolist(), n_free)
    d = [pr.dev(x) for x in (kv, new, dropped, table, free, [n_free])]
    out, left = torch.full((B + 1,), -2, dtype=torch.int32, device="cuda"), pr.dev([-2, -2])
    sdamd.op_page_release(d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), d[3].data_ptr(), table.shape[1], B, ps, n_pages, d[4].data_ptr(),
                          d[5].data_ptr(), out.data_ptr(), left.data_ptr())
    assert out.tolist() == want[0] + [-2] and left.tolist() == [want[2], -2]
    assert d[4].tolist() == want[1]


def test_release_of_more_than_the_stack_holds(sdamd):
    d = [pr.dev(x) for x in ([96, 96], [0, 0], [0, 0], [[0, 1, 2], [0, 1, 2]], [9, 9, 9, 9], [2])]
    out, left = pr.dev([0, 0]), pr.dev([0])
    sdamd.op_page_release(d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), d[3].data_ptr(), 3, 2, 32, 4, d[4].data_ptr(), d[5].data_ptr(),
                          out.data_ptr(), left.data_ptr())
    assert d[4].tolist() == [9, 9, 0, 1] and left.tolist() == [4] and out.tolist() == [96, 96]


# ---- a run of them all ----------------------------------------------------------------------------

def test_a_serving_loop_within_budgets(sdamd):
    """Requests with a budget each, steps of prompts and single tokens: plan, positions, table, prep, attention, weights, then
    eviction, moves and release.  A plain model keeps each head's rows as a list of (position, key, value, score) and drops
    from it what the kernels' own scores tell it to; attention over it, in 64 bits, is what every step must give, every row
    that stays must be there, and no page may be lost."""
    B, hq, hk, hd, rd, ps, n_pages, blocks, T = 4, 8, 2, 128, 64, 32, 40, 12, 128
    budgets, sink, recent = [70, 40, -1, 100], 2, 8
    g = torch.Generator("cuda").manual_seed(2)
    i32 = dict(dtype=torch.int32, device="cuda")
    freqs = sdamd.rope_freqs(rd, 1e4, sdamd.ROPE_PARTS, 4.0, 64.0, 1.0, 8.0)
    fd = torch.from_numpy(freqs).cuda()
    kp, vp = (torch.full((n_pages * hk * ps * hd,), math.nan, dtype=torch.half, device="cuda") for _ in range(2))
    scores, kpos = torch.full((n_pages, hk, ps), math.nan, device="cuda"), torch.full((n_pages, hk, ps), -1, **i32)
    table, free = torch.full((B, blocks), -1, **i32), torch.arange(n_pages, **i32)
    lens, dropped, n_free = torch.zeros(B, **i32), torch.zeros(B, **i32), torch.tensor([n_pages], **i32)
    cu, kv, slots, pos, status, new_lens = (torch.zeros(n, **i32) for n in (B + 1, B, T, T, 4, B))
    rows, dbudget = torch.arange(T, **i32), pr.dev(budgets)
    max_kv = blocks * ps
    q, out, angles = torch.zeros(T, hq, hd, device="cuda").half(), torch.zeros(T, hq * hd, device="cuda").half(), torch.zeros(T, rd // 2, 2, device="cuda")
    moves, counts = torch.zeros(B, hk, max_kv // 2, 2, **i32), torch.zeros(B, hk, **i32)
    gone, left = torch.zeros(B, **i32), torch.zeros(1, **i32)
    byte = dict(dtype=torch.uint8, device="cuda")
    wsa = torch.empty(max(sdamd.paged_attention_ws(B, T, T, max_kv, hq, hk, hd), 16), **byte)
    wsw = torch.empty(sdamd.paged_weights_ws(B, T, T, max_kv, hq, hk, hd), **byte)
    wse = torch.empty(max(sdamd.page_evict_ws(B, max_kv, hk), 16), **byte)
    p = lambda x: x.data_ptr()
    model = [[[] for _ in range(hk)] for _ in range(B)]  # [position, key, value] of every row, in row order
    total = [0] * B
    for step, news in enumerate([[50, 30, 20, 0], [1, 1, 1, 90], [33, 1, 1, 1]] + [[1, 1, 1, 1]] * 4 + [[0, 20, 0, 60], [1, 0, 1, 1]]):
        dn = pr.dev(news)
        n = sum(news)
        big = torch.randn(T, (hq + 2 * hk) * hd, generator=g, device="cuda").half()
        sdamd.op_page_plan(p(lens), p(dn), B, T, ps, n_pages, p(free), p(n_free), p(table), blocks, p(cu), p(kv), p(slots), p(pos), p(status))
        assert status.tolist()[:2] == [B, n]
        n_free.copy_(status[3:])
        sdamd.op_page_positions(p(cu), p(dropped), B, T, p(pos), p(pos))
        sdamd.op_rope_table(p(fd), rd // 2, p(pos), T, p(angles), magnitude=1.1)
        sdamd.op_paged_prep(p(big), big.shape[1], False, None, None, p(angles), T, p(rows), 1, None, p(slots), T, hq, hk, hd, rd, ps, n_pages, p(q),
                            p(kp), p(vp), 0)
        sdamd.op_paged_attention(p(q), None, 0, p(kp), p(vp), p(table), blocks, p(cu), p(kv), B, T, T, max_kv, hq, hk, hd, ps, n_pages, p(out),
                                 p(wsa), wsa.numel(), 0)
        sdamd.op_paged_weights(p(q), p(kp), p(table), blocks, p(cu), p(kv), B, T, T, max_kv, hq, hk, hd, ps, n_pages, p(scores), p(scores), p(wsw),
                               wsw.numel(), 0, pos=p(pos), kpos=p(kpos))
        # the model's new rows, and the attention over what it holds
        x = big.cpu().double().view(T, -1, hd)
        at, c = 0, pr.Cache.__new__(pr.Cache)
        c.__dict__.update(hk=hk, hd=hd, ps=ps, n_pages=n_pages, pstride=hk * ps * hd, k=kp, v=vp)
        cut = [[0] * hk for _ in range(B)]
        for b in range(B):
            new = news[b]
            true = np.arange(total[b], total[b] + new)
            total[b] += new
            assert pos[at:at + new].tolist() == true.tolist()
            old = len(model[b][0])
            s = pr.slots_of(table.cpu().numpy(), b, ps, 0, old + new)
            k, v = (t.cpu().double() for t in c.rows(s)) if len(s) else (None, None)
            if new:
                want, mag = er.rope(x[at:at + new, hq:hq + hk], true, freqs, 1.1, "half", False)
                assert ((k[old:] - want).abs() <= 2.0 ** -11 * want.abs() * 1.01 + 2.0 ** -18 * mag + 2.0 ** -25).all()
                assert torch.equal(v[old:], x[at:at + new, hq + hk:])
            for h in range(hk):
                for j, (tp, kk, vv) in enumerate(model[b][h]):
                    assert torch.equal(k[j, h], kk) and torch.equal(v[j, h], vv)
                model[b][h] += [[int(true[i]), k[old + i, h], v[old + i, h]] for i in range(new)]
            if new:
                qq = q[at:at + new].cpu().double()
                o, mag, top = pr.attend(qq, k, v, old + new, hd ** -0.5)
                err = (out[at:at + new].view(new, hq, hd).cpu().double() - o).abs()
                assert (err <= pr.attend_bound("f16", o, mag, top, hd, old + new)).all()
                assert [r[0] for r in model[b][0]] == kpos.cpu()[s // ps, 0, s % ps].tolist()
            at += new
        sc = scores.cpu()
        tb = table.cpu().numpy()
        sdamd.op_page_evict(p(scores), p(kpos), p(table), blocks, p(kv), p(dbudget), B, max_kv, hk, ps, n_pages, sink, recent, p(new_lens), p(moves),
                            p(counts), p(wse), wse.numel())
        sdamd.op_paged_move(p(moves), p(counts), p(table), blocks, B, max_kv, hk, hd, ps, n_pages, p(kp), p(vp), p(scores), p(kpos), 0)
        sdamd.op_page_release(p(kv), p(new_lens), p(dropped), p(table), blocks, B, ps, n_pages, p(free), p(n_free), p(gone), p(left))
        for b in range(B):
            held = len(model[b][0])
            m = budgets[b] if 0 <= budgets[b] < held else held
            for h in range(hk):
                if m < held:
                    s = pr.slots_of(tb, b, ps, 0, held)
                    for to, fr in er.evict(sc[s // ps, h, s % ps].numpy(), [r[0] for r in model[b][h]], held, m, sink, recent):
                        model[b][h][to] = model[b][h][fr]
                model[b][h] = model[b][h][:m]
                positions = {r[0] for r in model[b][h]}
                assert len(positions) == m and set(range(max(0, total[b] - min(recent, m)), total[b])) <= positions
            assert int(gone[b]) == total[b] - m
        assert new_lens.tolist() == [len(model[b][0]) for b in range(B)]
        lens.copy_(new_lens), dropped.copy_(gone), n_free.copy_(left)
        used = [int(t) for b in range(B) for t in table[b, :-(-len(model[b][0]) // ps)]]
        assert sorted(used + free[:int(n_free)].tolist()) == list(range(n_pages))
