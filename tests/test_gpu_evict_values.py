"""The weight that every cached key receives where scores are far from 1, sums are long, and work is cut: keys and rows are
chosen so that every weight is known.  Rows that go among infinite scores.  Calls on two streams at once."""
import math

import numpy as np
import pytest
import torch

import evict_ref as er
import paged_ref as pr
from test_gpu_evict import KIND, Step, run_evict

pytestmark = pytest.mark.gpu


def given(step, keys, rows):
    """The step's keys of each request [kv][hk][hd], and its queries [T][hq][hd], in place of random ones."""
    step.k = [k.to("cuda", pr.DT[step.kind]) for k in keys]
    for b, k in enumerate(step.k):
        step.cache.put(pr.slots_of(step.table, b, step.ps, 0, len(k)), k, torch.zeros_like(k))
    step.q = rows.to("cuda", pr.DT[step.kind])


def weights_of(step, b):
    """[kv][hk] of request b, f64 on the CPU."""
    s = torch.as_tensor(pr.slots_of(step.table, b, step.ps, 0, step.kv[b]))
    return step.out.cpu()[s // step.ps, :, s % step.ps].double()


# ---- scores of any size, rows of any neighbours ----------------------------------------------------

def one_hot(rng, old, n, hq, hd, kind, window=0):
    """64 rows, each with a dim of its own, and keys that have the 64 dims in turn: row r's scores are a_r on its keys and 0 on
    the others, some 2^16 to 2^22.8 in base 2, so that its n keys share its weight and the others get none."""
    s = Step(3, [old], [n], hq, 1, hd, 32, kind, decay=0.0, scale=500.0, window=window)
    kv, g = old + n, hq
    assert n * g == 64
    j, r = torch.arange(kv), torch.arange(64)
    k, q = torch.zeros(kv, 1, hd), torch.zeros(64, hd)
    k[j, 0, j % 64] = 1.0
    q[r, r] = torch.from_numpy(np.exp(rng.uniform(math.log(100), math.log(10000), 64))).float()
    p = old + r // g
    sees = (j[None] <= p[:, None]) & ((j[None] > (p - window)[:, None]) if window else True)
    own = sees & (j[None] % 64 == r[:, None])
    return s, k, q, sees, own


@pytest.mark.parametrize("late", [False, True])
@pytest.mark.parametrize("loud", [0, 17, 31, 40, 63])
@pytest.mark.parametrize("old,n,hq,hd,kind", [(100, 64, 1, 64, "f16"), (3000, 64, 1, 128, "f16"), (100, 16, 4, 256, "bf16"), (3000, 16, 4, 64, "bf16")])
def test_a_loud_row_leaves_the_others(sdamd, loud, old, n, hq, hd, kind, late):
    """A row's weights are what it gives alone, whatever the size of the scores of the rows beside it."""
    s, k, q, sees, own = one_hot(np.random.default_rng(loud), old, n, hq, hd, kind)
    q[loud] *= 60000.0 / q[loud, loud]  # 2^25.3
    if late:  # (its keys behind others')
        k[:old // 2, 0, loud] = 0.0
        own[loud] &= torch.arange(old + n) >= old // 2
    given(s, [k], q.view(n, hq, hd))
    s.run(sdamd)
    want = (own / own.sum(1, keepdim=True)).double().sum(0)
    # (equal scores: exponentials of 0, a whole number as the sum; its reciprocal within a step and a half, nothing else added)
    assert ((weights_of(s, 0)[:, 0] - want).abs() <= 4 * er.E32 * want).all()


@pytest.mark.parametrize("loud", [0, 8, 20, 40])
@pytest.mark.parametrize("old,hd", [(200, 64), (1000, 256)])
def test_an_infinite_row_leaves_the_others(sdamd, loud, old, hd):
    """Keys that a row with infinite scores sees become NaN; the weights of all others are what they are without it."""
    s, k, q, sees, own = one_hot(np.random.default_rng(loud), old, 64, 1, hd, "f16", window=64)
    q[loud] = math.inf
    given(s, [k], q.view(64, 1, hd))
    s.run(sdamd)
    got, want = weights_of(s, 0)[:, 0], (own / own.sum(1, keepdim=True)).double().sum(0)
    assert torch.equal(torch.isnan(got), sees[loud])
    assert (want > 0)[~sees[loud]].any()
    assert ((got - want).abs() <= 4 * er.E32 * want)[~sees[loud]].all()


@pytest.mark.parametrize("rising", [True, False])
@pytest.mark.parametrize("old,n,hq,hd", [(200, 40, 1, 64), (700, 16, 4, 128), (2500, 64, 2, 256)])
def test_scores_around_2_to_23(sdamd, old, n, hq, hd, rising):
    """Scores that are whole numbers around 6 million, steps of 1.4 in base 2 around 2^23: rows on both sides of it, and rows
    whose maximum passes it from one block of keys to the next."""
    scale = np.float32(8388608 / 6e6 * math.log(2))
    s = Step(4, [old], [n], hq, 1, hd, 32, "f16", decay=0.0, scale=float(scale))
    kv = old + n
    rng = np.random.default_rng(old)
    t = np.sort(rng.integers(-12, 13, kv))
    k, q = torch.zeros(kv, 1, hd), torch.zeros(n, hq, hd)
    k[:, 0, 0], k[:, 0, 1] = 100.0, torch.from_numpy(t if rising else t[::-1].copy()).float()
    q[..., 0], q[..., 1] = torch.from_numpy(rng.choice([59968.0, 60000.0, 60000.0, 60032.0], (n, hq))).float(), 1.0
    given(s, [k], q)
    s.run(sdamd)
    want, _ = er.weights(q.double(), k.double(), kv, float(scale))
    # scores and their differences are exact (below 2^24); up to 34 in base 2, times c of two roundings, one more, and an exponential
    # within 2 steps, in numerator and sum; sums of kv keys and of the rows, and a few more
    rel = 2 * (34 * 3 * math.log(2) + 2) + kv + n * hq + 16
    assert ((weights_of(s, 0)[:, 0] - want[0]).abs() <= rel * er.E32 * want[0] + 2.0 ** -126).all()


# ---- long sums -------------------------------------------------------------------------------------

def one_key_stands_out(sdamd, old, new, hq, hk, hd, at, depth, score, **kw):
    """Request `at` has one key of score x and others of 0: each row's sum is 1 and e^-x for every other key that it sees."""
    s = Step(5, old, new, hq, hk, hd, 128, "f16", decay=0.0, scale=0.125)
    keys = [torch.zeros(kv, hk, hd) for kv in s.kv]
    keys[at][0, :, 0] = 1.0
    q = torch.zeros(s.T, hq, hd)
    q[..., 0] = 8.0 * score
    given(s, keys, q)
    s.run(sdamd, **kw)
    j = np.arange(s.kv[at])
    total = np.zeros(len(j))
    for p in range(old[at], s.kv[at]):
        total[:p + 1] += hq // hk / (1 + p * math.exp(-score))
    want = torch.from_numpy(np.where(j == 0, 1.0, math.exp(-score)) * total)[:, None]
    # an exponent of 1.44 x in base 2 that has 3 roundings, an exponential within 2 steps, in a row's sum and in the weight; a block's sum
    # in pairs (5), with what the roundings leave out carried along (3), joined (12), a reciprocal, a product; `depth` rows added in turn
    rel = (2 * (3 * score + 2) + 5 + 3 + 12 + 3 + depth) * er.E32
    assert ((weights_of(s, at) - want).abs() <= rel * want).all(), float(((weights_of(s, at) - want).abs() / want).max() / er.E32)


@pytest.mark.parametrize("hd,score", [(64, 8), (128, 8), (256, 6)])
def test_long_sums_of_many_rows(sdamd, hd, score):
    """So many rows that no split of the keys is needed to fill the GPU: 32 thousand of a row's exponentials in one lane's sum."""
    one_key_stands_out(sdamd, [65536], [2048], 128, 8, hd, 0, 512 + 4, score)  # (parts of 16384 rows, 32 at a time, and the parts)


@pytest.mark.parametrize("score", [5, 6, 8, 9, 10])
def test_long_sums_of_single_tokens(sdamd, score):
    """So many requests that a head's keys are not split, one of them long."""
    rng = np.random.default_rng(1)
    old = rng.integers(0, 50, 1024)
    old[517] = 70000
    one_key_stands_out(sdamd, old.tolist(), [1] * 1024, 8, 8, 64, 517, 1, score)


# ---- work that is cut ------------------------------------------------------------------------------

@pytest.mark.parametrize("new,max_new,max_kv", [([1] * 40, 1, 20000), ([8] * 20, 8, 9000), ([1] * 30 + [70, 0, 9], 70, 30000)])
def test_workspaces_that_hold_some_requests(sdamd, new, max_new, max_kv):
    """With a smaller workspace requests go in turn, to the same bits; nothing behind it is written."""
    rng = np.random.default_rng(max_kv)
    old = rng.integers(0, 400, len(new))
    old[[3, len(new) - 1]] = 8500
    s = Step(6, old.tolist(), new, 8, 2, 128, 32, "bf16", decay=0.5)
    kw = dict(max_new=max_new, max_kv=max_kv)
    want = s.run(sdamd, **kw).clone()
    s.check()
    full = s.ws.numel() - 64
    with pytest.raises(sdamd.EngineError, match="at least") as e:
        s.run(sdamd, ws=torch.zeros(64, dtype=torch.uint8, device="cuda"), **kw)
    least = int(str(e.value).split("at least ")[1].split(",")[0])
    assert 0 < least < full
    for size in (least, least + 16, (full + least) // 2 & ~15, full - 16):
        ws = torch.full((size + 64,), 0xFF, dtype=torch.uint8, device="cuda")
        assert torch.equal(s.run(sdamd, ws=ws, **kw), want)
        assert (ws[size:] == 0xFF).all()
    with pytest.raises(sdamd.EngineError, match="at least"):
        s.run(sdamd, ws=torch.zeros(least + 48, dtype=torch.uint8, device="cuda"), **kw)


def spotted(sdamd, old, new, hq, hk, hd, depth, ps=128, **kw):
    """Keys of scores 0 to 3, each head's its own: every weight follows from running sums, and a key that is left out, counted twice or
    taken for another moves all of a row's."""
    s = Step(8, old, new, hq, hk, hd, ps, "f16", decay=0.0, scale=0.125)
    rng = np.random.default_rng(len(old) + sum(new))
    levels = [rng.integers(0, 4, (kv, hk)) for kv in s.kv]
    keys = []
    for x in levels:
        k = torch.zeros(len(x), hk, hd)
        k[:, :, 0] = torch.from_numpy(x)
        keys.append(k)
    q = torch.zeros(max(s.T, 1), hq, hd)
    q[..., 0] = 8.0
    given(s, keys, q)
    s.run(sdamd, **kw)
    # as above: exponents of 4.3 at most
    rel = (2 * (3 * 3 + 2) + 5 + 3 + 12 + 3 + depth) * er.E32
    for b, (o, n, x) in enumerate(zip(old, new, levels)):
        if n == 0:
            continue
        e = np.exp(x.astype(np.float64))
        each = hq / hk / np.cumsum(e, 0)[o:]  # of the rows, one by one
        rest = np.cumsum(each[::-1], 0)[::-1]
        want = torch.from_numpy(e * np.concatenate([np.broadcast_to(rest[:1], (o, hk)), rest]))
        got = weights_of(s, b)
        assert ((got - want).abs() <= rel * want).all(), (b, float(((got - want).abs() / want).max() / er.E32), rel / er.E32)
    return s


@pytest.mark.parametrize("old,new,hq,hk,hd,depth", [
    ([30011, 9000], [1, 1], 8, 2, 128, 4),  # splits
    ([8000, 5000, 1, 0] * 10, [1] * 40, 16, 8, 64, 2),  # scores in LDS
    ([30011, 9000], [40, 1], 8, 2, 256, 8),  # tiles of rows in splits, beside a single token
    ([70000] + [40] * 1023, [1] * 1024, 8, 8, 64, 1),  # more than 64 blocks of a wave
    ([65536], [2048], 128, 8, 64, 516),  # more than 32 blocks of a tile's split
    ([500, 3, 0, 80] * 10, [60, 300, 129, 65] * 10, 8, 2, 64, 16),  # requests of several parts, one behind the other
])
def test_every_key_counts(sdamd, old, new, hq, hk, hd, depth):
    spotted(sdamd, old, new, hq, hk, hd, depth)


@pytest.mark.parametrize("old,new,hq,depth", [(300000, 40, 8, 4), (266000, 4200, 32, 516)])
@pytest.mark.parametrize("bound", [None, 2200000])
def test_more_key_tiles_than_workgroups(sdamd, old, new, hq, depth, bound):
    """2344 tiles of 8 heads, with one part of the rows and with two; under the far bound a workgroup takes several."""
    spotted(sdamd, [old], [new], hq, 8, 64, depth, max_kv=bound)


def test_chunks_of_many_requests_under_a_far_bound(sdamd):
    """2048 requests with a few rows each, bounds of 4096 rows and 131072 keys for any of them."""
    rng = np.random.default_rng(2)
    old = rng.integers(0, 60, 2048)
    old[[0, 1000, 2047]] = 1500, 9000, 20000
    kw = dict(max_new=4096, max_kv=131072)
    new = rng.integers(1, 8, 2048).tolist()
    least = 34 * 131072 * 8 * 4 + (64 << 20)
    spotted(sdamd, old.tolist(), new, 32, 8, 64, 8, ws=torch.zeros(least, dtype=torch.uint8, device="cuda"), **kw)


# ---- rows that go, among infinite scores ------------------------------------------------------------

@pytest.mark.parametrize("n,m", [(2, 1), (300, 40), (5000, 1200), (20000, 3000), (40000, 9000)])
@pytest.mark.parametrize("sink,recent", [(0, 0), (1, 0), (20, 300), (0, 5000)])
def test_protected_rows_come_before_infinite_scores(sdamd, n, m, sink, recent):
    """Protected rows, then +inf, then numbers, -inf, NaN: with more protected and infinite rows than the budget, too."""
    rng = np.random.default_rng(n + sink + recent)
    ps, hk = 128, 2
    table, n_pages = pr.tables(rng, [n], ps)
    scores = rng.choice(np.array([math.inf, math.inf, 1.0, 2.0, -math.inf, math.nan], np.float32), (n_pages, hk, ps))
    kpos = rng.integers(0, 2 * n, (n_pages, hk, ps)).astype(np.int32)
    new, moves, counts = run_evict(sdamd, torch.from_numpy(scores).cuda(), torch.from_numpy(kpos).cuda(), table, [n], [m], hk, ps, n_pages, sink, recent)
    assert new == [m]
    j = np.arange(n)
    for h in range(hk):
        x, p = scores[table[0, j // ps], h, j % ps].astype(np.float64), kpos[table[0, j // ps], h, j % ps]
        safe = (p < sink) | (p > int(p.max()) - recent)
        order = np.lexsort((j, -np.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf), np.where(safe, 0, np.where(np.isnan(x), 2, 1))))
        # (nothing else decides between protected rows, or between NaN, than their order)
        order = np.concatenate([j[safe], order[~safe[order] & ~np.isnan(x[order])], j[~safe & np.isnan(x)]])
        kept = np.zeros(n, bool)
        kept[order[:m]] = True
        want = np.stack([j[:m][~kept[:m]], j[m:][kept[m:]]], 1)
        assert counts[0, h] == len(want) and (moves[0, h, :len(want)] == want).all()


# ---- calls on two streams at once -------------------------------------------------------------------

def on_two_streams(calls, outs, again):
    """calls[i](stream) fills outs[i]; each of them in turn on a stream of its own, without a wait between, ends as it does alone."""
    want = []
    for call, out in zip(calls, outs):
        again()
        torch.cuda.synchronize()
        call(None)
        torch.cuda.synchronize()
        want.append([t.clone() for t in out])
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        again()
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
        for _ in range(3):  # (each call's outputs are the same every time)
            for call, st in zip(calls, streams):
                call(st.cuda_stream)
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))


@pytest.mark.parametrize("new,old", [(([1, 1], [31, 1]), [4000, 900]), (([60, 1], [200, 90]), [9000, 3000]), (([1] * 40, [1] * 40), [2000] * 40)])
def test_weights_on_two_streams(sdamd, new, old):
    steps = [Step(30 + i, old, n, 8, 2, 128, 64, "f16") for i, n in enumerate(new)]
    outs, calls = [], []
    for s in steps:
        s.run(sdamd)
        s.check()
        outs.append([s.out, s.kpos])

        def call(stream, s=s):
            B = len(s.old)
            sdamd.op_paged_weights(s.q.data_ptr(), s.cache.k.data_ptr(), s.dtable.data_ptr(), s.dtable.shape[1], s.cu.data_ptr(), s.lens.data_ptr(), B,
                                   s.T, max(s.new), max(s.kv), s.hq, s.hk, s.hd, s.ps, s.n_pages, s.scores.data_ptr(), s.out.data_ptr(),
                                   s.ws.data_ptr(), s.ws.numel(), KIND[s.kind], pos=s.pos.data_ptr(), kpos=s.kpos.data_ptr(), stream=stream)

        calls.append(call)

    def again():
        for s in steps:
            s.out.fill_(-7.0), s.kpos.fill_(-9), s.ws.fill_(0xFF)

    on_two_streams(calls, outs, again)


@pytest.mark.parametrize("n", [3000, 40000])
def test_eviction_and_moves_on_two_streams(sdamd, n):
    rng = np.random.default_rng(n)
    ps, hk, hd, m = 64, 2, 64, n // 3
    i32 = dict(dtype=torch.int32, device="cuda")
    p = lambda t: t.data_ptr()
    calls, outs, keep = [], [], []
    for _ in range(2):
        table, n_pages = pr.tables(rng, [n, n - 7], ps)
        tb, kv, budgets = pr.dev(table), pr.dev([n, n - 7]), pr.dev([m, m + 5])
        scores, kpos = torch.rand(n_pages, hk, ps, device="cuda"), torch.randint(0, n, (n_pages, hk, ps), **i32)
        first = [torch.randn(n_pages * hk * ps * hd, device="cuda").half() for _ in range(2)]
        caches = [t.clone() for t in first]
        out = [torch.zeros(2, **i32), torch.zeros(2, hk, n // 2, 2, **i32), torch.zeros(2, hk, **i32)]
        ws = torch.zeros(max(sdamd.page_evict_ws(2, n, hk), 16), dtype=torch.uint8, device="cuda")
        keep.append((out, ws, first, caches))

        def call(stream, tb=tb, kv=kv, budgets=budgets, scores=scores, kpos=kpos, out=out, ws=ws, caches=caches, n_pages=n_pages):
            sdamd.op_page_evict(p(scores), p(kpos), p(tb), tb.shape[1], p(kv), p(budgets), 2, n, hk, ps, n_pages, 3, 20, p(out[0]), p(out[1]), p(out[2]),
                                p(ws), ws.numel(), stream=stream)
            sdamd.op_paged_move(p(out[1]), p(out[2]), p(tb), tb.shape[1], 2, n, hk, hd, ps, n_pages, p(caches[0]), p(caches[1]), None, None, 0, stream=stream)

        calls.append(call)
        outs.append(out + caches)

    def again():
        for out, ws, first, caches in keep:
            ws.fill_(0xFF)
            for t in out:
                t.fill_(-4)
            for a, b in zip(caches, first):
                a.copy_(b)

    on_two_streams(calls, outs, again)
