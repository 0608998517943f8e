"""Paged attention on the GPU with values and scores at the ends of their ranges."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from test_gpu_paged import attn_case, call  # noqa: E402


def results(d):
    """(request, want, tolerance, got) of every request that has rows."""
    got = d["out"].view(d["T"], d["hq"], d["hd"])
    for b, (kv, n) in enumerate(zip(d["kv"], d["new"])):
        if n:
            a = int(d["at"][b])
            want, mag, top = ref.attend_fast(d["q"][a:a + n].double(), d["ks"][b].double(), d["vs"][b].double(), kv, d["scale"])
            yield b, want, ref.attend_bound(d["kind"], want, mag, top, d["hd"], kv), got[a:a + n].double()


# ---- values that are seen with a weight of next to nothing, or of nothing ----

# one request whose keys are split, with a single token and with a chunk; the same unsplit
SPLIT = [("one token, split", 4, 2, 64, [(5000, 1)]), ("chunk, split", 8, 2, 128, [(5000, 40)]),
         ("one token, unsplit", 4, 2, 64, [(5000, 1)] + [(1, 1)] * 99), ("chunk, unsplit", 16, 4, 64, [(1200, 1100)])]


@pytest.mark.parametrize("far", [True, False])
@pytest.mark.parametrize("name,hq,hk,hd,reqs", SPLIT)
def test_a_seen_value_that_is_not_finite_is_never_lost(sdamd, name, hq, hk, hd, reqs, far):
    """The first keys' scores are 300 below the others' or -inf: their weights vanish in f32, in whole splits, but their
    infinities and NaN are seen, so these dims are not finite, however the keys are split.  The other dims are as ever."""
    low = 1000 if reqs[0][0] == 5000 else 64

    def poke(b, k, v):
        if b == 0:
            k[:] = 0
            k[:low, :, 0] = -300.0 if far else -math.inf
            v[7, :, 3], v[low // 2, :, 5], v[9, :, 9], v[low - 1, :, 11] = math.inf, math.nan, -math.inf, math.nan

    for kind in ("f16", "bf16"):
        d = attn_case(sdamd, kind, hq, hk, hd, 32, reqs, scale=1.0, poke=poke, seed=1)
        d["q"][:, :, 0] = 1.0
        call(sdamd, d)
        torch.cuda.synchronize()
        for b, want, tol, g in results(d):
            dims = torch.zeros(hd, dtype=torch.bool, device="cuda")
            if b == 0:
                dims[[3, 5, 9, 11]] = True
                # rows that see a key of a finite score (a row of -inf alone gives zeros)
                rows = torch.arange(len(g), device="cuda") + d["kv"][0] - len(g) >= low
                g, want, tol = g[rows], want[rows], tol[rows]
                assert int(g[..., dims].isfinite().sum()) == 0, (kind, "a seen value was lost")
                assert int((~g[..., [5, 11]].isnan()).sum()) == 0, (kind, "a seen NaN was lost")
            bad = ~((g - want).abs() <= tol)[..., ~dims]
            assert int(bad.sum()) == 0, (kind, b)


# ---- scores past the f32 integers ----

@pytest.mark.parametrize("kind,sizes", [("f16", [2.0 ** 6, 2.0 ** 11, 2.0 ** 12, 2.0 ** 13, 2.0 ** 14, 2.0 ** 15]),
                                        ("bf16", [2.0 ** 6, 2.0 ** 13, 2.0 ** 15, 2.0 ** 20, 2.0 ** 40, 2.0 ** 54])])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_of_any_size(sdamd, kind, sizes, sign):
    """Queries of `size`, keys of +-size times 1 or 5/4 and scores size^2 hd / sqrt(hd) and 5/4 of it, exact in f32: at
    this distance the lesser weights are 0, and a row's result is the mean of the values at its equal largest scores."""
    for hq, hk, hd, reqs in [(8, 2, 256, [(5000, 1)]), (4, 2, 64, [(900, 1), (300, 1)]), (8, 2, 128, [(700, 150), (65, 65)]),
                             (4, 1, 256, [(3000, 40), (90, 1)])]:
        for size in sizes:
            def poke(b, k, v):
                k[:] = sign * size
                k[-1, :, :] *= 1.25 if sign < 0 else 1.0
                k[5::29] = sign * size * (1.25 if sign > 0 else 1.0)
                k[:5] *= 1.25 if sign < 0 else 1.0
            d = attn_case(sdamd, kind, hq, hk, hd, 32, reqs, poke=poke, seed=3)
            d["q"].fill_(size)
            call(sdamd, d)
            torch.cuda.synchronize()
            got, u, e = d["out"].view(d["T"], hq, hd), ref.half_step(kind), 2.0 ** -24
            for b, (kv, n) in enumerate(zip(d["kv"], d["new"])):
                a, j = int(d["at"][b]), torch.arange(kv, device="cuda")
                s = d["ks"][b][:, 0, 0].double()
                for i in {0, n // 2, n - 1}:
                    seen = j <= kv - n + i
                    top = seen & (s == s[seen].max())
                    v = d["vs"][b][top].double().repeat_interleave(hq // hk, 1)
                    # the equal weights and the result are rounded to the type, sums are in f32 (as in attend_bound)
                    tol = u * v.mean(0).abs() + (u + (2 * kv + 16) * e) * v.abs().mean(0) * (1 + u) + 2.0 ** -25
                    bad = ~((got[a + i].double() - v.mean(0)).abs() <= tol)
                    assert int(bad.sum()) == 0, (kind, hd, reqs, size, b, i, int(bad.sum()))


# ---- values up to the type's largest ----

@pytest.mark.parametrize("hq,hk,hd", [(8, 2, 256), (4, 2, 64), (8, 2, 128)])
def test_values_up_to_the_largest(sdamd, hq, hk, hd):
    """Values of +-3e38 in bf16 and 65504 in f16 at keys whose weight is 1 (the others' are at most e^-20 in all, of
    values of the same size): the result is the value, not an infinity."""
    for kind, most in (("bf16", 3e38), ("f16", 65504.0)):
        for reqs in ([(4000, 1)], [(400, 1), (33, 1)], [(900, 200), (3, 1)], [(5000, 40)]):
            for at in (0, 1, -1):  # the key that counts: the first of all, the second, or the last of all
                def poke(b, k, v):
                    k[:] = 0
                    k[at, :, 0] = 32.0
                    v[:] = v.sign() * most
                d = attn_case(sdamd, kind, hq, hk, hd, 32, reqs, scale=1.0, poke=poke, seed=4)
                d["q"].zero_()
                d["q"][:, :, 0] = 1.0
                call(sdamd, d)
                torch.cuda.synchronize()
                got, u = d["out"].view(d["T"], hq, hd).double(), ref.half_step(kind)
                for b, (kv, n) in enumerate(zip(d["kv"], d["new"])):
                    a = int(d["at"][b])
                    # (a single row's own key is its last; the first row of a chunk sees the first keys)
                    g = got[a + n - 1] if at < 0 else got[a:a + n][torch.arange(n) + kv - n >= at]
                    want = d["vs"][b][at].double().repeat_interleave(hq // hk, 0)
                    # the weight and the result are rounded to the type; 5000 weights of e^-32, each value once more
                    tol = (2.02 * u + 2 * 5000 * math.exp(-32)) * want.abs()
                    bad = ~((g - want).abs() <= tol)
                    assert int(bad.sum()) == 0, (kind, hd, reqs, at, b, int(bad.sum()))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [1e-45, 1e-39, 1e-20])
def test_scales_that_make_all_weights_equal(sdamd, kind, scale):
    """The smallest scales (subnormal ones among them): a row's result is the mean of the values that it sees."""
    for hq, hk, hd, reqs in [(8, 2, 256, [(700, 1), (60, 50)]), (4, 2, 64, [(900, 1), (31, 1)]), (8, 2, 128, [(5000, 40)])]:
        d = attn_case(sdamd, kind, hq, hk, hd, 32, reqs, scale=scale, seed=5)
        call(sdamd, d)
        torch.cuda.synchronize()
        for b, want, tol, g in results(d):
            bad = ~((g - want).abs() <= tol)
            assert int(bad.sum()) == 0, (kind, hd, b, int(bad.sum()))
