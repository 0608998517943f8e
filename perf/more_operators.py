"""Streams that outlive their cache, as cases that can be timed and compared.

A program that serves many requests from a paged key/value cache bounds each request's rows: it adds up the attention
weight that every cached key receives (`weights`), picks the rows of each key/value head that go, and hands their pages
back (`evict`), and moves the rows that stay into the holes (`move`).  A request's positions then run on past the rows
that it holds, so they are counted apart from the cache, and its new rows are rotated at any position, with the angles
scaled for contexts longer than the trained one: as a table of the step's rows for the fused norm + rotation + cache
write (`angles`), or applied to the rows themselves, in either layout of the pairs (`rope`).  Head layouts: the engine's
attention layers (8 query and 2 key/value heads of 256, 64 rotated dims, output gates, f16) and generic ones.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes what the program has in hand
before the call, `run()` is one call (the plain form in 32 bits, or the framework's operators where `own` is set),
`work()` what the call cannot do without, `exact()` the results in 64 bits.
"""
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False


def _pkg():
    """The package of this repository (its folder's name is not a Python identifier)."""
    if "sdamd" not in sys.modules:
        here = os.path.join(os.getcwd(), "strands-decider-rs_amd")
        spec = importlib.util.spec_from_file_location("sdamd", os.path.join(here, "__init__.py"),
                                                      submodule_search_locations=[here])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["sdamd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["sdamd"]


TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
THETA = 1e7
TRAINED = 4096  # tokens of the context that the angles were trained on

# ---- cases ----------------------------------------------------------------------------------------
# Requests: b of them, with old_lo .. old_hi tokens in their pages (spread over the logarithm); the first
# `chunks` have `new` new tokens, the last `idle` none, the others one.  ps: rows per page.  far: the largest
# number of positions that a request has left behind.


def listed():
    return [
        # The rows of one token each of 64 requests, neighbouring dims as pairs, angles scaled in parts.
        dict(name="rope_step_t64", op="rope", t=64, hq=32, hk=8, hd=128, rd=128, layout="pairs", scaling="parts",
             factor=8.0, far=100000, gated=False, inverse=False, type="bf16"),
        # A prompt's rows through the engine's attention layer: a quarter of each head, pairs half the rotated dims apart.
        dict(name="rope_prompt_t8192", op="rope", t=8192, hq=8, hk=2, hd=256, rd=64, layout="half", scaling="linear",
             factor=4.0, far=20000, gated=True, inverse=False, type="f16"),
        # The angles of one token each of 64 requests that have run on for long.
        dict(name="angles_step_b64", op="angles", b=64, old_lo=100, old_hi=4096, chunks=0, new=1, idle=0, rd=64,
             scaling="parts", factor=16.0, far=2000000),
        # The angles of four long chunks.
        dict(name="angles_chunks_4x4099", op="angles", b=4, old_lo=3, old_hi=9000, chunks=4, new=4099, idle=0, rd=128,
             scaling="base", factor=4.0, far=50000),
        # One token of one short request: launches and latency.
        dict(name="weights_step_b1", op="weights", b=1, old_lo=700, old_hi=700, chunks=0, new=1, idle=0, ps=32, hq=8,
             hk=2, hd=256, window=0, obs=0, decay=1.0, type="f16"),
        # One token each of 64 requests of up to 8191 tokens: the keys' bandwidth.
        dict(name="weights_step_b64", op="weights", b=64, old_lo=1000, old_hi=8191, chunks=0, new=1, idle=0, ps=64,
             hq=32, hk=8, hd=128, window=0, obs=0, decay=1.0, type="bf16"),
        # Two very long caches, scored by the last 32 rows of a question of 40.
        dict(name="weights_observe_b2", op="weights", b=2, old_lo=60001, old_hi=131000, chunks=2, new=40, idle=0, ps=128,
             hq=8, hk=2, hd=256, window=0, obs=32, decay=0.0, type="f16"),
        # A first prompt as long as the engine's context, every row of it counted: the largest matrix work.
        dict(name="weights_prompt_4096", op="weights", b=1, old_lo=0, old_hi=0, chunks=1, new=4096, idle=0, ps=64, hq=8,
             hk=2, hd=256, window=0, obs=0, decay=0.0, type="f16"),
        # 64 requests a few rows over what they may hold: the smallest eviction, every few steps.
        dict(name="evict_step_b64", op="evict", b=64, old_lo=4097, old_hi=4128, hk=8, ps=64, budget=4096, sink=4,
             recent=128, far=100000),
        # Two very long caches cut to a third.
        dict(name="evict_long_b2", op="evict", b=2, old_lo=90001, old_hi=131000, hk=2, ps=128, budget=32768, sink=16,
             recent=1024, far=0),
        # The rows that the smallest eviction moves.
        dict(name="move_step_b64", op="move", b=64, old_lo=4097, old_hi=4128, hk=8, hd=128, ps=64, budget=4096,
             type="bf16"),
        # The rows that the largest moves.
        dict(name="move_long_b2", op="move", b=2, old_lo=90001, old_hi=131000, hk=2, hd=256, ps=128, budget=32768,
             type="f16"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(8, 2, 256), (8, 2, 256), (32, 8, 128), (16, 2, 128), (28, 4, 128), (24, 8, 64), (8, 8, 128), (12, 1, 64),
         (4, 4, 256)]


def draw(rng):
    op = rng.choice(["rope", "angles", "weights", "weights", "weights", "evict", "move"])
    ps = rng.choice([32, 32, 64, 128, 256])
    hq, hk, hd = rng.choice(HEADS)
    kind = rng.choice(["f16", "bf16"])
    scale = dict(scaling=rng.choice(["plain", "linear", "base", "parts"]), factor=rng.choice([1.0, 2.0, 8.0, 2.5]))
    if op == "rope":
        return dict(op=op, t=_logint(rng, 1, 6000), hq=hq, hk=hk, hd=hd, rd=rng.choice([hd, hd // 2, hd // 4, 24]),
                    layout=rng.choice(["half", "pairs"]), far=_logint(rng, 10, 3000000), gated=rng.random() < 0.3,
                    inverse=rng.random() < 0.3, type=rng.choice(["f16", "bf16", "f32"]), **scale)
    if op == "angles":
        b = _logint(rng, 1, 300)
        chunks = rng.randint(0, min(b, 4))
        return dict(op=op, b=b, old_lo=rng.randint(1, 60), old_hi=_logint(rng, 100, 20000), chunks=chunks,
                    new=_logint(rng, 2, 3500), idle=rng.randint(0, (b - chunks) // 4), rd=rng.choice([24, 64, 128, 256]),
                    far=_logint(rng, 10, 3000000), **scale)
    if op == "weights":
        shape = rng.choice(["step", "step", "observe", "mixed", "chunk"])
        window = rng.choice([0, 0, 0, _logint(rng, 64, 4096)])
        decay = rng.choice([0.0, 1.0, 0.9])
        chunks, new, obs = 0, 1, 0
        if shape == "step":
            b = _logint(rng, 1, 48)
            hi = _logint(rng, 200, 8000 if b > 4 else 60000)
        elif shape == "observe":
            b = chunks = rng.randint(1, 6)
            new, obs, hi = rng.randint(2, 300), rng.choice([1, 8, 16, 32, 48]), _logint(rng, 300, 40000)
        elif shape == "mixed":
            b, chunks = rng.randint(8, 32), rng.randint(1, 2)
            new, obs, hi = _logint(rng, 30, 1500), rng.choice([4, 16, 32]), _logint(rng, 200, 6000)
        else:
            b = chunks = rng.randint(1, 2)
            new, hi = _logint(rng, 30, 1500), _logint(rng, 100, 3000)
        lo = rng.randint(0, 1) if shape == "chunk" and rng.random() < 0.5 else max(1, hi // rng.randint(2, 20))
        return dict(op=op, b=b, old_lo=lo, old_hi=hi if lo else 0, chunks=chunks, new=new,
                    idle=rng.randint(0, (b - chunks) // 6), ps=ps, hq=hq, hk=hk, hd=hd, window=window, obs=obs,
                    decay=decay, type=kind)
    b = _logint(rng, 1, 64)
    hi = _logint(rng, 200, 2500 if b > 16 else 8000 if b > 4 else 20000 if b > 2 else 60000)
    lo = max(1, hi // rng.randint(1, 4))
    budget = max(1, int(hi * rng.choice([0.99, 0.9, 0.5, 0.25, 0.06])))
    if op == "evict":
        sink = rng.randint(0, min(16, budget // 4))
        return dict(op=op, b=b, old_lo=lo, old_hi=hi, hk=hk, ps=ps, budget=budget, sink=sink,
                    recent=rng.randint(0, budget // 3), far=rng.choice([0, 50, 1000000]))
    return dict(op=op, b=b, old_lo=lo, old_hi=hi, hk=hk, hd=hd, ps=ps, budget=budget, type=kind)


def _old(case):
    rng = random.Random(case["b"] * 7919 + case["old_hi"] * 31 + case.get("new", 0))
    lo, hi = case["old_lo"], case["old_hi"]
    return [0 if hi == 0 else _logint(rng, max(lo, 1), max(hi, 1)) for _ in range(case["b"])]


def _lens(case):
    """The requests' old and new token counts, from the case alone."""
    b = case["b"]
    new = [case["new"] if i < case["chunks"] else 0 if i >= b - case["idle"] else 1 for i in range(b)]
    if not sum(new):
        new[0] = 1
    return _old(case), new


def _pages(n, ps):
    return -(-n // ps)


# ---- inputs ---------------------------------------------------------------------------------------

def _gen(seed, salt):
    return torch.Generator("cuda").manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(seed, kv, ps, spare=3):
    """Pages in random order: the block table of the first `kv` tokens of every request, the others, and their number."""
    need = [_pages(n, ps) for n in kv]
    total = sum(need)
    pages = np.random.default_rng([int(seed), 91]).permutation(total + spare)
    table = np.full((len(kv), max(max(need), 1)), -1, np.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pages[at:at + n]
        at += n
    return table, pages[total:], total + spare


def _params(case):
    """The rotation's parameters; the magnitude that goes with scaling in parts, 1 + 0.1 ln(factor)."""
    parts = case["scaling"] == "parts"
    return dict(rotary_dim=case["rd"], scaling=case["scaling"], theta=THETA, factor=case["factor"],
                length=TRAINED, low=1.0, high=32.0, magnitude=1 + 0.1 * math.log(case["factor"]) if parts else 1.0)


def _rope_inputs(case, seed):
    t, hq, hk, hd = case["t"], case["hq"], case["hk"], case["hd"]
    g = _gen(seed, 3)
    big = torch.randn(t, (hq * (2 if case["gated"] else 1) + 2 * hk) * hd, generator=g, device="cuda")
    return big.to(TYPES[case["type"]]), np.random.default_rng([int(seed), 5]).integers(0, case["far"] + 1, t)


def _angles_inputs(case, seed):
    old, new = _lens(case)
    dropped = np.random.default_rng([int(seed), 7]).integers(0, case["far"] + 1, case["b"])
    return new, np.concatenate([np.arange(o, o + n) for o, n in zip(old, new)]), dropped


def _weights_inputs(case, seed):
    old, new = _lens(case)
    t, ps, dt = sum(new), case["ps"], TYPES[case["type"]]
    hq, hk, hd = case["hq"], case["hk"], case["hd"]
    g = _gen(seed, 9)
    kv = [o + n for o, n in zip(old, new)]
    table, _, n_pages = _tables(seed, kv, ps)
    # queries and keys as their norms leave them, the query's weights above one: some keys matter more than others
    q = (1.5 * torch.randn(t, hq, hd, generator=g, device="cuda")).to(dt)
    kp = torch.randn(n_pages * hk * ps * hd, generator=g, device="cuda").to(dt)
    scores = 4 * torch.rand(n_pages, hk, ps, generator=g, device="cuda").pow(3)
    ahead = np.random.default_rng([int(seed), 11]).integers(0, 5000, case["b"])
    pos = np.concatenate([a + np.arange(o, o + n) for a, o, n in zip(ahead, old, new)])
    return old, new, kv, table, n_pages, q, kp, scores, pos


def _evict_inputs(case, seed):
    n, ps, hk = _old(case), case["ps"], case["hk"]
    table, spare, n_pages = _tables(seed, n, ps, 9)
    g = _gen(seed, 13)
    # weight as attention leaves it: few keys have most of it, some exactly none
    scores = torch.randn(n_pages, hk, ps, generator=g, device="cuda").mul_(2).exp_()
    scores *= torch.rand(scores.shape, generator=g, device="cuda") > 0.02
    # positions: the rows in order, `far` of them long gone, and the last few in holes that earlier evictions left
    kpos = torch.zeros(n_pages, hk, ps, dtype=torch.int32, device="cuda")
    rng = np.random.default_rng([int(seed), 15])
    for b, m in enumerate(n):
        p = np.arange(m)
        if case["far"]:
            p = np.sort(rng.integers(0, case["far"] + 1, m)) + np.arange(m)
            k = min(m // 4, 40)
            i, j = rng.choice(m - k, k, replace=False), np.arange(m - k, m)
            p[i], p[j] = p[j], p[i].copy()
        page = torch.from_numpy(table[b, np.arange(m) // ps]).cuda()
        kpos[page, :, torch.arange(m, device="cuda") % ps] = torch.from_numpy(p.astype(np.int32)).cuda()[:, None]
    dropped = rng.integers(0, case["far"] + 1, case["b"])
    free = np.concatenate([rng.permutation(spare)[:5], np.full(n_pages - 5, -1)])  # (4 pages are another program's)
    return n, table, n_pages, scores, kpos, dropped, free


def _move_counts(case):
    """Moves of every request's heads: as many as rows picked at random would make, from the case alone."""
    rng = random.Random(case["b"] * 31 + case["budget"])
    out = []
    for n in _old(case):
        m = min(n, case["budget"])
        most = min(m, n - m)
        out.append([min(most, max(0, int(round(m * (n - m) / n * rng.uniform(0.9, 1.1))))) for _ in range(case["hk"])])
    return out


def _move_inputs(case, seed):
    n, ps, hk, hd, dt = _old(case), case["ps"], case["hk"], case["hd"], TYPES[case["type"]]
    table, _, n_pages = _tables(seed, n, ps)
    g = _gen(seed, 17)
    kp = torch.randn(n_pages * hk * ps * hd, generator=g, device="cuda").to(dt)
    vp = torch.randn(n_pages * hk * ps * hd, generator=g, device="cuda").to(dt)
    scores = torch.rand(n_pages, hk, ps, generator=g, device="cuda")
    kpos = torch.randint(0, 1 << 30, (n_pages, hk, ps), generator=g, device="cuda", dtype=torch.int32)
    counts = _move_counts(case)
    width = max(max(n) // 2, 1)
    moves = np.full((case["b"], hk, width, 2), -1, np.int32)
    rng = np.random.default_rng([int(seed), 19])
    for b, m in enumerate(n):
        keep = min(m, case["budget"])
        for h, c in enumerate(counts[b]):
            moves[b, h, :c, 0] = np.sort(rng.choice(keep, c, replace=False))
            moves[b, h, :c, 1] = keep + np.sort(rng.choice(m - keep, c, replace=False))
    return n, table, n_pages, kp, vp, scores, kpos, moves, counts


def prepare(case, seed):
    st = dict(case)
    if case["op"] == "rope":
        big, pos = _rope_inputs(case, seed)
        t, hd = case["t"], case["hd"]
        st.update(big=big, pos=_ints(pos.tolist()), params=_params(case), q=torch.zeros(t, case["hq"], hd, device="cuda", dtype=big.dtype),
                  k=torch.zeros(t, case["hk"], hd, device="cuda", dtype=big.dtype))
    elif case["op"] == "angles":
        new, pos, dropped = _angles_inputs(case, seed)
        t = sum(new)
        st.update(cu=_ints([0] + np.cumsum(new).tolist()), at=_ints(pos.tolist()), dropped=_ints(dropped.tolist()), t=t,
                  params=_params(case), pos=_ints([0] * t), table=torch.zeros(t, case["rd"] // 2, 2, device="cuda"))
    elif case["op"] == "weights":
        old, new, kv, table, n_pages, q, kp, scores, pos = _weights_inputs(case, seed)
        st.update(cu=_ints([0] + np.cumsum(new).tolist()), kv=_ints(kv), table=_ints(table.tolist()), n_pages=n_pages,
                  q=q, kp=kp, scores=scores, out=torch.zeros_like(scores), pos=_ints(pos.tolist()), t=sum(new),
                  kpos=torch.zeros(scores.shape, dtype=torch.int32, device="cuda"), max_new=max(new), max_kv=max(kv))
    elif case["op"] == "evict":
        n, table, n_pages, scores, kpos, dropped, free = _evict_inputs(case, seed)
        b, hk = case["b"], case["hk"]
        st.update(kv=_ints(n), table=_ints(table.tolist()), n_pages=n_pages, scores=scores, kpos=kpos, max_kv=max(n),
                  budgets=_ints([case["budget"]] * b), lens=_ints([0] * b), counts=torch.zeros(b, hk, dtype=torch.int32, device="cuda"),
                  moves=torch.full((b, hk, max(max(n) // 2, 1), 2), -1, dtype=torch.int32, device="cuda"),
                  dropped=_ints(dropped.tolist()), gone=_ints([0] * b), free=_ints(free.tolist()), n_free=_ints([5]), left=_ints([0]))
    else:
        n, table, n_pages, kp, vp, scores, kpos, moves, counts = _move_inputs(case, seed)
        st.update(kp=kp, vp=vp, scores=scores, kpos=kpos, moves=torch.from_numpy(moves).cuda(), counts=_ints(counts),
                  table=_ints(table.tolist()), n_pages=n_pages, max_kv=max(n))
    return st


# ---- one call -------------------------------------------------------------------------------------

def run(st):
    if own:
        return {"rope": _own_rope, "angles": _own_angles, "weights": _own_weights, "evict": _own_evict, "move": _own_move}[st["op"]](st)
    return {"rope": _plain_rope, "angles": _plain_angles, "weights": _plain_weights, "evict": _plain_evict, "move": _plain_move}[st["op"]](st)


def _own_freqs(st):
    """The pairs' frequencies on the device, made once for a state as a program makes them once for a model."""
    if "freqs" not in st:
        sd, p = _pkg(), st["params"]
        kinds = {"plain": sd.ROPE_PLAIN, "linear": sd.ROPE_LINEAR, "base": sd.ROPE_BASE, "parts": sd.ROPE_PARTS}
        f = sd.rope_freqs(p["rotary_dim"], p["theta"], kinds[p["scaling"]], p["factor"], p["length"], p["low"], p["high"])
        st["freqs"] = torch.from_numpy(f).cuda()
    return st["freqs"].data_ptr()


def _own_rope(st):
    sd = _pkg()
    big, hq, hk, hd = st["big"], st["hq"], st["hk"], st["hd"]
    step = hd * (2 if st["gated"] else 1)
    sd.op_rope(_own_freqs(st), st["rd"], sd.ROPE_HALF if st["layout"] == "half" else sd.ROPE_PAIRS, st["pos"].data_ptr(),
               st["t"], hd, big.data_ptr(), big.shape[1], step, hq, big.data_ptr() + hq * step * big.element_size(),
               big.shape[1], hd, hk, {"f16": sd.F16, "bf16": sd.BF16, "f32": sd.F32}[st["type"]],
               magnitude=st["params"]["magnitude"], inverse=st["inverse"], Qo=st["q"].data_ptr(), Ko=st["k"].data_ptr())
    return {"q": st["q"], "k": st["k"]}


def _own_angles(st):
    sd = _pkg()
    sd.op_page_positions(st["cu"].data_ptr(), st["dropped"].data_ptr(), st["b"], st["t"], st["at"].data_ptr(),
                         st["pos"].data_ptr())
    sd.op_rope_table(_own_freqs(st), st["rd"] // 2, st["pos"].data_ptr(), st["t"], st["table"].data_ptr(),
                     magnitude=st["params"]["magnitude"])
    return {"pos": st["pos"], "table": st["table"]}


def _own_weights(st):
    sd = _pkg()
    if "ws" not in st:
        st["ws"] = torch.empty(sd.paged_weights_ws(st["b"], st["t"], st["max_new"], st["max_kv"], st["hq"], st["hk"],
                                                   st["hd"], observers=st["obs"]), dtype=torch.uint8, device="cuda")
    sd.op_paged_weights(st["q"].data_ptr(), st["kp"].data_ptr(), st["table"].data_ptr(), st["table"].shape[1],
                        st["cu"].data_ptr(), st["kv"].data_ptr(), st["b"], st["t"], st["max_new"], st["max_kv"], st["hq"],
                        st["hk"], st["hd"], st["ps"], st["n_pages"], st["scores"].data_ptr(), st["out"].data_ptr(),
                        st["ws"].data_ptr(), st["ws"].numel(), sd.F16 if st["type"] == "f16" else sd.BF16,
                        decay=st["decay"], observers=st["obs"], window=st["window"], pos=st["pos"].data_ptr(),
                        kpos=st["kpos"].data_ptr())
    return {"scores": st["out"], "kpos": st["kpos"]}


def _own_evict(st):
    sd = _pkg()
    if "ews" not in st:
        st["ews"] = torch.empty(max(sd.page_evict_ws(st["b"], st["max_kv"], st["hk"]), 16), dtype=torch.uint8, device="cuda")
    sd.op_page_evict(st["scores"].data_ptr(), st["kpos"].data_ptr(), st["table"].data_ptr(), st["table"].shape[1],
                     st["kv"].data_ptr(), st["budgets"].data_ptr(), st["b"], st["max_kv"], st["hk"], st["ps"],
                     st["n_pages"], st["sink"], st["recent"], st["lens"].data_ptr(), st["moves"].data_ptr(),
                     st["counts"].data_ptr(), st["ews"].data_ptr(), st["ews"].numel())
    sd.op_page_release(st["kv"].data_ptr(), st["lens"].data_ptr(), st["dropped"].data_ptr(), st["table"].data_ptr(),
                       st["table"].shape[1], st["b"], st["ps"], st["n_pages"], st["free"].data_ptr(),
                       st["n_free"].data_ptr(), st["gone"].data_ptr(), st["left"].data_ptr())
    return {"lens": st["lens"], "moves": st["moves"], "counts": st["counts"], "dropped": st["gone"], "free": st["free"],
            "n_free": st["left"]}


def _own_move(st):
    sd = _pkg()
    sd.op_paged_move(st["moves"].data_ptr(), st["counts"].data_ptr(), st["table"].data_ptr(), st["table"].shape[1],
                     st["b"], st["max_kv"], st["hk"], st["hd"], st["ps"], st["n_pages"], st["kp"].data_ptr(),
                     st["vp"].data_ptr(), st["scores"].data_ptr(), st["kpos"].data_ptr(),
                     sd.F16 if st["type"] == "f16" else sd.BF16)
    return {k: st[k] for k in ("kp", "vp", "scores", "kpos")}


def _plain_turns(p, pos):
    """[rows][pairs] cosines and sines, the angles in 64 bits: positions of millions lose theirs in 32."""
    rd, s = p["rotary_dim"], p["factor"]
    j = torch.arange(0, rd, 2, dtype=torch.float64, device=pos.device) / rd
    theta = p["theta"] * s ** (rd / (rd - 2)) if p["scaling"] == "base" else p["theta"]
    f = theta ** -j
    if p["scaling"] == "linear":
        f = f / s
    if p["scaling"] == "parts":  # by the turns that a pair makes over the trained length
        keep = ((p["length"] * f / (2 * math.pi) - p["low"]) / (p["high"] - p["low"])).clamp(0, 1)
        f = f * (keep + (1 - keep) / s)
    a = pos.double()[:, None] * f
    return a.cos() * p["magnitude"], a.sin() * p["magnitude"]


def _plain_rope(st):
    t, hq, hk, hd, rd = st["t"], st["hq"], st["hk"], st["hd"], st["rd"]
    per = 2 if st["gated"] else 1
    x = st["big"].view(t, hq * per + 2 * hk, hd)
    x = torch.cat([x[:, :hq * per:per], x[:, hq * per:hq * per + hk]], 1).float()
    c, s = (y.float()[:, None] for y in _plain_turns(st["params"], st["pos"]))
    if st["inverse"]:
        s = -s
    if st["layout"] == "half":
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        y = torch.cat([a * c - b * s, b * c + a * s, x[..., rd:]], -1)
    else:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        y = torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., rd:]], -1)
    y = y.to(st["big"].dtype)
    return {"q": y[:, :hq].contiguous(), "k": y[:, hq:].contiguous()}


def _plain_angles(st):
    t = torch.arange(st["t"], device=st["at"].device)
    pos = st["at"] + st["dropped"][(t[:, None] >= st["cu"][1:]).sum(1)]
    return {"pos": pos, "table": torch.stack(_plain_turns(st["params"], pos), -1).float()}


def _rows_at(st, n):
    """[requests][heads][n]: where each cached row's score lies."""
    hk, ps = st["hk"], st["ps"]
    j = torch.arange(n, device=st["table"].device)
    page = st["table"].long()[:, j // ps].clamp(min=0)
    return (page[:, None] * hk + torch.arange(hk, device=page.device)[:, None]) * ps + j % ps


def _plain_weights(st):
    b, hq, hk, hd, ps = st["b"], st["hq"], st["hk"], st["hd"], st["ps"]
    n, g, dev = st["max_kv"], hq // hk, st["q"].device
    r = min(st["obs"] or st["max_new"], st["max_new"])  # rows that are counted, at most
    cu, kv = st["cu"].long(), st["kv"].long()
    new = cu[1:] - cu[:-1]
    i = (new - r).clamp(min=0)[:, None] + torch.arange(r, device=dev)
    q = st["q"][(cu[:-1, None] + i).clamp(max=st["t"] - 1)].float()
    q = q.view(b, r, hk, g, hd).transpose(1, 2).reshape(b, hk, r * g, hd)
    k = st["kp"].view(-1, hk, ps // 32, hd // 32, 32, 32)[st["table"].long()[:, :_pages(n, ps)].clamp(min=0)]
    k = k.permute(0, 2, 1, 3, 5, 4, 6).reshape(b, hk, -1, hd)[:, :, :n].float()
    s = (q @ k.transpose(2, 3).contiguous()).view(b, hk, r, g, n) * (1 / math.sqrt(hd))
    j = torch.arange(n, device=dev)
    p = ((kv - new)[:, None] + i)[..., None]
    seen = (j <= p) & (i < new[:, None])[..., None]
    if st["window"]:
        seen &= j > p - st["window"]
    seen = seen[:, None, :, None]
    s = s.masked_fill(~seen, -math.inf)
    e = torch.where(seen, (s - s.max(-1, keepdim=True).values).exp(), 0)
    w = (e / e.sum(-1, keepdim=True).clamp(min=1e-30)).sum((2, 3))  # [requests][heads][n]
    at = _rows_at(st, n)
    first = (kv - new)[:, None, None]
    total = torch.where(j < first, st["decay"] * st["scores"].view(-1)[at], 0) + w
    live = ((j < kv[:, None, None]) & (new > 0)[:, None, None]).expand_as(at)
    st["out"].view(-1)[at[live]] = total[live]
    fresh = live & (j >= first)
    row = (cu[:-1, None, None] + j - first).clamp(0, st["t"] - 1).expand_as(at)
    st["kpos"].view(-1)[at[fresh]] = st["pos"][row[fresh]]
    return {"scores": st["out"], "kpos": st["kpos"]}


def _plain_evict(st):
    b, hk, ps, n = st["b"], st["hk"], st["ps"], st["max_kv"]
    at, kv = _rows_at(st, n), st["kv"].long()
    j = torch.arange(n, device=at.device)
    live = j < kv[:, None, None]
    m = torch.minimum(kv, st["budgets"].long())
    p = torch.where(live, st["kpos"].view(-1)[at], -1)
    newest = p.max(-1, keepdim=True).values
    key = torch.where((p < st["sink"]) | (p > newest - st["recent"]), math.inf, st["scores"].view(-1)[at])
    order = torch.where(live, key, -math.inf).sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros(at.shape, dtype=torch.bool, device=at.device)
    kept.scatter_(2, order, (j < m[:, None, None]).expand_as(order))
    inside = j < m[:, None, None]
    for_hole, for_row = inside & ~kept, ~inside & kept & live
    counts = for_row.sum(-1)
    moves = st["moves"].view(b * hk, -1, 2)
    for_hole, for_row = (x.view(b * hk, n) for x in (for_hole, for_row))
    for e, x in ((0, for_hole), (1, for_row)):
        head, row = x.nonzero(as_tuple=True)
        moves[head, (x.cumsum(-1) - 1)[head, row], e] = row.int()
    # pages behind the rows that stay, request by request, onto the free stack
    blk = torch.arange(st["table"].shape[1], device=at.device)
    gone = (blk >= ((m + ps - 1) // ps)[:, None]) & (blk < ((kv + ps - 1) // ps)[:, None])
    pages = st["table"][gone]
    at = st["n_free"].long() + torch.arange(pages.numel(), device=pages.device)
    st["free"][at] = pages
    return {"lens": m.int(), "moves": st["moves"], "counts": counts.int(), "dropped": st["dropped"] + (kv - m).int(),
            "free": st["free"], "n_free": st["n_free"] + pages.numel()}


def _plain_move(st):
    hk, hd, ps = st["hk"], st["hd"], st["ps"]
    b, h, i = (torch.arange(st["moves"].shape[2], device=st["moves"].device) < st["counts"][..., None]).nonzero(as_tuple=True)
    to, fr = st["moves"][b, h, i].long().unbind(-1)
    kp, vp = st["kp"].view(-1, hk, ps // 32, hd // 32, 32, 32), st["vp"].view(-1, hk, ps // 32, hd, 32)
    table = st["table"].long()
    p, x = table[b, to // ps], table[b, fr // ps]
    kp[p, h, to % ps // 32, :, to % 32] = kp[x, h, fr % ps // 32, :, fr % 32]
    vp[p, h, to % ps // 32, :, to % 32] = vp[x, h, fr % ps // 32, :, fr % 32]
    st["scores"][p, h, to % ps] = st["scores"][x, h, fr % ps]
    st["kpos"][p, h, to % ps] = st["kpos"][x, h, fr % ps]
    return {k: st[k] for k in ("kp", "vp", "scores", "kpos")}


# ---- what a call cannot do without ----------------------------------------------------------------

def work(case):
    if case["op"] == "rope":
        heads, size = case["hq"] + case["hk"], TYPES[case["type"]].itemsize
        return {"bytes": case["t"] * (2 * heads * case["hd"] * size + 4), "flops": 3 * case["t"] * heads * case["rd"]}
    if case["op"] == "angles":
        t = sum(_lens(case)[1])
        return {"bytes": 4 * (2 * case["b"] + 1 + 2 * t + t * case["rd"]), "flops": t * case["rd"]}
    if case["op"] == "weights":
        old, new = _lens(case)
        hq, hk, hd, w = case["hq"], case["hk"], case["hd"], case["window"]
        size = flops = 0
        for o, n in zip(old, new):
            if not n:
                continue
            r = min(n, case["obs"] or n)
            first, kv = o + n - r, o + n  # the position of the first row that is counted
            pairs = sum(min(w, p + 1) if w else p + 1 for p in range(first, kv))
            keys = kv - max(0, first - w + 1) if w else kv
            size += 2 * hk * hd * keys + 2 * r * hq * hd + 4 * hk * (kv + n + (o if case["decay"] else 0)) + 4 * n
            flops += 2 * hq * hd * pairs
        return {"bytes": size, "flops": flops}
    if case["op"] == "evict":
        size = 0
        for n in _old(case):
            m = min(n, case["budget"])
            size += case["hk"] * ((8 * n if m < n else 0) + 8 * m * (n - m) // n + 4) + 16 + 8 * (_pages(n, case["ps"]) - _pages(m, case["ps"]))
        return {"bytes": size, "flops": 0}
    rows = sum(map(sum, _move_counts(case)))
    return {"bytes": rows * (2 * (4 * case["hd"] + 8) + 8) + 4 * case["b"] * case["hk"], "flops": 0}


# ---- 64-bit results -------------------------------------------------------------------------------

def _exact_freqs(p):
    """Radians per position of every pair, one by one."""
    out, rd, s = [], p["rotary_dim"], p["factor"]
    for i in range(rd // 2):
        base = p["theta"] * (s ** (rd / (rd - 2)) if p["scaling"] == "base" else 1.0)
        f = math.exp(-2 * i / rd * math.log(base))
        if p["scaling"] == "linear":
            f /= s
        elif p["scaling"] == "parts":
            turns = p["length"] * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - p["low"]) / (p["high"] - p["low"])))
            f = keep * f + (1 - keep) * f / s
        out.append(f)
    return np.array(out)


def _exact_rope(case, seed):
    big, pos = _rope_inputs(case, seed)
    p, rd, hq, hk = _params(case), case["rd"], case["hq"], case["hk"]
    angle = torch.from_numpy(np.outer(pos, _exact_freqs(p))).cuda() * (-1 if case["inverse"] else 1)
    turn = torch.polar(torch.full_like(angle, p["magnitude"]), angle)[:, None]
    x = big.double().unflatten(1, (-1, case["hd"]))
    q = x[:, 0:2 * hq:2] if case["gated"] else x[:, :hq]
    out = []
    for z in (q, x[:, -2 * hk:-hk]):
        z = z.clone()
        i = torch.arange(rd // 2, device="cuda")
        first, second = (i, i + rd // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        y = torch.complex(z[..., first], z[..., second]) * turn
        z[..., first], z[..., second] = y.real, y.imag
        out.append(z)
    return {"q": out[0], "k": out[1]}


def _exact_angles(case, seed):
    new, at, dropped = _angles_inputs(case, seed)
    p = _params(case)
    pos = at + np.repeat(dropped, new)
    a = torch.from_numpy(np.outer(pos, _exact_freqs(p))).cuda()
    return {"pos": _ints(pos.tolist()), "table": torch.view_as_real(torch.polar(torch.full_like(a, p["magnitude"]), a))}


def _exact_weights(case, seed):
    old, new, kvs, table, n_pages, q, kp, scores, pos = _weights_inputs(case, seed)
    hq, hk, hd, ps, w = case["hq"], case["hk"], case["hd"], case["ps"], case["window"]
    g, out = hq // hk, torch.zeros(scores.shape, dtype=torch.float64, device="cuda").view(-1)
    kpos, scores = torch.zeros(scores.shape, dtype=torch.int32, device="cuda"), scores.double().view(-1)
    d, at = torch.arange(hd, device="cuda"), 0
    for b, (o, n, kv) in enumerate(zip(old, new, kvs)):
        if n == 0:
            continue
        r = min(n, case["obs"] or n)
        j = np.arange(kv)
        page = table[b, j // ps]
        kpos[torch.from_numpy(page[o:]).cuda(), :, torch.from_numpy(j[o:] % ps).cuda()] = _ints(pos[at:at + n].tolist())[:, None]
        for h in range(hk):
            block = torch.from_numpy((page * hk + h) * ps + j % ps // 32 * 32).cuda()[:, None] * hd
            k = kp[block + d // 32 * 1024 + torch.from_numpy(j % 32).cuda()[:, None] * 32 + d % 32].double()
            total = torch.zeros(kv, dtype=torch.float64, device="cuda")
            for t0 in range(n - r, n, 512):
                t1 = min(n, t0 + 512)
                z = q[at + t0:at + t1, h * g:(h + 1) * g].double().reshape(-1, hd) @ k.T / math.sqrt(hd)
                back = torch.arange(o + t0, o + t1, device="cuda")[:, None] - torch.arange(kv, device="cuda")
                hide = (back < 0) | (back >= w) if w else back < 0
                total += torch.softmax(z.view(t1 - t0, g, kv).masked_fill(hide[:, None], -math.inf), -1).sum((0, 1))
            row = torch.from_numpy((page * hk + h) * ps + j % ps).cuda()
            total[:o] += case["decay"] * scores[row[:o]]
            out[row] = total
        at += n
    return {"scores": out.view(kpos.shape), "kpos": kpos}


def _exact_evict(case, seed):
    """The definition, head by head."""
    n, table, n_pages, scores, kpos, dropped, free = _evict_inputs(case, seed)
    ps, hk = case["ps"], case["hk"]
    scores, kpos, free, left = scores.cpu().numpy(), kpos.cpu().numpy(), free.copy(), 5
    lens = [min(m, case["budget"]) for m in n]
    moves = np.full((case["b"], hk, max(max(n) // 2, 1), 2), -1, np.int32)
    counts = np.zeros((case["b"], hk), np.int32)
    for b, (m, keep) in enumerate(zip(n, lens)):
        j = np.arange(m)
        page = table[b, j // ps]
        for h in range(hk):
            s, p = scores[page, h, j % ps].astype(np.float64), kpos[page, h, j % ps].astype(np.int64)
            s[(p < case["sink"]) | (p > p.max() - case["recent"])] = np.inf
            stay = np.sort(np.lexsort((j, -s))[:keep])
            rows = stay[stay >= keep]
            holes = np.setdiff1d(np.arange(keep), stay)
            counts[b, h] = len(rows)
            moves[b, h, :len(rows), 0], moves[b, h, :len(rows), 1] = holes, rows
        for i in range(_pages(keep, ps), _pages(m, ps)):
            free[left] = table[b, i]
            left += 1
    return {"lens": _ints(lens), "moves": _ints(moves.tolist()), "counts": _ints(counts.tolist()),
            "dropped": _ints([d + m - k for d, m, k in zip(dropped.tolist(), n, lens)]), "free": _ints(free.tolist()),
            "n_free": _ints([left])}


def _exact_move(case, seed):
    """Row by row of a head's (key, value, score, position), addressed element by element."""
    n, table, n_pages, kp, vp, scores, kpos, moves, counts = _move_inputs(case, seed)
    hk, hd, ps = case["hk"], case["hd"], case["ps"]
    d = torch.arange(hd, device="cuda")
    kp, vp, score, pos = kp.double(), vp.double(), scores.double().view(-1), kpos.view(-1)
    for b in range(case["b"]):
        for h in range(hk):
            c = counts[b][h]
            to, fr = ((table[b, x // ps] * hk + h) * ps + x % ps for x in (moves[b, h, :c, 0], moves[b, h, :c, 1]))
            to, fr = (torch.from_numpy(x).cuda() for x in (to, fr))
            score[to], pos[to] = score[fr], pos[fr]
            k = [(x // 32 * 32 * hd)[:, None] + d // 32 * 1024 + (x % 32)[:, None] * 32 + d % 32 for x in (to, fr)]
            v = [(x // 32 * 32 * hd)[:, None] + d * 32 + (x % 32)[:, None] for x in (to, fr)]
            kp[k[0]], vp[v[0]] = kp[k[1]], vp[v[1]]
    return {"kp": kp, "vp": vp, "scores": score.view(scores.shape), "kpos": kpos}


def exact(case, seed):
    return {"rope": _exact_rope, "angles": _exact_angles, "weights": _exact_weights, "evict": _exact_evict,
            "move": _exact_move}[case["op"]](case, seed)
