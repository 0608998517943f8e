"""Serving many requests from a paged key/value cache, as cases that can be timed and compared.

A step of such a program gives the requests' new tokens their pages (`plan`), writes their rotated keys and
their values into the pages (`prep`), and lets their queries attend every request's own pages (`attend`).
Head layouts: the engine's attention layers (8 query and 2 key/value heads of 256, 64 rotated dims, output
gates, f16) and generic ones of 128 and 64 dims, f16 and bf16.  A step holds single tokens, drafts of a few,
chunks of a prompt, and mixtures of them.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes what the program has in
hand before the call, `run()` is one call (the plain form in 32 bits, or the framework's operators where `own`
is set), `work()` what the call cannot do without, `exact()` the results in 64 bits.
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


TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
THETA = 1e7
EPS = 1e-6

# ---- cases ----------------------------------------------------------------------------------------
# Requests: b of them, with old_lo .. old_hi tokens in their pages (spread over the logarithm); the first
# `chunks` have `new` new tokens, the last `idle` none, the others one.  ps: rows per page.


def listed():
    return [
        # Pages for one token each of 8 requests: the smallest call of a step.
        dict(name="plan_step_b8", op="plan", b=8, old_lo=40, old_hi=3500, chunks=0, new=1, idle=0, ps=32, short=False),
        # 384 requests: 24 prompts being read in chunks of 500, single tokens, some idle.
        dict(name="plan_admit_b384", op="plan", b=384, old_lo=1, old_hi=30000, chunks=24, new=500, idle=9, ps=64,
             short=False),
        # One token each of 16 requests through the engine's attention layer.
        dict(name="prep_step_b16", op="prep", b=16, old_lo=30, old_hi=4000, chunks=0, new=1, idle=0, ps=32, hq=8,
             hk=2, hd=256, rd=64, axes=1, gated=True, type="f16"),
        # Prompts with images: three position axes, every dim rotated, ragged chunks.
        dict(name="prep_image_t4099", op="prep", b=4, old_lo=3, old_hi=900, chunks=3, new=1366, idle=0, ps=64, hq=32,
             hk=8, hd=128, rd=128, axes=3, gated=False, type="bf16"),
        # One token of one short request: launches and latency.
        dict(name="attend_step_b1", op="attend", b=1, old_lo=700, old_hi=700, chunks=0, new=1, idle=0, ps=32, hq=8,
             hk=2, hd=256, window=0, gated=True, type="f16"),
        # One token each of 64 requests of up to 8191 tokens: the cache's bandwidth.
        dict(name="attend_step_b64", op="attend", b=64, old_lo=1000, old_hi=8191, chunks=0, new=1, idle=0, ps=64,
             hq=32, hk=8, hd=128, window=0, gated=False, type="bf16"),
        # Two requests with very long caches: work split over a long axis.
        dict(name="attend_long_b2", op="attend", b=2, old_lo=90001, old_hi=131000, chunks=0, new=1, idle=0, ps=128,
             hq=8, hk=2, hd=256, window=0, gated=True, type="f16"),
        # Drafts of 6 tokens, 3 query heads of 64 dims per key/value head: 18 rows share a key.
        dict(name="attend_draft_b32", op="attend", b=32, old_lo=300, old_hi=4000, chunks=32, new=6, idle=0, ps=32,
             hq=24, hk=8, hd=64, window=0, gated=False, type="bf16"),
        # A 511-token question on a long state, the engine's heads.
        dict(name="attend_chunk_511", op="attend", b=1, old_lo=3489, old_hi=3489, chunks=1, new=511, idle=0, ps=32,
             hq=8, hk=2, hd=256, window=0, gated=True, type="f16"),
        # A first prompt of 8192 tokens, the engine's heads.
        dict(name="attend_prompt_8192", op="attend", b=1, old_lo=0, old_hi=0, chunks=1, new=8192, idle=0, ps=256,
             hq=8, hk=2, hd=256, window=0, gated=True, type="f16"),
        # Four prompts in chunks of 2048 over what they have read so far: the largest matrix work.
        dict(name="attend_chunks_4x2048", op="attend", b=4, old_lo=2048, old_hi=8192, chunks=4, new=2048, idle=0,
             ps=64, hq=32, hk=8, hd=128, window=0, gated=False, type="bf16"),
        # A ragged chunk among 40 single tokens, a sliding window of 1024, one request idle.
        dict(name="attend_mixed_window", op="attend", b=42, old_lo=100, old_hi=6000, chunks=1, new=1501, idle=1,
             ps=32, hq=16, hk=4, hd=128, window=1024, gated=False, type="bf16"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(8, 2, 256), (8, 2, 256), (32, 8, 128), (16, 2, 128), (28, 4, 128), (24, 8, 64), (8, 8, 128), (12, 1, 64),
         (4, 4, 256)]


def draw(rng):
    op = rng.choice(["plan", "prep", "attend", "attend", "attend"])
    ps = rng.choice([32, 32, 64, 128, 256])
    if op == "plan":
        b = _logint(rng, 1, 400)
        chunks = rng.randint(0, max(1, b // 8))
        return dict(op=op, b=b, old_lo=rng.randint(1, 60), old_hi=_logint(rng, 100, 30000), chunks=chunks,
                    new=_logint(rng, 2, 500), idle=rng.randint(0, (b - chunks) // 4), ps=ps, short=rng.random() < 0.25)
    hq, hk, hd = rng.choice(HEADS)
    kind = rng.choice(["f16", "bf16"])
    if op == "prep":
        b = _logint(rng, 1, 64)
        chunks = rng.randint(0, min(b, 3))
        rd = rng.choice([hd, hd // 2, 64, 24])
        return dict(op=op, b=b, old_lo=rng.randint(1, 60), old_hi=_logint(rng, 100, 4000), chunks=chunks,
                    new=_logint(rng, 2, 1300), idle=rng.randint(0, (b - chunks) // 4), ps=ps, hq=hq, hk=hk, hd=hd,
                    rd=rd, axes=rng.choice([1, 1, 3]), gated=rng.random() < 0.5, type=kind)
    window = rng.choice([0, 0, 0, _logint(rng, 64, 4096)])
    shape = rng.choice(["step", "step", "draft", "chunk", "mixed"])
    if shape == "step":
        b, chunks, new = _logint(rng, 1, 64), 0, 1
        hi = _logint(rng, 200, 8000 if b > 4 else 100000)
    elif shape == "draft":
        b = chunks = _logint(rng, 1, 48)
        new, hi = rng.randint(2, 12), _logint(rng, 200, 5000)
    elif shape == "chunk":
        b = chunks = rng.randint(1, 4)
        new, hi = _logint(rng, 30, 2000), _logint(rng, 100, 6000)
    else:
        b, chunks = rng.randint(8, 48), rng.randint(1, 2)
        new, hi = _logint(rng, 30, 1500), _logint(rng, 200, 6000)
    lo = rng.randint(0, 1) if shape == "chunk" and rng.random() < 0.5 else max(1, hi // rng.randint(2, 20))
    if lo == 0:
        hi = 0
    return dict(op=op, b=b, old_lo=lo, old_hi=max(lo, hi), chunks=chunks, new=new,
                idle=rng.randint(0, (b - chunks) // 6), ps=ps, hq=hq, hk=hk, hd=hd, window=window,
                gated=rng.random() < 0.5, type=kind)


def _lens(case):
    """The requests' old and new token counts, from the case alone."""
    rng = random.Random(case["b"] * 7919 + case["old_hi"] * 31 + case["new"])
    b, lo, hi = case["b"], case["old_lo"], case["old_hi"]
    old = [0 if hi == 0 else _logint(rng, max(lo, 1), max(hi, 1)) for _ in range(b)]
    new = [case["new"] if i < case["chunks"] else 0 if i >= b - case["idle"] else 1 for i in range(b)]
    return old, new


def _pages(n, ps):
    return -(-n // ps)


# ---- inputs ---------------------------------------------------------------------------------------

def _gen(seed, salt):
    return torch.Generator("cuda").manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _slots(table, old, new, ps):
    """[rows] of the flat cache row of every new token (numpy)."""
    out = []
    for b, (o, n) in enumerate(zip(old, new)):
        p = np.arange(o, o + n)
        out.append(table[b, p // ps] * ps + p % ps)
    return np.concatenate(out)


def _tables(seed, old, kv, ps, spare=3):
    """Pages in random order: the block table of the first `kv` tokens of every request, and the free ones."""
    need = [_pages(n, ps) for n in kv]
    total = sum(need)
    pages = np.random.default_rng([int(seed), 91]).permutation(total + spare)
    width = max(max(_pages(max(o, k), ps) for o, k in zip(old, kv)), 1)
    table = np.full((len(kv), width), -1, np.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pages[at:at + n]
        at += n
    return table, pages[total:], total + spare


_TABLE = {}


def _rope(rd):
    """[16384][rd / 2][2] cosines and sines, angles in 64 bits."""
    if rd not in _TABLE:
        t = torch.arange(16384, dtype=torch.float64)[:, None]
        a = t / THETA ** (torch.arange(0, rd, 2, dtype=torch.float64) / rd)
        _TABLE[rd] = torch.stack([a.cos(), a.sin()], -1).float().cuda().contiguous()
    return _TABLE[rd]


def _axis_of(rd, axes):
    """Each pair's axis: the time, height and width of an image's patches in turn."""
    return [j % axes for j in range(rd // 2)]


def _plan_inputs(case, seed):
    old, new = _lens(case)
    ps = case["ps"]
    need = sum(_pages(o + n, ps) - _pages(o, ps) for o, n in zip(old, new))
    table, free, n_pages = _tables(seed, [o + n for o, n in zip(old, new)], old, ps, need + 5)
    n_free = (need * 2) // 3 if case["short"] else len(free)
    return old, new, table, free, n_free, n_pages


def _prep_inputs(case, seed):
    old, new = _lens(case)
    t, ps, dt = sum(new), case["ps"], TYPES[case["type"]]
    hq, hk, hd = case["hq"], case["hk"], case["hd"]
    g = _gen(seed, 7)
    big = torch.randn(t, (hq * (2 if case["gated"] else 1) + 2 * hk) * hd, generator=g, device="cuda").to(dt)
    qw = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
    kw = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
    table, _, n_pages = _tables(seed, old, [o + n for o, n in zip(old, new)], ps)
    kp = torch.randn(n_pages * hk * ps * hd, generator=g, device="cuda").to(dt)
    vp = torch.randn(n_pages * hk * ps * hd, generator=g, device="cuda").to(dt)
    linear = np.concatenate([np.arange(o, o + n) for o, n in zip(old, new)])
    rng = np.random.default_rng([int(seed), 17])
    pos = np.stack([linear] + [rng.integers(0, 64, t) for _ in range(case["axes"] - 1)])
    return big, qw, kw, kp, vp, pos, _slots(table, old, new, ps), n_pages


def _attend_inputs(case, seed):
    old, new = _lens(case)
    t, ps, dt = sum(new), case["ps"], TYPES[case["type"]]
    hq, hk, hd = case["hq"], case["hk"], case["hd"]
    g = _gen(seed, 9)
    kv = [o + n for o, n in zip(old, new)]
    table, _, n_pages = _tables(seed, old, kv, ps)
    # queries and keys as their norms leave them, the query's weights above one: some keys matter more than others
    q = (1.5 * torch.randn(t, hq, hd, generator=g, device="cuda")).to(dt)
    kp = torch.randn(n_pages * hk * ps * hd, generator=g, device="cuda").to(dt)
    vp = torch.randn(n_pages * hk * ps * hd, generator=g, device="cuda").to(dt)
    big = torch.randn(t, (2 * hq + 2 * hk) * hd, generator=g, device="cuda").to(dt) if case["gated"] else None
    return old, new, kv, table, n_pages, q, kp, vp, big


def prepare(case, seed):
    st = dict(case)
    if case["op"] == "plan":
        old, new, table, free, n_free, n_pages = _plan_inputs(case, seed)
        b, t = case["b"], sum(new) + 7  # room for a few more rows than this step has
        st.update(lens=_ints(old), news=_ints(new), table=_ints(table.tolist()), free=torch.full((n_pages,), -1,
                  dtype=torch.int32, device="cuda"), n_free=_ints([n_free]), n_pages=n_pages, t=t,
                  cu=_ints([0] * (b + 1)), kv=_ints([0] * b), slots=_ints([0] * t), pos=_ints([0] * t),
                  status=_ints([0] * 4))
        st["free"][:len(free)] = _ints(free.tolist())
        return st
    if case["op"] == "prep":
        big, qw, kw, kp, vp, pos, slots, n_pages = _prep_inputs(case, seed)
        t = big.shape[0]
        st.update(big=big, qw=qw, kw=kw, rope=_rope(case["rd"]), pos=_ints(pos.tolist()), slots=_ints(slots.tolist()),
                  axis=torch.tensor(_axis_of(case["rd"], case["axes"]), dtype=torch.uint8, device="cuda"), t=t, kp=kp,
                  vp=vp, n_pages=n_pages, q=torch.zeros(t, case["hq"], case["hd"], device="cuda", dtype=big.dtype))
        return st
    old, new, kv, table, n_pages, q, kp, vp, big = _attend_inputs(case, seed)
    t = sum(new)
    st.update(new=max(new), news=new, kvs=kv, cu=_ints([0] + np.cumsum(new).tolist()), kv=_ints(kv),
              table=_ints(table.tolist()), n_pages=n_pages, q=q, kp=kp, vp=vp, big=big, t=t,
              out=torch.zeros(t, case["hq"] * case["hd"], device="cuda", dtype=q.dtype))
    if own:
        st["ws"] = torch.empty(_pkg().paged_attention_ws(case["b"], t, max(new), max(kv), case["hq"], case["hk"],
                                                         case["hd"]), dtype=torch.uint8, device="cuda")
    return st


# ---- one call -------------------------------------------------------------------------------------

def run(st):
    if own:
        return {"plan": _own_plan, "prep": _own_prep, "attend": _own_attend}[st["op"]](st)
    return {"plan": _plain_plan, "prep": _plain_prep, "attend": _plain_attend}[st["op"]](st)


def _own_plan(st):
    _pkg().op_page_plan(st["lens"].data_ptr(), st["news"].data_ptr(), st["b"], st["t"], st["ps"], st["n_pages"],
                        st["free"].data_ptr(), st["n_free"].data_ptr(), st["table"].data_ptr(), st["table"].shape[1],
                        st["cu"].data_ptr(), st["kv"].data_ptr(), st["slots"].data_ptr(), st["pos"].data_ptr(),
                        st["status"].data_ptr())
    return {k: st[k] for k in ("table", "cu", "kv", "slots", "pos", "status")}


def _own_prep(st):
    sd = _pkg()
    sd.op_paged_prep(st["big"].data_ptr(), st["big"].shape[1], st["gated"], st["qw"].data_ptr(), st["kw"].data_ptr(),
                     st["rope"].data_ptr(), st["rope"].shape[0], st["pos"].data_ptr(), st["axes"],
                     st["axis"].data_ptr(), st["slots"].data_ptr(), st["t"], st["hq"], st["hk"], st["hd"], st["rd"],
                     st["ps"], st["n_pages"], st["q"].data_ptr(), st["kp"].data_ptr(), st["vp"].data_ptr(),
                     sd.F16 if st["type"] == "f16" else sd.BF16)
    return {k: st[k] for k in ("q", "kp", "vp")}


def _own_attend(st):
    sd = _pkg()
    sd.op_paged_attention(st["q"].data_ptr(), st["big"].data_ptr() if st["gated"] else None,
                          st["big"].shape[1] if st["gated"] else 0, st["kp"].data_ptr(), st["vp"].data_ptr(),
                          st["table"].data_ptr(), st["table"].shape[1], st["cu"].data_ptr(), st["kv"].data_ptr(),
                          st["b"], st["t"], st["new"], max(st["kvs"]), st["hq"], st["hk"], st["hd"], st["ps"],
                          st["n_pages"], st["out"].data_ptr(), st["ws"].data_ptr(), st["ws"].numel(),
                          sd.F16 if st["type"] == "f16" else sd.BF16, window=st["window"])
    return st["out"]


def _plain_plan(st):
    ps, t, b = st["ps"], st["t"], st["b"]
    lens, news, table = st["lens"].long(), st["news"].long(), st["table"]
    dev = lens.device
    have, want = (lens + ps - 1) // ps, (lens + news + ps - 1) // ps
    need = want - have
    rows_to, pages_to = news.cumsum(0), need.cumsum(0)
    n_free = st["n_free"].long()
    fits = (rows_to <= t) & (pages_to <= n_free) & (want <= table.shape[1])
    admitted = fits.long().cumprod(0)
    news, need = news * admitted, need * admitted
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), news.cumsum(0)])
    first = need.cumsum(0) - need  # the pages taken before each request's
    j = torch.arange(table.shape[1], device=dev)
    k = first[:, None] + j - have[:, None]
    taken = (j >= have[:, None]) & (j < (have + need)[:, None])
    page = st["free"].long()[(n_free - 1 - k).clamp(0, st["n_pages"] - 1)]
    table.copy_(torch.where(taken, page, table.long()))
    r = torch.arange(t, device=dev)
    seq = (r[:, None] >= cu[1:]).sum(1)
    live = seq < b
    seq = seq.clamp(max=b - 1)
    p = lens[seq] + r - cu[seq]
    slot = table.long()[seq, (p // ps).clamp(0, table.shape[1] - 1)] * ps + p % ps
    status = torch.stack([admitted.sum(), news.sum(), need.sum(), (n_free - need.sum())[0]])
    return {"table": table, "cu": cu.int(), "kv": (lens + news).int(), "slots": torch.where(live, slot, -1).int(),
            "pos": torch.where(live, p, 0).int(), "status": status.int()}


def _norm_rotate(x, w, cos, sin, rd):
    """[rows][heads][hd] f32: RMSNorm, then the rotation of dims j and j + rd / 2 by the pair's angle."""
    x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w
    lo, hi = x[..., :rd // 2], x[..., rd // 2:rd]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., rd:]], -1)


def _plain_prep(st):
    t, hq, hk, hd, rd, ps = st["t"], st["hq"], st["hk"], st["hd"], st["rd"], st["ps"]
    big, qd = st["big"], hq * hd * (2 if st["gated"] else 1)
    q = big[:, :qd].view(t, hq, -1)[:, :, :hd].float()
    k = big[:, qd:qd + hk * hd].view(t, hk, hd).float()
    v = big[:, qd + hk * hd:qd + 2 * hk * hd].view(t, hk, hd)
    pos = st["pos"].long()[st["axis"].long()]  # [rd / 2][rows]
    cs = st["rope"][pos, torch.arange(rd // 2, device=big.device)[:, None]].transpose(0, 1)[:, None]
    q = _norm_rotate(q, st["qw"], cs[..., 0], cs[..., 1], rd).to(big.dtype)
    k = _norm_rotate(k, st["kw"], cs[..., 0], cs[..., 1], rd).to(big.dtype)
    slot = st["slots"].long()
    page, blk, row = slot // ps, slot % ps // 32, slot % 32
    st["kp"].view(-1, hk, ps // 32, hd // 32, 32, 32)[page, :, blk, :, row] = k.view(t, hk, hd // 32, 32)
    st["vp"].view(-1, hk, ps // 32, hd, 32)[page, :, blk, :, row] = v
    return {"q": q, "kp": st["kp"], "vp": st["vp"]}


def _plain_attend(st):
    hq, hk, hd, ps = st["hq"], st["hk"], st["hd"], st["ps"]
    q, dev = st["q"], st["q"].device
    kp = st["kp"].view(-1, hk, ps // 32, hd // 32, 32, 32)
    vp = st["vp"].view(-1, hk, ps // 32, hd, 32)
    out, at = torch.zeros(st["t"], hq, hd, device=dev), 0
    for b, (n, kv) in enumerate(zip(st["news"], st["kvs"])):
        if n == 0:
            continue
        pages = st["table"][b, :_pages(kv, ps)].long()
        k = kp[pages].permute(1, 0, 2, 4, 3, 5).reshape(hk, -1, hd)[:, :kv].float()
        v = vp[pages].permute(1, 0, 2, 4, 3).reshape(hk, -1, hd)[:, :kv].float()
        p = torch.arange(kv - n, kv, device=dev)[:, None]
        j = torch.arange(kv, device=dev)
        seen = j <= p
        if st["window"]:
            seen &= j > p - st["window"]
        # the query heads of a key/value head are rows of one product
        x = q[at:at + n].float().view(n, hk, -1, hd).transpose(0, 1).reshape(hk, -1, hd)
        s = (x @ k.transpose(1, 2).contiguous()).view(hk, n, -1, kv) * (1 / math.sqrt(hd))
        s = s.masked_fill(~seen[:, None], -math.inf)
        e = (s - s.max(-1, keepdim=True).values).exp()
        o = (e.view(hk, -1, kv) @ v).view(hk, n, -1, hd) / e.sum(-1, keepdim=True)
        out[at:at + n] = o.transpose(0, 1).reshape(n, hq, hd)
        at += n
    if st["gated"]:
        gate = st["big"][:, :2 * hq * hd].view(-1, hq, 2, hd)[:, :, 1].float()
        out = out / (1 + (-gate).exp())
    return out.to(q.dtype).view(st["t"], hq * hd)


# ---- what a call cannot do without ----------------------------------------------------------------

def _seen(old, new, window):
    """Keys that the rows of one request see, summed over its rows, and the distinct ones among them."""
    if not window:
        return new * old + new * (new + 1) // 2, old + new if new else 0
    pairs = sum(min(window, old + i + 1) for i in range(new))
    return pairs, min(old + new, window + new - 1) if new else 0


def work(case):
    old, new = _lens(case)
    t = sum(new)
    if case["op"] == "plan":
        ps = case["ps"]
        need = sum(_pages(o + n, ps) - _pages(o, ps) for o, n in zip(old, new))
        return {"bytes": 4 * (4 * case["b"] + 2 * need + 2 * t + 6), "flops": 0}
    hq, hk, hd = case["hq"], case["hk"], case["hd"]
    if case["op"] == "prep":
        row = (hq + 2 * hk) * hd
        return {"bytes": 4 * t * row + 4 * t * (1 + case["axes"]) + 4 * t * case["rd"] + 8 * hd,
                "flops": t * (hq + hk) * (4 * hd + 3 * case["rd"])}
    pairs = [_seen(o, n, case["window"]) for o, n in zip(old, new)]
    return {"bytes": 4 * hk * hd * sum(p[1] for p in pairs) + 2 * t * hq * hd * (3 if case["gated"] else 2),
            "flops": 4 * hq * hd * sum(p[0] for p in pairs)}


# ---- 64-bit results -------------------------------------------------------------------------------

def _exact_plan(case, seed):
    """The definition, request by request."""
    old, new, table, free, n_free, n_pages = _plan_inputs(case, seed)
    ps, b, t = case["ps"], case["b"], sum(new) + 7
    table, left = table.copy(), n_free
    cu, kv, slots, pos, open_, admitted = [0], [], [], [], True, 0
    for i in range(b):
        need = list(range(_pages(old[i], ps), _pages(old[i] + new[i], ps)))
        open_ = open_ and cu[-1] + new[i] <= t and len(need) <= left and _pages(old[i] + new[i], ps) <= table.shape[1]
        n = 0
        if open_:
            admitted, n = admitted + 1, new[i]
            for j in need:
                left -= 1
                table[i, j] = free[left]
            for p in range(old[i], old[i] + n):
                slots.append(int(table[i, p // ps]) * ps + p % ps)
                pos.append(p)
        cu.append(cu[-1] + n)
        kv.append(old[i] + n)
    slots += [-1] * (t - len(slots))
    pos += [0] * (t - len(pos))
    return {"table": _ints(table.tolist()), "cu": _ints(cu), "kv": _ints(kv), "slots": _ints(slots), "pos": _ints(pos),
            "status": _ints([admitted, cu[-1], n_free - left, left])}


def _exact_prep(case, seed):
    big, qw, kw, kp, vp, pos, slots, n_pages = _prep_inputs(case, seed)
    hq, hk, hd, rd, ps = case["hq"], case["hk"], case["hd"], case["rd"], case["ps"]
    t, per = big.shape[0], 2 if case["gated"] else 1
    x = big.double().view(t, hq * per + 2 * hk, hd)
    turn = torch.ones(t, rd // 2, dtype=torch.complex128, device="cuda")
    for j, a in enumerate(_axis_of(rd, case["axes"])):
        cs = _rope(rd)[torch.from_numpy(pos[a]).cuda(), j].double()
        turn[:, j] = torch.complex(cs[:, 0], cs[:, 1])

    def heads(x, w):
        x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / hd + EPS) * w.double()
        z = torch.complex(x[..., :rd // 2], x[..., rd // 2:rd]) * turn[:, None]
        return torch.cat([z.real, z.imag, x[..., rd:]], -1)

    q, k = heads(x[:, :hq * per:per], qw), heads(x[:, hq * per:hq * per + hk], kw)
    v = x[:, hq * per + hk:]
    slot = torch.from_numpy(slots).cuda()
    # element (head h, dim d) of a slot: in the block of 32 rows h * (ps / 32) + row / 32 of its page
    h, d = torch.arange(hk, device="cuda")[:, None], torch.arange(hd, device="cuda")
    block = (slot // ps * hk * ps)[:, None, None] + h * ps + (slot % ps // 32 * 32)[:, None, None]
    row = (slot % 32)[:, None, None]
    kp, vp = kp.double(), vp.double()
    kp[block * hd + d // 32 * 1024 + row * 32 + d % 32] = k
    vp[block * hd + d * 32 + row] = v
    return {"q": q, "kp": kp, "vp": vp}


def _exact_attend(case, seed):
    old, new, kvs, table, n_pages, q, kp, vp, big = _attend_inputs(case, seed)
    hq, hk, hd, ps = case["hq"], case["hk"], case["hd"], case["ps"]
    g, w = hq // hk, case["window"]
    out, at = torch.zeros(sum(new), hq, hd, dtype=torch.float64, device="cuda"), 0
    d = torch.arange(hd, device="cuda")
    for b, (n, kv) in enumerate(zip(new, kvs)):
        if n == 0:
            continue
        p = np.arange(kv)
        row = torch.from_numpy(table[b, p // ps] * ps * hk + p % ps // 32 * 32).cuda()[:, None]  # head 0's block
        inside = torch.from_numpy(p % 32).cuda()[:, None]
        for kh in range(hk):
            block = (row + kh * ps) * hd
            k = kp[block + d // 32 * 1024 + inside * 32 + d % 32].double()
            v = vp[block + d * 32 + inside].double()
            for t0 in range(0, n, 512):
                t1 = min(n, t0 + 512)
                first = max(0, kv - n + t0 - w + 1) if w else 0
                last = kv - n + t1
                z = q[at + t0:at + t1, kh * g:(kh + 1) * g].double().reshape(-1, hd) @ k[first:last].T / math.sqrt(hd)
                z = z.view(t1 - t0, g, -1)
                back = torch.arange(kv - n + t0, kv - n + t1, device="cuda")[:, None] - torch.arange(first, last, device="cuda")
                hide = back < 0
                if w:
                    hide |= back >= w
                z = torch.softmax(z.masked_fill(hide[:, None], -math.inf), -1)
                out[at + t0:at + t1, kh * g:(kh + 1) * g] = (z.view(-1, last - first) @ v[first:last]).view(t1 - t0, g, hd)
        at += n
    if big is not None:
        out *= torch.sigmoid(big.double()[:, :2 * hq * hd].reshape(-1, hq, 2, hd)[:, :, 1])
    return out.reshape(-1, hq * hd)


def exact(case, seed):
    return {"plan": _exact_plan, "prep": _exact_prep, "attend": _exact_attend}[case["op"]](case, seed)
