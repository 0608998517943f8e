"""What the entry points of rotary positions and of rows that leave the paged cache refuse, on the CPU: every refusal comes
before any device call, so the addresses here are never used."""
import math

import numpy as np
import pytest

import evict_ref as er

A = 1 << 20  # an aligned address that is not there
M = 1 << 20


def refuses(sdamd, call, base, kw, who, message):
    with pytest.raises(sdamd.EngineError, match=who + ": .*" + message):
        call(**{**base, **kw})


@pytest.mark.parametrize("kw,message", [
    (dict(RD=3), "rotary_dim"), (dict(RD=2, scaling=2), "rotary_dim"), (dict(RD=258), "rotary_dim"), (dict(RD=0), "rotary_dim"),
    (dict(theta=0.5), "theta"), (dict(theta=math.inf), "theta"), (dict(theta=math.nan), "theta"), (dict(factor=0.5), "theta"),
    (dict(factor=math.nan), "theta"), (dict(scaling=4), "no such"), (dict(scaling=-1), "no such"), (dict(scaling=3), "in parts"),
    (dict(scaling=3, length=4096.0, low=2.0, high=2.0), "in parts"), (dict(scaling=3, length=4096.0, low=-1.0, high=2.0), "in parts"),
    (dict(scaling=3, length=math.inf, low=1.0, high=2.0), "in parts"), (dict(scaling=3, length=1.0, low=1.0, high=math.inf), "in parts"),
])
def test_freqs_refuses(sdamd, kw, message):
    refuses(sdamd, sdamd.rope_freqs, dict(RD=64, theta=1e4, scaling=1, factor=2.0), kw, "sd_rope_freqs", message)


@pytest.mark.parametrize("rd,theta,factor", [(4, 1e4, 1e160), (64, 1e300, 1e9)])
def test_freqs_refuses_a_base_past_all_numbers(sdamd, rd, theta, factor):
    """(All frequencies but the first would be 0.)"""
    refuses(sdamd, sdamd.rope_freqs, dict(RD=rd, theta=theta, scaling=2, factor=factor), {}, "sd_rope_freqs", "theta scaled")


@pytest.mark.parametrize("rd,theta,kw", [
    (64, 1e7, {}), (2, 1e4, {}), (256, 1e6, dict(scaling="linear", factor=8.0)), (24, 1e4, dict(scaling="base", factor=4.0)),
    (4, 1e4, dict(scaling="base", factor=1.0)), (128, 5e5, dict(scaling="parts", factor=8.0, length=8192.0, low=1.0, high=4.0)),
    (64, 1.0, dict(scaling="parts", factor=1.0, length=1.0, low=0.0, high=1.0)),
])
def test_freqs(sdamd, rd, theta, kw):
    """Against the definition: pow within 2 roundings of f64, the rest a few more."""
    kinds = dict(plain=0, linear=1, base=2, parts=3)
    got = sdamd.rope_freqs(rd, theta, **{**kw, "scaling": kinds[kw.get("scaling", "plain")]})
    want = er.freqs(rd, theta, **kw)
    np.testing.assert_allclose(got, want, rtol=64 * 2.0 ** -53, atol=0)


TABLE = dict(freqs=A, pairs=32, pos=A + 4096, n=100, table=A + 8192)


@pytest.mark.parametrize("kw,message", [
    (dict(freqs=None), "null"), (dict(table=None), "null"), (dict(pairs=0), "pairs"), (dict(pairs=129), "pairs"), (dict(n=0), "at least one row"),
    (dict(n=1 << 26), "2\\^31"), (dict(magnitude=math.inf), "magnitude"), (dict(freqs=A + 4), "aligned"), (dict(table=A + 8196), "aligned"),
    (dict(pos=A + 4098), "aligned"), (dict(pos=A + 8192 + 25596), "overlaps an input"), (dict(table=A + 248), "overlaps an input"),
])
def test_table_refuses(sdamd, kw, message):
    refuses(sdamd, sdamd.op_rope_table, TABLE, kw, "sd_op_rope_table", message)


ROPE = dict(freqs=A, RD=64, layout=0, pos=A + 1024, T=4, HD=128, Q=A + M, q_stride=768, q_step=128, HQ=4, K=A + M + 1024, k_stride=768,
            k_step=128, HK=1, type=0)
OUT = dict(Qo=A + 2 * M, Ko=A + 3 * M)


@pytest.mark.parametrize("kw,message", [
    (dict(freqs=None), "null"), (dict(Q=None), "null"), (dict(T=0), "at least one row"), (dict(HQ=0), "q heads"), (dict(HQ=1025), "q heads"),
    (dict(HK=0), "q heads"), (dict(HD=100), "head_dim"), (dict(HD=2048), "head_dim"), (dict(HD=4), "head_dim"), (dict(RD=0), "rotary_dim"), (dict(RD=63), "rotary_dim"),
    (dict(RD=130), "rotary_dim"), (dict(HD=512, RD=258, q_step=512, q_stride=4096, k_step=512, k_stride=4096), "rotary_dim"), (dict(layout=2), "layout"), (dict(type=3), "type"),
    (dict(magnitude=math.nan), "magnitude"), (dict(Ko=A + 3 * M), "both q and k"), (dict(Qo=A + 2 * M), "both q and k"), (dict(OUT, K=None), "both q and k"),
    (dict(q_stride=772), "multiples of 8"), (dict(k_step=129), "multiples of 8"), (dict(q_stride=504), "heads overlap"), (dict(q_step=120), "heads overlap"),
    (dict(k_stride=64), "heads overlap"), (dict(OUT, qo_stride=256), "heads overlap"), (dict(q_stride=0), "heads overlap"), (dict(q_stride=1 << 41), "multiples of 8"),
    (dict(Q=A + M + 8), "16 bytes"), (dict(OUT, Ko=A + 3 * M + 2), "16 bytes"), (dict(freqs=A + 4), "8 bytes"), (dict(pos=A + 1026), "aligned"),
    (dict(OUT, Qo=A + M + 16), "overlaps an input"), (dict(OUT, Ko=A + M), "overlaps an input"), (dict(pos=A + M + 64), "overlaps an input"),
    (dict(freqs=A + M), "overlaps an input"),
])
def test_rope_refuses(sdamd, kw, message):
    refuses(sdamd, sdamd.op_rope, ROPE, kw, "sd_op_rope", message)


HERE = dict(Qo=A + M, qo_stride=768, qo_step=128, Ko=A + M + 1024, ko_stride=768, ko_step=128)  # ROPE's own rows
ONLY = dict(K=None, k_stride=0, k_step=0, HK=0)


@pytest.mark.parametrize("kw,message", [
    (dict(Qo=A + M, Ko=A + 3 * M), "overlaps an input"), (dict(ONLY, Qo=A + M), "overlaps an input"),  # dense rows over strided ones
    (dict(HERE, qo_stride=1536), "overlaps an input"), (dict(HERE, ko_stride=1536), "overlaps an input"), (dict(HERE, qo_step=136), "overlaps an input"),
    (dict(HERE, Ko=A + M), "overlaps an input"), (dict(HERE, Ko=A + M + 1040), "overlaps an input"), (dict(HERE, Ko=A + M + 768), "overlaps an input"),
    (dict(HERE, Qo=A + M + 256), "overlaps an input"), (dict(OUT, Ko=A + 2 * M), "q head overlaps a k head"), (dict(OUT, Ko=A + 2 * M + 1024), "q head overlaps a k head"),
    (dict(OUT, qo_stride=768, ko_stride=768, Ko=A + 2 * M + 768), "q head overlaps a k head"),
    (dict(OUT, qo_stride=768, ko_stride=760, Ko=A + 2 * M + 1024), "q head overlaps a k head"),  # (row 3's: 24 dims of it)
    (dict(OUT, qo_stride=768, ko_stride=768, Ko=A + 2 * M + 1040, HK=2), "q head overlaps a k head"),  # (in the next row's first)
    (dict(K=A + M), "q head overlaps a k head"), (dict(K=A + M + 128 * 2), "q head overlaps a k head"), (dict(K=A + M + 1008), "q head overlaps a k head"),
    (dict(K=A + M + 768 * 2 - 128 * 2, HK=2), "q head overlaps a k head"), (dict(T=1, K=A + M + 768), "q head overlaps a k head"),
    (dict(HERE, K=A + M + 768, Ko=A + 3 * M), "q head overlaps a k head"),  # (q in place over k that is read)
])
def test_rope_refuses_rows_over_rows(sdamd, kw, message):
    """What is written is the heads' own place, or apart from all that is read and written."""
    refuses(sdamd, sdamd.op_rope, ROPE, kw, "sd_op_rope", message)


POSITIONS = dict(cu=A, dropped=A + 4096, B=8, T=100, pos=A + 8192, out=A + 12288)


@pytest.mark.parametrize("kw,message", [
    (dict(cu=None), "null"), (dict(dropped=None), "null"), (dict(pos=None), "null"), (dict(out=None), "null"), (dict(B=0), "requests"), (dict(B=8193), "requests"),
    (dict(T=0), "rows"), (dict(T=(1 << 30) + 1), "rows"), (dict(out=A + 12290), "aligned"), (dict(out=A + 8196), "overlaps an input"), (dict(out=A + 32), "overlaps an input"),
    (dict(out=A + 4096 - 396), "overlaps an input"),
])
def test_positions_refuses(sdamd, kw, message):
    refuses(sdamd, sdamd.op_page_positions, POSITIONS, kw, "sd_op_page_positions", message)


WEIGHTS = dict(Q=A, Kp=A + M, table=A + 2 * M, max_blocks=8, cu=A + 3 * M, kv_lens=A + 4 * M, B=2, T=4, max_new=2, max_kv=200, HQ=4, HK=1, HD=128,
               page_size=32, n_pages=10, scores=A + 5 * M, out=A + 6 * M, ws=A + 64 * M, ws_bytes=1 << 40, type=1, pos=A + 7 * M, kpos=A + 8 * M)
LONG = dict(max_blocks=2048, max_kv=60000)  # (short ones need no workspace)


@pytest.mark.parametrize("kw,message", [
    (dict(Q=None), "null"), (dict(Kp=None), "null"), (dict(out=None), "null"), (dict(cu=None), "null"), (dict(pos=None), "positions of both"), (dict(kpos=None), "positions of both"),
    (dict(scores=None), "decay needs"), (dict(decay=math.inf), "decay"), (dict(decay=math.nan), "decay"), (dict(HD=96), "head_dim"), (dict(HQ=3, HK=2), "multiple of kv heads"),
    (dict(type=2), "type"), (dict(page_size=48), "power of two"), (dict(n_pages=0), "at least one page"), (dict(page_stride=8), "page stride"), (dict(B=0), "requests"),
    (dict(B=8193), "requests"), (dict(T=0), "at least one row"), (dict(T=1 << 29), "2\\^30"), (dict(max_new=0), "max_new"), (dict(max_kv=0), "max_new"), (dict(max_kv=257), "more than a table row"),
    (dict(max_blocks=0), "table row"), (dict(max_blocks=1 << 26), "table row"), (dict(window=-1), "window"), (dict(observers=-1), "observers"), (dict(scale=0.0), "scale"),
    (dict(scale=math.nan), "scale"), (dict(scale=2.4e38), "scale"), (dict(Q=A + 8), "16 bytes"), (dict(ws=A + 64 * M + 4), "16 bytes"), (dict(out=A + 6 * M + 2), "4 bytes"),
    (dict(out=A + 5 * M + 4), "overlaps an input"), (dict(out=A + M), "overlaps an input"), (dict(kpos=A + 6 * M), "outputs overlap"), (dict(kpos=A + 5 * M), "overlaps an input"),
    (dict(LONG, ws_bytes=0), "workspace"), (dict(LONG, ws=None), "workspace"), (dict(LONG, ws=A), "overlaps an input"),
    (dict(LONG, out=A + 32 * M, ws=A + 32 * M), "outputs overlap"), (dict(LONG, ws=A + 5 * M), "overlaps"),
    (dict(LONG, scores=A + 5 * M, out=A + 5 * M, ws=A + 5 * M), "overlap"), (dict(T=100, max_new=50, ws_bytes=1024), "workspace"),
])
def test_weights_refuses(sdamd, kw, message):
    refuses(sdamd, sdamd.op_paged_weights, WEIGHTS, kw, "sd_op_paged_weights", message)


def test_weights_workspace(sdamd):
    for B, T, new, kv in [(1, 1, 1, 1), (64, 64, 1, 8192), (1, 1, 1, 2 ** 31 - 1), (8192, 8192, 1, 100), (2, 4096, 4096, 4096)]:
        for hq, hk, hd in [(8, 2, 256), (32, 8, 128), (12, 1, 64)]:
            for obs in (0, 1, 40):
                need = sdamd.paged_weights_ws(B, T, new, kv, hq, hk, hd, obs)
                assert 0 <= need < 1 << 44 and need % 16 == 0
                assert need or kv <= 8192  # (short caches, whose few rows' scores fit into LDS, need none)
    for bad in [(0, 1, 1, 1, 8, 2, 256), (1, 0, 1, 1, 8, 2, 256), (1, 1, 0, 1, 8, 2, 256), (1, 1, 1, 0, 8, 2, 256), (1, 1, 1, 1, 7, 2, 256),
                (1, 1, 1, 1, 8, 2, 100), (1, 1, 1, 1, 8, 2, 64, -1)]:
        with pytest.raises(sdamd.EngineError, match="sd_op_paged_weights_ws: "):
            sdamd.paged_weights_ws(*bad)


def least_workspace(sdamd, **kw):
    with pytest.raises(sdamd.EngineError, match="at least [0-9]+, got 16$") as e:
        sdamd.op_paged_weights(**{**WEIGHTS, **kw, "ws_bytes": 16})
    return int(str(e.value).split("at least ")[1].split(",")[0])


@pytest.mark.parametrize("B,new,max_new", [(1024, 1, 1), (256, 16, 3841), (64, 8, 8)])
def test_weights_least_workspace(sdamd, B, new, max_new):
    """The scores of one request under a far bound, where all requests' would be gigabytes."""
    T, hq, hk, hd, kv = B * new, 32, 8, 128, 131072
    least = least_workspace(sdamd, B=B, T=T, max_new=max_new, max_kv=kv, HQ=hq, HK=hk, HD=hd, max_blocks=4096)
    rows = min(new, 8) * 4 if max_new == new else 4
    one = hk * rows * kv * 4
    assert one < least < 1.3 * one + T * hq * 16 + (64 << 20)
    assert sdamd.paged_weights_ws(B, T, max_new, kv, hq, hk, hd) >= B * one


def test_weights_workspace_of_parts(sdamd):
    """A chunk in several parts beside single tokens: slots for its parts alone, whatever the requests."""
    sizes = dict(T=8447, max_new=8192, max_kv=131072, HQ=32, HK=8, HD=128, max_blocks=4096)
    few = [least_workspace(sdamd, B=b, **sizes) for b in (2, 256, 1024)]
    assert max(few) < min(few) + (8 << 20) and max(few) < 120 << 20


@pytest.mark.parametrize("B,T,max_new,max_kv,ok", [(2048, 8192, 4096, 131072, True), (8192, 16000, 100, 262016, True), (8192, 16000, 100, 262144, False), (8192, 16000, 100, 1 << 20, False),
                                                   (8192, 8192, 1, 1 << 20, True), (1, 4096, 4096, (1 << 31) - 128, True), (2, 4096, 4096, (1 << 31) - 1, False)])
def test_weights_largest(sdamd, B, T, max_new, max_kv, ok):
    """Requests times tiles of keys that a call takes: below 2^24."""
    call = lambda: sdamd.paged_weights_ws(B, T, max_new, max_kv, 32, 8, 128)
    if ok:
        assert call() > 0
    else:
        with pytest.raises(sdamd.EngineError, match="too many rows and keys"):
            call()


EVICT = dict(scores=A, kpos=A + M, table=A + 2 * M, max_blocks=8, kv_lens=A + 3 * M, budgets=A + 4 * M, B=2, max_kv=200, HK=2, page_size=32,
             n_pages=20, sink=0, recent=0, new_lens=A + 5 * M, moves=A + 6 * M, counts=A + 7 * M, ws=A + 8 * M, ws_bytes=1 << 40)


@pytest.mark.parametrize("kw,message", [
    (dict(scores=None), "null"), (dict(budgets=None), "null"), (dict(moves=None), "null"), (dict(counts=None), "null"), (dict(new_lens=None), "null"), (dict(B=0), "requests"),
    (dict(B=8193), "requests"), (dict(HK=0), "kv heads"), (dict(HK=1025), "kv heads"), (dict(page_size=31), "power of two"), (dict(n_pages=0), "at least one page"), (dict(max_kv=0), "max_kv"),
    (dict(max_kv=257), "more than a table row"), (dict(max_blocks=0), "table row"), (dict(sink=-1), "sink"), (dict(recent=-1), "recent"), (dict(moves=A + 6 * M + 2), "4 bytes"),
    (dict(new_lens=A + 3 * M), "overlaps an input"), (dict(moves=A + M), "overlaps an input"), (dict(counts=A + 6 * M + 8), "outputs overlap"), (dict(ws=A + 8 * M + 8), "16 bytes"),
    (dict(max_blocks=2048, max_kv=40000, ws_bytes=1024), "workspace"), (dict(max_blocks=2048, max_kv=40000, ws=None), "workspace"),
    (dict(max_blocks=2048, max_kv=40000, ws=A), "overlaps an input"), (dict(max_blocks=2048, max_kv=40000, ws=A + 6 * M), "outputs overlap"),
])
def test_evict_refuses(sdamd, kw, message):
    refuses(sdamd, sdamd.op_page_evict, EVICT, kw, "sd_op_page_evict", message)


def test_evict_workspace(sdamd):
    for B, kv, hk in [(1, 1, 1), (64, 8192, 8), (8192, 100, 2), (2, 131072, 2), (1, 2 ** 31 - 1, 1)]:
        assert 0 <= sdamd.page_evict_ws(B, kv, hk) < 1 << 40
    for bad in [(0, 1, 1), (8193, 1, 1), (1, 0, 1), (1, 1, 0)]:
        with pytest.raises(sdamd.EngineError, match="sd_op_page_evict_ws: "):
            sdamd.page_evict_ws(*bad)


MOVE = dict(moves=A, counts=A + M, table=A + 2 * M, max_blocks=8, B=2, max_kv=200, HK=2, HD=64, page_size=32, n_pages=20, Kp=A + 3 * M, Vp=A + 4 * M,
            scores=A + 5 * M, kpos=A + 6 * M, type=0)


@pytest.mark.parametrize("kw,message", [
    (dict(moves=None), "null"), (dict(counts=None), "null"), (dict(Kp=None), "null"), (dict(Vp=None), "null"), (dict(B=0), "requests"), (dict(HD=32), "head_dim"), (dict(type=2), "type"),
    (dict(page_stride=100), "page stride"), (dict(max_kv=0), "max_kv"), (dict(max_kv=300), "more than a table row"), (dict(Kp=A + 3 * M + 8), "16 bytes"), (dict(kpos=A + 6 * M + 1), "4 bytes"),
    (dict(scores=A + 6 * M), "outputs overlap"), (dict(Vp=A), "overlaps an input"), (dict(scores=A + 3 * M), "overlaps an input"), (dict(kpos=A + 4 * M), "overlap"),
    (dict(Kp=A + 2 * M), "overlaps an input"),
])
def test_move_refuses(sdamd, kw, message):
    refuses(sdamd, sdamd.op_paged_move, MOVE, kw, "sd_op_paged_move", message)


RELEASE = dict(kv_lens=A, new_lens=A + 4096, dropped=A + 8192, table=A + 12288, max_blocks=4, B=4, page_size=32, n_pages=20, free_pages=A + 16384,
               n_free=A + 20480, dropped_out=A + 24576, n_free_out=A + 28672)


@pytest.mark.parametrize("kw,message", [
    (dict(kv_lens=None), "null"), (dict(free_pages=None), "null"), (dict(n_free_out=None), "null"), (dict(B=0), "requests"), (dict(B=8193), "requests"), (dict(page_size=16), "power of two"),
    (dict(n_pages=0), "at least one page"), (dict(max_blocks=0), "table row"), (dict(max_blocks=1 << 26), "table row"), (dict(n_free=A + 20482), "4 bytes"),
    (dict(n_free_out=A + 20480), "overlaps an input"), (dict(dropped_out=A + 8192), "overlaps an input"), (dict(n_free_out=A + 24588), "outputs overlap"),
])
def test_release_refuses(sdamd, kw, message):
    refuses(sdamd, sdamd.op_page_release, RELEASE, kw, "sd_op_page_release", message)
