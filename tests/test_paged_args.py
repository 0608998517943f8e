"""What the paged cache's entry points refuse, on the CPU: every refusal comes before any device call, so the addresses
here are never used."""
import pytest

A = 1 << 20  # an aligned address that is not there


def plan(sdamd, **kw):
    a = dict(lens=A, news=A + 4096, B=4, T=8, page_size=32, n_pages=10, free_pages=A + 8192, n_free=A + 12288, table=A + 16384,
             max_blocks=4, cu=A + 20480, kv_lens=A + 24576, slots=A + 28672, pos=A + 32768, status=A + 36864)
    a.update(kw)
    sdamd.op_page_plan(**a)


def prep(sdamd, **kw):
    a = dict(big=A, stride=768, gated=False, qw=A, kw=A, rope=A, rope_len=100, pos=A, axes=1, pair_axis=None, slots=A, T=4, HQ=4,
             HK=1, HD=128, RD=64, page_size=32, n_pages=10, Q=A, Kp=A, Vp=A, type=0)
    a.update(kw)
    sdamd.op_paged_prep(**a)


def attn(sdamd, **kw):
    a = dict(Q=A, big=None, stride=0, Kp=A, Vp=A, table=A, max_blocks=8, cu=A, kv_lens=A, B=2, T=4, max_new=2, max_kv=200, HQ=4,
             HK=1, HD=128, page_size=32, n_pages=10, out=A + 65536, ws=A, ws_bytes=1 << 40, type=1)
    a.update(kw)
    sdamd.op_paged_attention(**a)


@pytest.mark.parametrize("kw,message", [
    (dict(lens=None), "null argument"), (dict(status=None), "null argument"), (dict(free_pages=None), "null argument"),
    (dict(B=0), "requests"), (dict(B=8193), "requests"), (dict(T=0), "rows"), (dict(T=(1 << 30) + 1), "rows"),
    (dict(page_size=16), "power of two"), (dict(page_size=48), "power of two"), (dict(page_size=0), "power of two"),
    (dict(page_size=-32), "power of two"), (dict(n_pages=0), "at least one page"), (dict(n_pages=1 << 26), "2\\^31"),
    (dict(max_blocks=0), "table row"), (dict(max_blocks=1 << 26), "table row"),
    (dict(kv_lens=A), "overlaps an input"), (dict(status=A + 12288), "overlaps an input"), (dict(slots=A + 8192 + 36), "overlaps an input"),
    (dict(cu=A + 24576 + 12), "two outputs overlap"), (dict(table=A + 28672 - 4), "two outputs overlap"),
    (dict(pos=A + 32770), "aligned"), (dict(lens=A + 1), "aligned"),
])
def test_plan_refuses(sdamd, kw, message):
    with pytest.raises(sdamd.EngineError, match="sd_op_page_plan: .*" + message):
        plan(sdamd, **kw)


@pytest.mark.parametrize("kw,message", [
    (dict(big=None), "null argument"), (dict(Q=None), "null argument"), (dict(slots=None), "null argument"),
    (dict(T=0), "at least one row"), (dict(T=1 << 29, HQ=4), "2\\^30"), (dict(HQ=3, HK=2), "multiple of kv heads"),
    (dict(HK=0), "multiple of kv heads"), (dict(HQ=2048, stride=1 << 20), "multiple of kv heads"), (dict(HD=96), "head_dim"), (dict(HD=512), "head_dim"),
    (dict(type=2), "type"), (dict(type=-1), "type"), (dict(qw=None), "both q and k"), (dict(kw=None), "both q and k"),
    (dict(RD=3), "rotary_dim"), (dict(RD=130), "rotary_dim"), (dict(RD=-2), "rotary_dim"), (dict(rope=None), "table and the positions"),
    (dict(pos=None), "table and the positions"), (dict(rope_len=0), "table and the positions"), (dict(axes=0), "axes"),
    (dict(axes=5, pair_axis=A), "axes"), (dict(axes=3), "each pair's axis"), (dict(stride=767), "row stride"),
    (dict(stride=760), "row stride"), (dict(gated=True), "row stride"), (dict(big=A + 8), "16 bytes"), (dict(Vp=A + 2), "16 bytes"),
    (dict(rope=A + 4), "8 bytes"), (dict(page_stride=4088), "page stride"), (dict(page_stride=4100), "page stride"),
    (dict(page_size=8), "power of two"), (dict(n_pages=-1), "at least one page"), (dict(Q=A + 6128), "Q overlaps big"),
    (dict(T=1 << 28, HQ=1, HD=64, stride=192, Q=1 << 50), "too many rows"),
])
def test_prep_refuses(sdamd, kw, message):
    with pytest.raises(sdamd.EngineError, match="sd_op_paged_prep: .*" + message):
        prep(sdamd, **kw)


@pytest.mark.parametrize("kw,message", [
    (dict(Q=None), "null argument"), (dict(out=None), "null argument"), (dict(cu=None), "null argument"),
    (dict(B=0), "requests"), (dict(B=8193), "requests"), (dict(T=0), "at least one row"), (dict(T=1 << 29), "2\\^30"),
    (dict(max_new=0), "max_new"), (dict(max_kv=0), "max_new"), (dict(max_kv=257), "more than a table row"),
    (dict(max_blocks=0), "table row"), (dict(max_blocks=1 << 26), "table row"), (dict(window=-1), "window"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(big=A, stride=1016), "gates' row stride"), (dict(big=A, stride=1028), "gates' row stride"), (dict(Q=A + 8), "16 bytes"),
    (dict(Kp=A + 8), "16 bytes"), (dict(out=A + 65537), "16 bytes"), (dict(table=A + 2), "4 bytes"), (dict(out=A), "out overlaps Q"),
    (dict(out=A + 4080), "out overlaps Q"), (dict(big=A + 65536 - 4096, stride=1024), "out overlaps the gates"),
    (dict(HD=80), "head_dim"), (dict(HQ=5, HK=2), "multiple of kv heads"), (dict(type=3), "type"), (dict(page_size=33), "power of two"),
    (dict(page_stride=8), "page stride"),
    (dict(B=1, T=1, max_new=1, max_blocks=4000, max_kv=100000, ws=A + 65536), "workspace overlaps"),
    (dict(B=1, T=1, max_new=1, max_blocks=4000, max_kv=100000, ws=A), "workspace overlaps"),
    (dict(B=8192, T=1 << 19, max_new=1 << 19, HQ=1024, HK=1024, HD=64, out=1 << 50), "too many rows"),
])
def test_attention_refuses(sdamd, kw, message):
    with pytest.raises(sdamd.EngineError, match="sd_op_paged_attention: .*" + message):
        attn(sdamd, **kw)


def test_workspace_sizes(sdamd):
    """A size for every allowed call, refusals as the call's own."""
    for B, T, new, kv in [(1, 1, 1, 1), (64, 64, 1, 8192), (1, 1, 1, 2 ** 31 - 1), (8192, 8192, 1, 100), (2, 4096, 4096, 4096)]:
        for hq, hk, hd in [(8, 2, 256), (32, 8, 128), (12, 1, 64)]:
            assert 0 <= sdamd.paged_attention_ws(B, T, new, kv, hq, hk, hd) < 1 << 40
    for bad in [(0, 1, 1, 1, 8, 2, 256), (1, 0, 1, 1, 8, 2, 256), (1, 1, 0, 1, 8, 2, 256), (1, 1, 1, 0, 8, 2, 256),
                (1, 1, 1, 1, 7, 2, 256), (1, 1, 1, 1, 8, 2, 100)]:
        with pytest.raises(sdamd.EngineError, match="sd_op_paged_attention_ws: "):
            sdamd.paged_attention_ws(*bad)


def test_attention_refuses_a_small_workspace(sdamd):
    need = sdamd.paged_attention_ws(1, 1, 1, 100000, 8, 2, 256)
    if need:
        for ws, n in ((A, need - 1), (None, need), (A, 0)):
            with pytest.raises(sdamd.EngineError, match="workspace"):
                attn(sdamd, B=1, T=1, max_new=1, max_blocks=4000, max_kv=100000, HQ=8, HK=2, HD=256, ws=ws, ws_bytes=n)


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_attention_refuses_a_scale_past_its_range(sdamd, scale):
    """A scale that is finite, but not in base 2 (times log2 e): 0 times it would not be 0."""
    with pytest.raises(sdamd.EngineError, match="sd_op_paged_attention: .*scale"):
        attn(sdamd, scale=scale)
