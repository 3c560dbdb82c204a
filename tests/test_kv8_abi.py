"""CPU tests of include/qrope.h and include/qkv8.h: the frequencies that
qc_rope_init works out, sizes, and the calls that are refused before anything
reaches a GPU (an argument is checked before the first device pointer is)."""
import ctypes as C
import math

import numpy as np
import pytest


def refused(qcache, fn, text):
    with pytest.raises(qcache.QCacheError) as e:
        fn()
    assert e.value.code == qcache.QC_ERR_ARG, str(e.value)
    assert text in str(e.value), str(e.value)


# ------------------------------------------------------------------- rope

@pytest.mark.parametrize("rot,base", [(2, 10.0), (24, 1e4), (64, 1e7), (256, 5e5)])
def test_frequencies(qcache, rot, base):
    i = np.arange(rot // 2)
    w = np.array([math.pow(base, -2 * k / rot) for k in i])

    def freq(**kw):
        r = qcache.Rope(rot, base=base, **kw)
        assert r.freq.rot_dim == rot
        return np.array(r.freq.inv_freq[: rot // 2]), r.freq.mscale

    # pow and a few products in IEEE double: a few units in the last place
    close = dict(rtol=1e-14, atol=0)
    f, m = freq()
    np.testing.assert_allclose(f, w, **close)
    assert m == 1.0
    f, m = freq(scaling=qcache.ROPE_LINEAR, factor=4.0)
    np.testing.assert_allclose(f, w / 4, **close)
    assert m == 1.0
    if rot > 2:
        f, m = freq(scaling=qcache.ROPE_NTK, factor=4.0)
        b = base * 4.0 ** (rot / (rot - 2))
        np.testing.assert_allclose(f, [math.pow(b, -2 * k / rot) for k in i], rtol=1e-13)
    f, m = freq(scaling=qcache.ROPE_YARN, factor=4.0, orig_ctx=32768)
    assert m == pytest.approx(0.1 * math.log(4.0) + 1.0, rel=1e-15)
    # pairs that turn often keep their frequency, those that hardly turn are divided
    turns = w * 32768 / (2 * math.pi)
    np.testing.assert_allclose(f[turns > 32 * base ** (2 / rot)], w[turns > 32 * base ** (2 / rot)], **close)
    np.testing.assert_allclose(f[turns < base ** (-2 / rot)], w[turns < base ** (-2 / rot)] / 4, **close)
    assert np.all(f <= w * (1 + 1e-14)) and np.all(f >= w / 4 * (1 - 1e-14))
    assert freq(scaling=qcache.ROPE_YARN, factor=1.0, orig_ctx=32768)[1] == 1.0
    assert freq(mscale=0.5)[1] == 0.5


def test_rope_init_refuses(qcache):
    r = lambda text, rot=64, **kw: refused(qcache, lambda: qcache.Rope(rot, **kw), text)  # noqa: E731
    for rot in (0, 1, 63, -2, 258):
        r("rot_dim", rot)
    r("layout", layout=2)
    r("scaling", scaling=4)
    for base in (1.0, 0.0, -5.0, math.inf, math.nan):
        r("base", base=base)
    for f in (0.0, -1.0, math.nan, math.inf):
        r("factor", scaling=qcache.ROPE_LINEAR, factor=f)
    r("NTK", rot=2, scaling=qcache.ROPE_NTK, factor=2.0)
    r("YARN", scaling=qcache.ROPE_YARN, factor=2.0, orig_ctx=0)
    r("YARN", scaling=qcache.ROPE_YARN, factor=2.0, orig_ctx=10, beta_slow=-1.0)
    r("mscale", mscale=-1.0)
    r("infinite", scaling=qcache.ROPE_LINEAR, factor=1e-320)
    assert qcache.lib().qc_rope_init(None, None) == qcache.QC_ERR_ARG


def test_rope_apply_refuses(qcache):
    rope = qcache.Rope(64)
    good = dict(x=16, out=16, n_heads=4, x_ld=1024, x_head=256, out_ld=1024, out_head=256)

    def call(text, dim=256, rows=1, parts=None, eps=1e-6, pos=16, **kw):
        ps = parts if parts is not None else [qcache.RopePart(**{**good, **kw})]
        refused(qcache, lambda: rope.apply(dim, pos, rows, ps, eps), text)

    for dim in (0, 60, 62, 264, -8):
        call("head_dim", dim=dim)
    call("head_dim", dim=56)                    # fewer dims than are rotated
    call("n_rows", rows=-1)
    call("n_parts", parts=[])
    call("n_parts", parts=[qcache.RopePart(**good)] * 5)
    call("eps", eps=-1.0)
    call("eps", eps=math.nan)
    call("n_heads", n_heads=0)
    call("n_heads", n_heads=16385)
    for s in ("x_ld", "x_head", "out_ld", "out_head"):
        call("multiples of 8", **{s: 1020})
    for s in ("x", "out", "norm_w"):
        call("aligned", **{s: 24})
    call("pos_dev is null", pos=0)
    rope.apply(256, 0, 0, [qcache.RopePart(**good)])   # no rows: nothing to do
    bad = qcache.Rope(64)
    bad.freq.rot_dim = 63
    refused(qcache, lambda: bad.apply(256, 16, 1, [qcache.RopePart(**good)]), "qc_rope_init")


# -------------------------------------------------------------------- kv8

def test_page_bytes(qcache):
    for kv in (1, 4, 256):
        for dim in (64, 128, 256):
            # per block of 16 tokens: 16 bytes of scales, K and V codes
            assert qcache.kv8_page_bytes(kv, dim) == kv * 4 * (16 + 2 * 16 * dim)
    for kv, dim in ((0, 64), (-1, 64), (257, 64), (4, 0), (4, 32), (4, 96), (4, 512)):
        assert qcache.kv8_page_bytes(kv, dim) == 0


@pytest.mark.parametrize("name", ["write", "read"])
def test_rows_refuse(qcache, name):
    def call(text, kv=4, dim=256, pages=8, pool=16, table=16, stride=4, pos=16, start=16, n=2, rows=3, k=16,
             k_ld=1024, v=16, v_ld=1024):
        c = qcache.Kv8Cache(pool, pages, kv, dim)
        refused(qcache, lambda: getattr(c, name)(table, stride, pos, start, n, rows, k, k_ld, v, v_ld), text)

    call("KV heads", kv=0)
    call("KV heads", dim=96)
    call("n_pages", pages=0)
    call("pool is not 16-byte", pool=24)
    call("the pool is null", pool=0)
    call("n_rows", rows=-1)
    call("without row_start", start=0)
    call("row strides", k_ld=1016)
    call("row strides", v_ld=1028)
    call("aligned", k=8)
    call("aligned", v=2)
    call("sequences", n=-1)
    call("sequences", n=1025)
    call("pt_stride", stride=0)
    c = qcache.Kv8Cache(16, 8, 4, 256)
    getattr(c, name)(16, 4, 16, 16, 0, 0, 16, 1024, 16, 1024)     # no sequences: nothing to do


def test_attention_refuses(qcache):
    def call(text, kv=4, dim=256, pages=8, pool=16, table=16, stride=4, ln=16, n=2, heads=16, q=16, q_ld=8192,
             q_head=512, gate=0, out=16, out_ld=4096, ws=16, ws_bytes=1 << 30):
        c = qcache.Kv8Cache(pool, pages, kv, dim)
        refused(qcache, lambda: c.attn_decode(table, stride, ln, n, heads, q, q_ld, q_head, gate, 0.0625, out, out_ld,
                                              ws, ws_bytes), text)

    call("KV heads", kv=0, heads=4)
    call("query heads", heads=15)
    call("query heads", heads=0)
    call("query heads", heads=36)
    call("multiples of 8", q_ld=8190)
    call("multiples of 8", q_head=511)
    call("multiples of 8", out_ld=4100)
    call("out_ld", out_ld=4088)
    for a in ("q", "gate", "out", "ws"):
        call("aligned", **{a: 24})
    call("sequences", n=1025)
    call("pt_stride", stride=0)
    call("the pool is null", pool=0)
    c = qcache.Kv8Cache(16, 8, 4, 256)
    assert c.attn_workspace_bytes(2, 15) == 0 and c.attn_workspace_bytes(1025, 16) == 0
    assert qcache.Kv8Cache(16, 8, 4, 96).attn_workspace_bytes(2, 16) == 0
    assert c.attn_workspace_bytes(64, 16) >= c.attn_workspace_bytes(1, 16) > 0
    c.attn_decode(16, 4, 16, 0, 16, 16, 8192, 512, 0, 0.0625, 16, 4096, 16, 1 << 30)   # nothing to do


def test_descriptions_match_the_header(qcache):
    """The ctypes layouts are those of the C structs."""
    assert C.sizeof(qcache.RopeConfig) == 4 * 4 + 5 * 8
    assert C.sizeof(qcache.RopeFrequencies) == 8 + 8 + 128 * 8
    assert C.sizeof(qcache.RopePart) == 8 * 8
    assert C.sizeof(qcache.Kv8Desc) == 8 + 4 * 4
