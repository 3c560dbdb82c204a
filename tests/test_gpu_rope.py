"""qc_rope_apply (include/qrope.h) against the formula in 64 bits.

Tolerance, per element, worked out before the first run.  The result rounds to
bf16 once: at most 2^-8 of its value (half a step).  In front of that stand f32
operations on y1, y2 (the pair) with cosine and sine: the angle in turns rounds
to f32 once (2^-25 of half a turn, pi 2^-24 in radians), sincospif is within 2
units of 2^-23, the products, the sum and mscale round to 2^-24 each: together
under 16 * 2^-24 (|y1| + |y2|) mscale.  The norm adds a sum of up to 256 squares
(8 in a lane, then a tree of 5), a division, a root and two products: its
relative error is under 24 * 2^-24, on both terms.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

EPS = 1e-6


def reference(x, pos, freq, mscale, rot, half, w):
    """(result, |y1| + |y2| per element) in 64 bits."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
    a = pos.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = torch.cos(a), torch.sin(a)
    i = torch.arange(rot // 2, device=x.device)
    p, q = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
    out, mag = y.clone(), y.abs()
    out[..., p] = mscale * (y[..., p] * c - y[..., q] * s)
    out[..., q] = mscale * (y[..., q] * c + y[..., p] * s)
    mag[..., p] = mag[..., q] = mscale * (y[..., p].abs() + y[..., q].abs())
    return out, mag


def check(got, ref, mag):
    err = (got.double() - ref).abs()
    tol = ref.abs() * 2.0 ** -8 + 40 * 2.0 ** -24 * mag + 1e-38
    assert bool((err <= tol).all()), float((err - tol).max())


def positions(rows, seed):
    r = np.random.default_rng(seed)
    p = np.concatenate([[0, 1, 2, 131071, 1 << 20, 2 ** 31 - 1, -1, -77777], r.integers(0, 1 << 20, rows)])[:rows]
    return torch.from_numpy(p.astype(np.int32)).cuda()


def parts_of(qcache, q, k, qo, ko, qw, kw):
    ptr = lambda t: t.data_ptr() if t is not None else 0  # noqa: E731
    return [qcache.RopePart(x.data_ptr(), o.data_ptr(), x.shape[1], x.stride(0), x.stride(1), o.stride(0), o.stride(1), ptr(w))
            for x, o, w in ((q, qo, qw), (k, ko, kw))]


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dim,rot,nq,nk,rows", [
    (256, 64, 16, 4, 9), (256, 256, 3, 1, 33), (128, 128, 32, 8, 5), (64, 64, 5, 5, 200), (64, 16, 7, 1, 1),
    (128, 24, 9, 3, 17), (96, 96, 6, 2, 11), (8, 2, 1, 1, 3), (40, 38, 2, 70, 4), (256, 254, 1, 1, 65), (256, 64, 16, 4, 3001),
    (64, 64, 16, 16, 20000), (8, 8, 16384, 16384, 1),
])
def test_matches_64_bits(qcache, dim, rot, nq, nk, rows, norm, half):
    g = torch.Generator(device="cuda")
    g.manual_seed(dim * rows + rot)
    q = torch.randn(rows, nq, dim, generator=g, device="cuda").bfloat16()
    k = torch.randn(rows, nk, dim, generator=g, device="cuda").bfloat16()
    qw = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda") if norm else None
    kw = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda") if norm else None
    pos = positions(rows, rows)
    rope = qcache.Rope(rot, layout=qcache.ROPE_HALF if half else qcache.ROPE_INTERLEAVED, base=1e7,
                       scaling=qcache.ROPE_YARN, factor=4.0, orig_ctx=32768)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    rope.apply(dim, pos.data_ptr(), rows, parts_of(qcache, q, k, qo, ko, qw, kw), EPS)
    freq, m = list(rope.freq.inv_freq[: rot // 2]), rope.freq.mscale
    torch.cuda.synchronize()
    check(qo, *reference(q, pos, freq, m, rot, half, qw))
    check(ko, *reference(k, pos, freq, m, rot, half, kw))


def test_projection_rows_in_place_and_untouched_neighbours(qcache):
    """The model's rows [16][q | gate], k, v: q and k rotate in place, gate, v
    and the padding behind a row keep their bits."""
    rows, ld = 37, 10240 + 24
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    proj = torch.randn(rows, ld, generator=g, device="cuda").bfloat16()
    before = proj.clone()
    q = proj[:, :8192].unflatten(1, (16, 512))[:, :, :256]
    k = proj[:, 8192:9216].unflatten(1, (4, 256))
    qw = 1 + 0.02 * torch.randn(256, generator=g, device="cuda")
    kw = 1 + 0.02 * torch.randn(256, generator=g, device="cuda")
    pos = positions(rows, 1)
    rope = qcache.Rope(64)
    rope.apply(256, pos.data_ptr(), rows, parts_of(qcache, q, k, q, k, qw, kw), EPS)
    torch.cuda.synchronize()
    f = list(rope.freq.inv_freq[:32])
    b = before[:, :8192].unflatten(1, (16, 512))
    check(q, *reference(b[:, :, :256], pos, f, 1.0, 64, True, qw))
    check(k, *reference(before[:, 8192:9216].unflatten(1, (4, 256)), pos, f, 1.0, 64, True, kw))
    assert torch.equal(proj[:, :8192].unflatten(1, (16, 512))[:, :, 256:].view(torch.int16), b[:, :, 256:].view(torch.int16))
    assert torch.equal(proj[:, 9216:].view(torch.int16), before[:, 9216:].view(torch.int16))


def test_four_parts_with_and_without_norm(qcache):
    """Parts of different sizes in one launch; one reads a single row's heads
    out of order (a negative head stride)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    rows, dim, heads = 70, 128, [3, 1, 17, 6]
    pos = positions(rows, 2)
    rope = qcache.Rope(128, layout=qcache.ROPE_INTERLEAVED, base=1e4, scaling=qcache.ROPE_NTK, factor=8.0)
    f = list(rope.freq.inv_freq[:64])
    xs = [torch.randn(rows, h, dim, generator=g, device="cuda").bfloat16() for h in heads]
    outs = [torch.empty_like(x) for x in xs]
    ws = [1 + 0.1 * torch.randn(dim, generator=g, device="cuda"), None, None, torch.ones(dim, device="cuda")]
    parts = [qcache.RopePart(x.data_ptr(), o.data_ptr(), h, x.stride(0), dim, o.stride(0), dim, w.data_ptr() if w is not None else 0)
             for x, o, h, w in zip(xs, outs, heads, ws)]
    parts[3].x, parts[3].x_head = xs[3].data_ptr() + 2 * 5 * dim, -dim
    rope.apply(dim, pos.data_ptr(), rows, parts, EPS)
    torch.cuda.synchronize()
    xs[3] = xs[3].flip(1)
    for x, o, w in zip(xs, outs, ws):
        check(o, *reference(x, pos, f, 1.0, 128, False, w))


def test_position_zero_without_norm_keeps_the_bits(qcache):
    x = torch.randn(3, 4, 128, device="cuda").bfloat16()
    x[0, 0, :4] = torch.tensor([0.0, -0.0, 1e-40, 3e38])
    o = torch.full_like(x, 7.0)
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    part = qcache.RopePart(x.data_ptr(), o.data_ptr(), 4, x.stride(0), 128, o.stride(0), 128)
    qcache.Rope(64, layout=qcache.ROPE_INTERLEAVED).apply(128, pos.data_ptr(), 3, [part])
    torch.cuda.synchronize()
    assert torch.equal(o, x)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("norm", [True, False])
def test_non_finite_values_stay_in_their_head(qcache, bad, norm):
    x = torch.randn(2, 3, 64, device="cuda").bfloat16()
    x[1, 1, 5] = bad
    w = torch.ones(64, device="cuda")
    o = torch.empty_like(x)
    pos = torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    part = qcache.RopePart(x.data_ptr(), o.data_ptr(), 3, 192, 64, 192, 64, w.data_ptr() if norm else 0)
    qcache.Rope(32).apply(64, pos.data_ptr(), 2, [part])
    torch.cuda.synchronize()
    odd = ~torch.isfinite(o)
    assert odd[1, 1].any()
    touched = torch.zeros_like(odd)
    if norm:
        touched[1, 1] = True
    else:
        touched[1, 1, [5, 21]] = True
    assert not (odd & ~touched).any()


def test_zero_row_with_norm_is_zero(qcache):
    x = torch.zeros(1, 1, 256, device="cuda", dtype=torch.bfloat16)
    o = torch.full_like(x, 9.0)
    w = torch.ones(256, device="cuda")
    pos = torch.tensor([1000], dtype=torch.int32, device="cuda")
    qcache.Rope(64).apply(256, pos.data_ptr(), 1, [qcache.RopePart(x.data_ptr(), o.data_ptr(), 1, 256, 256, 256, 256, w.data_ptr())])
    torch.cuda.synchronize()
    assert bool((o == 0).all())


def test_captured_replayed_and_on_a_side_stream(qcache):
    rope = qcache.Rope(64)
    x = torch.randn(8, 4, 256, device="cuda").bfloat16()
    o = torch.empty_like(x)
    pos = torch.arange(8, dtype=torch.int32, device="cuda")
    part = qcache.RopePart(x.data_ptr(), o.data_ptr(), 4, 1024, 256, 1024, 256)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        rope.apply(256, pos.data_ptr(), 8, [part], stream=torch.cuda.current_stream().cuda_stream)
    f = list(rope.freq.inv_freq[:32])
    for step in range(3):
        x.copy_(torch.randn(8, 4, 256, device="cuda").bfloat16())
        pos.add_(1000 * step)
        graph.replay()
        torch.cuda.synchronize()
        check(o, *reference(x, pos, f, 1.0, 64, True, None))


def test_host_memory_is_refused(qcache):
    x = torch.zeros(1, 1, 64, device="cuda", dtype=torch.bfloat16)
    h = torch.zeros(64, dtype=torch.bfloat16).pin_memory()
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    for a, b in ((h.data_ptr(), x.data_ptr()), (x.data_ptr(), h.data_ptr())):
        with pytest.raises(qcache.QCacheError) as e:
            qcache.Rope(64).apply(64, pos.data_ptr(), 1, [qcache.RopePart(a, b, 1, 64, 64, 64, 64)])
        assert e.value.code == qcache.QC_ERR_ARG and "device memory" in str(e.value)
