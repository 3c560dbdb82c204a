"""qc_rope_apply's norm over the whole range of bf16, against the formula in 64 bits.

The tolerance is the one worked out in test_gpu_rope.py: the power of two by which
a head's values are brought into range is exact, and what it makes subnormal is
2^-126 of the head's largest and less.
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_rope import check, positions  # noqa: E402


def reference(x, pos, freq, rot, half, w, eps):
    """(result, |y1| + |y2| per element) in 64 bits."""
    y = x.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    a = pos.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = torch.cos(a), torch.sin(a)
    i = torch.arange(rot // 2, device=x.device)
    p, q = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
    out, mag = y.clone(), y.abs()
    out[..., p] = y[..., p] * c - y[..., q] * s
    out[..., q] = y[..., q] * c + y[..., p] * s
    mag[..., p] = mag[..., q] = y[..., p].abs() + y[..., q].abs()
    return out, mag


def apply(qcache, rope, x, pos, w, eps):
    rows, heads, dim = x.shape
    out = torch.empty_like(x)
    part = qcache.RopePart(x.data_ptr(), out.data_ptr(), heads, heads * dim, dim, heads * dim, dim, w.data_ptr())
    rope.apply(dim, pos.data_ptr(), rows, [part], eps)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("dim,rot", [(256, 64), (128, 128), (64, 64), (40, 38), (96, 24), (8, 2)])
@pytest.mark.parametrize("power,eps", [(0, 1e-6), (62, 1e-6), (64, 1e-6), (90, 0.0), (126, 1e-6), (-40, 0.0), (-60, 0.0),
                                       (-70, 1e-30), (-100, 1e-38), (-125, 0.0), (-131, 0.0), (-50, 1e-30)])
def test_norm_of_very_large_and_small_heads(qcache, dim, rot, half, power, eps):
    """Heads whose squares leave f32 beside ordinary ones, which keep their bits."""
    g = torch.Generator(device="cuda")
    g.manual_seed(dim + power + 200)
    rows, heads = 21, 5
    x = torch.randn(rows, heads, dim, generator=g, device="cuda").bfloat16()
    x[0, 0, 1:] *= 2.0 ** -30                 # one dim far above the others of its head
    odd = torch.rand(rows, heads, generator=g, device="cuda") < 0.5
    odd[0, 0] = True
    plain = x.clone()
    x[odd] = (x[odd].double() * 2.0 ** power).clamp(-3e38, 3e38).bfloat16()
    x[odd & (x == 0).all(-1)] = 2.0 ** -133
    w = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda")
    pos = positions(rows, 7)
    rope = qcache.Rope(rot, layout=qcache.ROPE_HALF if half else qcache.ROPE_INTERLEAVED, base=1e4)
    out = apply(qcache, rope, x, pos, w, eps)
    check(out, *reference(x, pos, list(rope.freq.inv_freq[: rot // 2]), rot, half, w, eps))
    beside = apply(qcache, rope, plain, pos, w, eps)
    assert torch.equal(out[~odd].view(torch.int16), beside[~odd].view(torch.int16))


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("dim,rot,at", [(64, 32, 5), (64, 32, 21), (64, 32, 50), (256, 64, 255), (40, 38, 3), (40, 38, 39)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_values_through_the_norm(qcache, bad, dim, rot, at, half):
    """A NaN takes its whole head; an infinity is NaN in its pair and 0 elsewhere; the
    other heads keep their bits."""
    g = torch.Generator(device="cuda")
    g.manual_seed(dim + at)
    x = torch.randn(2, 3, dim, generator=g, device="cuda").bfloat16()
    pos = torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    w = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda")
    rope = qcache.Rope(rot, layout=qcache.ROPE_HALF if half else qcache.ROPE_INTERLEAVED)
    clean = apply(qcache, rope, x, pos, w, 1e-6)
    x[1, 1, at] = bad
    got = apply(qcache, rope, x, pos, w, 1e-6)
    pair = {at} if at >= rot else {at, (at + rot // 2) % rot if half else at ^ 1}
    for d in range(dim):
        y = float(got[1, 1, d])
        if bad != bad or d in pair:
            assert y != y, (d, y)
        else:
            assert y == 0, (d, y)
    got[1, 1] = clean[1, 1]
    assert torch.equal(got.view(torch.int16), clean.view(torch.int16))
