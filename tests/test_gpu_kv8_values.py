"""The 8-bit cache's attention where its arithmetic is tight: weights that cancel,
whatever the number of query heads to a KV head.

The results are compared with the softmax in 64 bits over the values read back.
Tolerance per element, worked out before the first run, with A = sum p |v|, S =
scale * sum |q_d k_d| at its largest over the tokens, N = len / 16 blocks:
  - the bf16 result rounds once: 2^-8 |y| (half a step);
  - a query value is exact in f16 if it is 2^-30 of its head's largest or more, else off
    by at most 2^-38 of that;
  - a weight w enters the second product as two f16, w and the rest: the rest is at
    most 2^-11 w and off by at most 2^-11 of itself, 2^-22 w;
  - f32 sums of D products of q and k: (D + 8) 2^-23 S on a score, so as much on
    the weight; the exponential and its argument 8 * 2^-23 (1 + S);
  - f32 sums over N + 16 blocks' weights and products: (N + 16) 2^-23 A, twice
    (numerator and denominator);
  - f16 ends at 2^-24, so a weight is off by up to 2^-25 however small it is, while
    the largest is 2^7 or more: len 2^-31 max_j(p_j u_j), u_j the largest |v| of token
    j's block.
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_kv8 import Pool, attend, gen, rows_of  # noqa: E402


def check(got, q, k, v, scale, off=0.0):
    """One sequence's rows got [heads][dim] against 64 bits over k, v [len][kv][dim];
    off: what a score may be off by besides."""
    heads, dim = q.shape
    kv = k.shape[1]
    qi = q.double().unflatten(0, (kv, heads // kv))
    kk, vv = k.double().permute(1, 2, 0), v.double().transpose(0, 1)
    p = torch.softmax(qi @ kk * scale, -1)
    y, a = p @ vv, p @ vv.abs()
    s = (qi.abs() @ kk.abs() * abs(scale)).amax(-1, keepdim=True)
    n = len(k) / 16
    f = 2.0 ** -22 + 2 * off + (dim + 8) * 2.0 ** -23 * s + 8 * 2.0 ** -23 * (1 + s)
    u = torch.cat([b.abs().amax((1, 2), keepdim=True).expand(-1, b.shape[1], 1) for b in vv.split(16, 1)], 1)
    tol = a * (f + 2 * (n + 16) * 2.0 ** -23) + len(k) * 2.0 ** -31 * (p * u.transpose(1, 2)).amax(-1, keepdim=True)
    tol = tol + (y.abs() + tol) * 2.0 ** -8 + 1e-38
    err = (got.double().unflatten(0, (kv, heads // kv)) - y).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("kv,group,dim", [(2, 1, 64), (1, 4, 256), (3, 5, 128), (2, 6, 128), (1, 6, 256), (1, 7, 64), (2, 8, 64),
                                          (1, 8, 256)])
def test_weights_that_cancel(qcache, kv, group, dim):
    """Values of opposite sign under nearly equal weights: what is left of them is
    far below the sum of their magnitudes, so that weights of 11 bits would show."""
    g = gen(100 * group + dim)
    lens = [2, 3, 17, 40, 301, 5000]
    pool = Pool(qcache, len(lens), 79, kv, dim)
    sign = [torch.tensor([(-1.0) ** j for j in range(n)], device="cuda")[:, None, None] for n in lens]
    v = torch.cat([s * torch.randn(1, kv, dim, generator=g, device="cuda") for s in sign]).bfloat16()
    k = rows_of(g, sum(lens), kv, dim)
    q = rows_of(g, len(lens), kv * group, dim, 0.02)
    pool.write([0] * len(lens), lens, k, v)
    k, v = pool.read([0] * len(lens), lens)
    got = attend(qcache, pool.cache, pool.table, lens, q)
    for i, (ki, vi) in enumerate(zip(k.split(lens), v.split(lens))):
        check(got[i], q[i], ki, vi, dim ** -0.5)
    qcache.kv8_check()


@pytest.mark.parametrize("a,b,c", [(0, 0, 0), (120, -118, -2), (115, -119, 4), (122, -120, 2), (124, -122, 2), (-126, 124, 2), (-120, 118, 2), (-60, -60, 120),
                                   (100, 30, -126), (30, 100, -127), (-110, -10, 120)])
@pytest.mark.parametrize("group,dim", [(4, 256), (8, 128), (2, 64)])
def test_moderate_scores_of_extreme_factors(qcache, group, dim, a, b, c):
    """Queries near 2^a, keys near 2^b and a scale near 2^c whose product is moderate:
    no step on the way to a score leaves f32, whichever of them is large."""
    g = gen(200 + a)
    lens = [1, 20, 700]
    pool = Pool(qcache, 3, 11, 2, dim)
    k, v = (rows_of(g, sum(lens), 2, dim).double() * 2.0 ** b).bfloat16(), rows_of(g, sum(lens), 2, dim)
    q = (rows_of(g, 3, 2 * group, dim).double() * 2.0 ** a).bfloat16()
    scale = dim ** -0.5 * 2.0 ** c
    pool.write([0] * 3, lens, k, v)
    k, v = pool.read([0] * 3, lens)
    got = attend(qcache, pool.cache, pool.table, lens, q, scale=scale)
    for i, (ki, vi) in enumerate(zip(k.split(lens), v.split(lens))):
        check(got[i], q[i], ki, vi, scale)
    qcache.kv8_check()


@pytest.mark.parametrize("r", [0, 16, 24, 27, 34])
@pytest.mark.parametrize("group,dim", [(4, 256), (6, 128), (1, 64)])
def test_query_values_far_below_their_largest(qcache, group, dim, r):
    """One large query value over keys that are 0 there; the others, 2^-r of it, make
    the scores.  Down to 2^-30 they count in full."""
    g = gen(300 + r)
    lens = [2, 50, 700]
    pool = Pool(qcache, 3, 11, 2, dim)
    k, v = rows_of(g, sum(lens), 2, dim), rows_of(g, sum(lens), 2, dim)
    k[:, :, 3] = 0
    q = (rows_of(g, 3, 2 * group, dim).abs().clamp(0.125, 4) * 2.0 ** -r).bfloat16()
    q = torch.where(torch.rand(q.shape, generator=g, device="cuda") < 0.5, q, -q)
    q[:, :, 3] = 1
    scale = dim ** -0.5 * 2.0 ** r
    pool.write([0] * 3, lens, k, v)
    k, v = pool.read([0] * 3, lens)
    got = attend(qcache, pool.cache, pool.table, lens, q, scale=scale)
    for i, (ki, vi) in enumerate(zip(k.split(lens), v.split(lens))):
        off = float(ki.double().abs().sum(-1).max()) * scale * 2.0 ** -38 if r > 27 else 0.0
        check(got[i], q[i], ki, vi, scale, off)
    qcache.kv8_check()
