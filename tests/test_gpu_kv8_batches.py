"""The 8-bit cache over batch sizes: the searches that place a call's blocks and steps
change with the number of sequences, and their arithmetic with the heads of a block.

Write and read are compared bit for bit with the definition on the host, attention
within the bounds worked out in test_gpu_kv8.py."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_kv8 import B, Model, Pool, attend, check_attention, equal, filled, gen, rows_of  # noqa: E402


def check_rows(pool, model, lens):
    got = pool.read([0] * len(lens), lens)
    off = 0
    for i, n in enumerate(lens):
        if n:
            want = model.values(i, 0, n)
            equal(got[0][off:off + n], want[0])
            equal(got[1][off:off + n], want[1])
        off += n


@pytest.mark.parametrize("kv,dim", [(3, 64), (5, 128), (3, 256), (7, 64), (1, 256)])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 64, 65, 100, 128, 129, 300])
def test_writes_of_many_sequences(qcache, n, kv, dim):
    """Chunks of ragged lengths, many empty, that go on inside blocks which keep older
    tokens, then a token for each; the heads of a block fall on different CTAs."""
    r, g = np.random.default_rng(n + kv), gen(n + kv)
    pool, model, at = Pool(qcache, n, 2, kv, dim, seed=n), Model(n, kv, dim), [0] * n
    for std, most in ((1.0, 40), (3.0, 20), (0.3, None), (6.0, 30)):
        counts = [1] * n if most is None else [int(c) if r.random() < 0.6 else 0 for c in r.integers(1, most, n)]
        if sum(counts) == 0:
            counts[-1] = 5
        k, v = rows_of(g, sum(counts), kv, dim, std), rows_of(g, sum(counts), kv, dim, std)
        pool.write(at, None if most is None else counts, k, v)
        off = 0
        for i, c in enumerate(counts):
            if c:
                model.write(i, at[i], k[off:off + c], v[off:off + c])
            off, at[i] = off + c, at[i] + c
    check_rows(pool, model, at)
    qcache.kv8_check()


def test_write_of_the_most_sequences(qcache):
    """1024 sequences, each going on inside a block of three heads."""
    n, kv, dim, g = 1024, 3, 64, gen(9)
    pool, model = Pool(qcache, n, 1, kv, dim, seed=2), Model(n, kv, dim)
    first = [(7 * i) % B for i in range(n)]
    then = [(5 * i + 3) % 21 for i in range(n)]
    at = [0] * n
    for counts in (first, then):
        k, v = rows_of(g, sum(counts), kv, dim), rows_of(g, sum(counts), kv, dim)
        pool.write(at, counts, k, v)
        off = 0
        for i, c in enumerate(counts):
            if c:
                model.write(i, at[i], k[off:off + c], v[off:off + c])
            off, at[i] = off + c, at[i] + c
    check_rows(pool, model, at)
    qcache.kv8_check()


@pytest.mark.parametrize("n,kv,group,dim", [(300, 5, 2, 128), (330, 4, 4, 256), (200, 8, 8, 128), (400, 3, 5, 256), (600, 4, 1, 64),
                                            (31, 2, 3, 128), (32, 3, 4, 64), (33, 1, 6, 256), (128, 2, 8, 64), (129, 4, 2, 256)])
def test_attention_of_many_sequences(qcache, n, kv, group, dim):
    """Ragged lengths with empty ones among them and at both ends; also more pairs of
    sequence and head than warps."""
    r = np.random.default_rng(n)
    lens = [int(x) if r.random() < 0.8 else 0 for x in np.exp(r.uniform(0, np.log(700), n))]
    lens[0] = lens[-1] = 0
    lens[1] = 640
    pool, kvs, g = filled(qcache, lens, kv, dim, seed=n, fill=0xFF)
    qg = rows_of(g, n, kv * group, 2 * dim, 1.5)
    q, gate = qg[:, :, :dim], qg[:, :, dim:]
    got = attend(qcache, pool.cache, pool.table, lens, q, gate)
    check_attention(got, q, gate, kvs, dim ** -0.5)
    again = attend(qcache, pool.cache, pool.table, lens, q, gate)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    qcache.kv8_check()


def test_attention_of_empty_batches(qcache):
    """No sequence has a token: zeros, and nothing to merge."""
    for n in (1, 32, 33, 500):
        pool = Pool(qcache, n, 1, 2, 128, fill=0xFF)
        q = rows_of(gen(n), n, 8, 128)
        assert bool((attend(qcache, pool.cache, pool.table, [0] * n, q) == 0).all())
    qcache.kv8_check()


@pytest.mark.parametrize("seed", range(40))
def test_attention_of_drawn_shapes(qcache, seed):
    """Shapes drawn from the whole range: from one long context to many short ones."""
    r = np.random.default_rng(1000 + seed)
    dim, kv, group = int(r.choice([64, 128, 256])), int(r.choice([1, 2, 3, 4, 8])), int(r.integers(1, 9))
    n = int(np.exp(r.uniform(0, np.log(160))))
    most = max(1, int(np.exp(r.uniform(0, np.log(40000 * 512 / (n * kv * dim) + 2)))))
    lens = [int(x) for x in r.integers(0 if r.random() < 0.5 else most, most + 1, n)]
    pool, kvs, g = filled(qcache, lens, kv, dim, seed=seed, fill=0xFF)
    q = rows_of(g, n, kv * group, dim, float(r.choice([0.1, 1.0, 4.0])))
    check_attention(attend(qcache, pool.cache, pool.table, lens, q), q, None, kvs, dim ** -0.5)
    qcache.kv8_check()
