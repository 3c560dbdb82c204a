"""The 8-bit paged KV cache (include/qkv8.h) against its definition in 64 bits.

Write and read are exact: the codes and scales follow from the rows by a rule
in which every step is exact or a single rounding to nearest even, so the
values read back have to be equal bit for bit.

Attention is compared with the softmax in 64 bits over the values read back.
Tolerance per element, worked out before the first run, with A = sum p |v| (the
sum of weights times magnitudes, p the exact weights), S = scale * sum |q_d k_d|
at its largest over the tokens, and N = len / 16 blocks:
  - the bf16 result rounds once: 2^-8 |y| (half a step);
  - weights and queries enter the matrix products as f16 pairs (value and
    rest, 2^-22 of the value) for groups of up to 4 query heads; for larger
    groups weights as one f16: 2^-11 A (a bf16 query is exact in f16);
  - f32 sums of D products of q and k: (D + 8) 2^-23 S on a score, so as much
    on the weight's exponent; the exponential and its argument 8 * 2^-23 (1 + S);
  - f32 sums over N + 16 blocks' weights and products: (N + 16) 2^-23 A, twice
    (numerator and denominator);
  - f16 ends at 2^-24: a weight w_j = 2^(x_j - r) sv_j (sv_j the block's V scale)
    is off by up to 2^-25 however small it is.  The largest w_j was at least 2^7
    when r was last set, so 2^(r - m) / l <= 2^-7 max_j(p_j sv_j), and the len
    weights' errors on codes of at most 127 come to len 2^-25 127 2^-7
    max_j(p_j sv_j) <= len 2^-31 max_j(p_j u_j), u_j the largest |v| of token j's
    block (127 sv <= 2 u).  It matters only for a dim in which the tokens with
    the weight have code 0.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

B, PAGE = 16, 64


def i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def quantise(x, old_codes=None, old_scale=None):
    """One block's new rows x [rows][D] (f64) behind older codes: (codes, scale)."""
    most = 127.0 * 2.0 ** 120
    x = np.clip(np.nan_to_num(x, nan=0.0, posinf=np.inf, neginf=-np.inf), -most, most)
    amax = np.abs(x).max(initial=0.0)
    scale = 2.0 ** -126
    while 127.0 * scale < amax:
        scale *= 2.0
    kept = np.zeros((0, x.shape[1]))
    if old_codes is not None and len(old_codes):
        scale = max(scale, old_scale)
        kept = np.rint(old_codes * (old_scale / scale))
    return np.concatenate([kept, np.rint(x / scale)]), scale


class Model:
    """The cache by its definition, on the host: per sequence, head and block (codes, scale)."""

    def __init__(self, n, kv, dim):
        self.kv, self.dim = kv, dim
        self.blocks = [[[{} for _ in range(kv)] for _ in range(n)] for _ in "kv"]

    def write(self, i, pos, k, v):
        for w, x in enumerate((k, v)):
            x = x.double().cpu().numpy()
            for h in range(self.kv):
                p, r = pos, 0
                while r < len(x):
                    b, s = divmod(p, B)
                    take = min(B - s, len(x) - r)
                    codes, scale = self.blocks[w][i][h].get(b, (np.zeros((0, self.dim)), 0.0))
                    self.blocks[w][i][h][b] = quantise(x[r:r + take, h], codes[:s], scale)
                    p, r = p + take, r + take

    def values(self, i, lo, hi):
        """[2][hi - lo][kv][dim] in f64."""
        out = np.zeros((2, hi - lo, self.kv, self.dim))
        for w in range(2):
            for h in range(self.kv):
                for p in range(lo, hi):
                    codes, scale = self.blocks[w][i][h][p // B]
                    out[w, p - lo, h] = codes[p % B] * scale
        return out


class Pool:
    """A pool of permuted pages on the device and its cache description."""

    def __init__(self, qcache, n, pages_each, kv, dim, spare=3, fill=0, seed=0):
        self.n, self.kv, self.dim, self.width = n, kv, dim, pages_each
        self.pages = n * pages_each + spare
        self.bytes = qcache.kv8_page_bytes(kv, dim)
        self.pool = torch.full((self.pages * self.bytes,), fill, dtype=torch.uint8, device="cuda")
        self.cache = qcache.Kv8Cache(self.pool.data_ptr(), self.pages, kv, dim)
        ids = np.random.default_rng(seed).permutation(self.pages)[: n * pages_each].reshape(n, pages_each)
        self.ids, self.table = ids, i32(ids)

    def write(self, pos, counts, k, v, stream=0):
        start = i32(np.concatenate([[0], np.cumsum(counts)])) if counts is not None else None
        p = i32(pos)
        self.cache.write(self.table.data_ptr(), self.width, p.data_ptr(), start.data_ptr() if start is not None else 0,
                         len(pos), k.shape[0], k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), stream)
        torch.cuda.synchronize()

    def read(self, pos, counts):
        rows = int(sum(counts))
        k = torch.full((rows, self.kv, self.dim), 7.0, dtype=torch.bfloat16, device="cuda")
        v = torch.full_like(k, 7.0)
        start, p = i32(np.concatenate([[0], np.cumsum(counts)])), i32(pos)
        self.cache.read(self.table.data_ptr(), self.width, p.data_ptr(), start.data_ptr(), len(pos), rows, k.data_ptr(),
                        k.stride(0), v.data_ptr(), v.stride(0))
        torch.cuda.synchronize()
        return k, v


def rows_of(g, rows, kv, dim, std=1.0):
    return (torch.randn(rows, kv, dim, generator=g, device="cuda") * std).bfloat16()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def equal(got, want):
    assert np.array_equal(got.double().cpu().numpy(), want), float(np.abs(got.double().cpu().numpy() - want).max())


# ----------------------------------------------------------- write and read

@pytest.mark.parametrize("kv,dim,pos,counts", [
    (4, 256, [0], [1]), (4, 256, [0], [64]), (4, 256, [0], [130]), (1, 64, [0, 0, 0], [1, 16, 17]),
    (3, 128, [0, 0], [15, 0]), (2, 64, [0, 0, 0, 0, 0], [0, 0, 5, 0, 63]), (8, 128, [0], [200]),
    (2, 256, [0] * 9, [1, 2, 3, 31, 32, 33, 0, 64, 65]),
])
def test_prompt_then_chunk_then_single_tokens(qcache, kv, dim, pos, counts):
    """A first write, a second chunk from wherever it ended, then single tokens
    with growing and shrinking values, each followed by a whole read."""
    g, n = gen(dim + kv), len(pos)
    pool, model = Pool(qcache, n, 6, kv, dim, seed=kv), Model(n, kv, dim)
    at = list(pos)
    chunk = [(7 * i + 3) % 40 for i in range(n)]
    for std, cnt in ((1.0, counts), (2.7, chunk), (0.2, None), (30.0, None), (1e-3, None), (500.0, None)):
        c = cnt if cnt is not None else [1] * n
        k, v = rows_of(g, sum(c), kv, dim, std), rows_of(g, sum(c), kv, dim, 0.3 * std)
        pool.write(at, cnt, k, v)
        off = 0
        for i in range(n):
            model.write(i, at[i], k[off:off + c[i]], v[off:off + c[i]])
            off, at[i] = off + c[i], at[i] + c[i]
        got_k, got_v = pool.read([0] * n, at)
        off = 0
        for i in range(n):
            want = model.values(i, 0, at[i])
            equal(got_k[off:off + at[i]], want[0])
            equal(got_v[off:off + at[i]], want[1])
            off += at[i]
    qcache.kv8_check()


def test_read_of_a_range_and_truncation(qcache):
    """Reads that start and end inside blocks; a write at an earlier position
    drops what stood behind it and keeps the older tokens of its block."""
    g = gen(5)
    pool, model = Pool(qcache, 2, 4, 2, 128), Model(2, 2, 128)
    k, v = rows_of(g, 300, 2, 128), rows_of(g, 300, 2, 128)
    pool.write([0, 0], [200, 100], k, v)
    model.write(0, 0, k[:200], v[:200])
    model.write(1, 0, k[200:], v[200:])
    got = pool.read([37, 99], [101, 1])
    for w in range(2):
        equal(got[w][:101], model.values(0, 37, 138)[w])
        equal(got[w][101:], model.values(1, 99, 100)[w])
    k2, v2 = rows_of(g, 3, 2, 128, 0.1), rows_of(g, 3, 2, 128, 9.0)
    pool.write([59, 64], [2, 1], k2, v2)
    model.write(0, 59, k2[:2], v2[:2])
    model.write(1, 64, k2[2:], v2[2:])
    got = pool.read([0, 0], [61, 65])
    for w in range(2):
        equal(got[w][:61], model.values(0, 0, 61)[w])
        equal(got[w][61:], model.values(1, 0, 65)[w])


def test_special_values(qcache):
    """Zeros, subnormals, the largest bf16, infinities and NaN, in a whole block
    and in one that goes on; every block's own scale."""
    nan, inf, top = math.nan, math.inf, 3.3895314e38
    tiny = 2.0 ** -133                                  # the smallest bf16
    firsts = [[0.0, -0.0], [tiny, -tiny], [2.0 ** -126, tiny], [top, -top], [inf, 1.0], [-inf, nan], [nan, nan],
              [nan, 3.0], [127.0, 126.5], [127.5, -127.0], [128.0, 0.5], [1.9921875, 1.0], [1.984375, 0.0078125],
              [2.0 ** 126, -1.0]]
    n, kv, dim = len(firsts), 1, 64
    for cnt in (16, 3):
        g = gen(cnt)
        pool, model = Pool(qcache, n, 1, kv, dim), Model(n, kv, dim)
        x = torch.zeros(n * cnt, kv, dim, dtype=torch.bfloat16, device="cuda")
        for i, f in enumerate(firsts):
            x[i * cnt + cnt // 2, 0, 5], x[i * cnt, 0, 60] = f[0], f[1]
        pool.write([0] * n, [cnt] * n, x, x.flip(2).contiguous())
        more = rows_of(g, n, kv, dim)
        for i in range(n):
            model.write(i, 0, x[i * cnt:(i + 1) * cnt], x.flip(2)[i * cnt:(i + 1) * cnt])
        got = pool.read([0] * n, [cnt] * n)
        for i in range(n):
            for w in range(2):
                equal(got[w][i * cnt:(i + 1) * cnt], model.values(i, 0, cnt)[w])
        pool.write([cnt] * n, None, more, more)
        for i in range(n):
            model.write(i, cnt, more[i:i + 1], more[i:i + 1])
        got = pool.read([0] * n, [cnt + 1] * n)
        for i in range(n):
            for w in range(2):
                equal(got[w][i * (cnt + 1):(i + 1) * (cnt + 1)], model.values(i, 0, cnt + 1)[w])
        assert all(bool(torch.isfinite(t).all()) for t in got)


def test_rows_inside_projection_rows_and_strides(qcache):
    """k and v as slices of one projection row with a row stride of their own;
    the read writes its rows alone."""
    g = gen(11)
    pool, model = Pool(qcache, 1, 2, 4, 256), Model(1, 4, 256)
    proj = torch.randn(70, 10240 + 8, generator=g, device="cuda").bfloat16()
    k, v = proj[:, 8192:9216].unflatten(1, (4, 256)), proj[:, 9216:10240].unflatten(1, (4, 256))
    pool.write([3 * 0], [70], k, v)
    model.write(0, 0, k, v)
    out = torch.full((70, 2, 5, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    start, pos = i32([0, 70]), i32([0])
    pool.cache.read(pool.table.data_ptr(), 2, pos.data_ptr(), start.data_ptr(), 1, 70, out.data_ptr(), out.stride(0),
                    out[:, 1].data_ptr(), out.stride(0))
    torch.cuda.synchronize()
    for w in range(2):
        equal(out[:, w, :4], model.values(0, 0, 70)[w])
    assert bool((out[:, :, 4] == 7.0).all())


def test_other_pages_and_blocks_keep_their_bytes(qcache):
    pool = Pool(qcache, 3, 2, 2, 64, fill=0x5A)
    before = pool.pool.clone().view(pool.pages, 2, 4, -1)
    k, v = rows_of(gen(1), 20, 2, 64), rows_of(gen(2), 20, 2, 64)
    pool.write([16, 60, 0], [16, 4, 0], k, v)                 # block 1 of page 0; the end of block 3 of page 0
    after = pool.pool.view(pool.pages, 2, 4, -1)
    same = (before == after).all(-1).all(1)                    # [page][block]
    touched = torch.zeros_like(same)
    touched[pool.ids[0, 0], 1] = touched[pool.ids[1, 0], 3] = True
    assert bool((same | touched).all())
    qcache.kv8_check()


def test_rows_behind_the_last_sequence(qcache):
    """More rows than the sequences take (a padded batch): those are not read on
    a write and stay as they were on a read."""
    pool, model, g = Pool(qcache, 2, 2, 2, 128), Model(2, 2, 128), gen(12)
    k, v = rows_of(g, 100, 2, 128), rows_of(g, 100, 2, 128)
    k[60:], v[60:] = math.nan, math.inf
    # every index array stays referenced until the kernels that read it are done
    zero, pos, start0, start, back = (i32(x) for x in ([0, 0], [0, 7], [5, 12, 19], [5, 25, 60], [3, 23, 65]))
    pool.cache.write(pool.table.data_ptr(), 2, zero.data_ptr(), start0.data_ptr(), 2, 100, k.data_ptr(), 256, v.data_ptr(), 256)
    model.write(0, 0, k[5:12], v[5:12])
    model.write(1, 0, k[12:19], v[12:19])
    pool.cache.write(pool.table.data_ptr(), 2, pos.data_ptr(), start.data_ptr(), 2, 100, k.data_ptr(), 256, v.data_ptr(), 256)
    model.write(0, 0, k[5:25], v[5:25])
    model.write(1, 7, k[25:60], v[25:60])
    ko, vo = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    pool.cache.read(pool.table.data_ptr(), 2, zero.data_ptr(), back.data_ptr(), 2, 100, ko.data_ptr(), 256, vo.data_ptr(), 256)
    torch.cuda.synchronize()
    qcache.kv8_check()
    for got, w in ((ko, 0), (vo, 1)):
        equal(got[3:23], model.values(0, 0, 20)[w])
        equal(got[23:65], model.values(1, 0, 42)[w])
        assert bool((got[:3] == 7.0).all()) and bool((got[65:] == 7.0).all())


def test_pages_behind_four_gigabytes(qcache):
    """Pages whose byte offset passes 32 bits; the pool is not filled, only its
    last and first pages are touched."""
    pages = (1 << 32) // qcache.kv8_page_bytes(4, 256) + 9
    pool = torch.empty(pages * qcache.kv8_page_bytes(4, 256), dtype=torch.uint8, device="cuda")
    cache = qcache.Kv8Cache(pool.data_ptr(), pages, 4, 256)
    table, g, model = i32([[pages - 1, 0, pages - 7]]), gen(8), Model(1, 4, 256)
    k, v, start, pos = rows_of(g, 150, 4, 256), rows_of(g, 150, 4, 256), i32([0, 150]), i32([0])
    cache.write(table.data_ptr(), 3, pos.data_ptr(), start.data_ptr(), 1, 150, k.data_ptr(), 1024, v.data_ptr(), 1024)
    model.write(0, 0, k, v)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    cache.read(table.data_ptr(), 3, pos.data_ptr(), start.data_ptr(), 1, 150, ko.data_ptr(), 1024, vo.data_ptr(), 1024)
    torch.cuda.synchronize()
    equal(ko, model.values(0, 0, 150)[0])
    equal(vo, model.values(0, 0, 150)[1])
    q = rows_of(g, 1, 16, 256)
    got = attend(qcache, cache, table, [150], q)
    check_attention(got, q, None, [(ko, vo)], 256 ** -0.5)


def test_many_sequences(qcache):
    """The most sequences of one call, most of them with nothing to write."""
    n, g = 1024, gen(4)
    counts = [(i * 37) % 23 if i % 5 == 0 else 0 for i in range(n)]
    pos = [(i * 11) % 41 for i in range(n)]
    pool, model = Pool(qcache, n, 1, 1, 64, fill=0), Model(n, 1, 64)
    k, v = rows_of(g, sum(counts), 1, 64), rows_of(g, sum(counts), 1, 64)
    pool.write([p // 16 * 16 for p in pos], counts, k, v)
    off = 0
    for i in range(n):
        model.write(i, pos[i] // 16 * 16, k[off:off + counts[i]], v[off:off + counts[i]])
        off += counts[i]
    got = pool.read([p // 16 * 16 for p in pos], counts)
    off = 0
    for i in range(n):
        if counts[i]:
            want = model.values(i, pos[i] // 16 * 16, pos[i] // 16 * 16 + counts[i])
            equal(got[0][off:off + counts[i]], want[0])
            equal(got[1][off:off + counts[i]], want[1])
        off += counts[i]
    qcache.kv8_check()


@pytest.mark.parametrize("what", ["page", "negative page", "position", "negative position", "rows", "negative rows"])
def test_out_of_range_is_skipped_and_reported(qcache, what):
    """The kernel checks every index before it uses it: the bad sequence's rows
    are skipped, the good one's are written, and qc_kv8_check says so once."""
    pool, g = Pool(qcache, 2, 2, 2, 64), gen(6)
    k, v = rows_of(g, 40, 2, 64), rows_of(g, 40, 2, 64)
    table, pos, start, rows = pool.ids.copy(), [0, 0], [0, 20, 40], 40
    if what == "page":
        table[1, 0] = pool.pages
    if what == "negative page":
        table[1, 0] = -1
    if what == "position":
        pos[1] = 128                     # the table's row has two pages
    if what == "negative position":
        pos[1] = -3
    if what == "rows":
        start[2], rows = 60, 40
    if what == "negative rows":
        start[1:] = [20, 5]
    t, p, s = i32(table), i32(pos), i32(start)
    pool.cache.write(t.data_ptr(), 2, p.data_ptr(), s.data_ptr(), 2, rows, k.data_ptr(), 128, v.data_ptr(), 128)
    if what == "negative rows":          # an empty sequence by the rule (no rows)
        qcache.kv8_check()
    else:
        with pytest.raises(qcache.QCacheError) as e:
            qcache.kv8_check()
        assert e.value.code == 5
    qcache.kv8_check()
    model = Model(1, 2, 64)
    model.write(0, 0, k[:20], v[:20])
    got = pool.read([0, 0], [20, 0])
    equal(got[0], model.values(0, 0, 20)[0])
    equal(got[1], model.values(0, 0, 20)[1])
    qcache.kv8_check()


# ---------------------------------------------------------------- attention

def attend(qcache, cache, table, lens, q, gate=None, scale=None, out=None, stream=0):
    n, heads, dim = q.shape
    if out is None:
        out = torch.full((n, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(max(1, cache.attn_workspace_bytes(n, heads)), dtype=torch.uint8, device="cuda")
    ws.fill_(0xFF)                       # NaN patterns: the contents must not matter
    ln = i32(lens)
    cache.attn_decode(table.data_ptr(), table.shape[1], ln.data_ptr(), n, heads, q.data_ptr(), q.stride(0), q.stride(1),
                      gate.data_ptr() if gate is not None else 0, dim ** -0.5 if scale is None else scale,
                      out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(), stream)
    torch.cuda.synchronize()
    return out


def check_attention(got, q, gate, kvs, scale):
    """got against the softmax in 64 bits over kvs[i] = (k, v) [len][kv][dim]."""
    for i, (k, v) in enumerate(kvs):
        heads, dim = q.shape[1:]
        if not len(k):
            assert bool((got[i] == 0).all())
            continue
        kv, group = k.shape[1], q.shape[1] // k.shape[1]
        qi = q[i].double().unflatten(0, (kv, group))
        kk, vv = k.double().permute(1, 2, 0), v.double().transpose(0, 1)
        p = torch.softmax(qi @ kk * scale, -1)
        y, a = p @ vv, p @ vv.abs()
        s = (qi.abs() @ kk.abs() * abs(scale)).amax(-1, keepdim=True)
        n = len(k) / 16
        f = (0 if group <= 4 else 2.0 ** -11) + 4 * 2.0 ** -22 + (dim + 8) * 2.0 ** -23 * s + 8 * 2.0 ** -23 * (1 + s)
        u = torch.cat([b.abs().amax((1, 2), keepdim=True).expand(-1, b.shape[1], 1) for b in vv.split(16, 1)], 1)
        end = len(k) * 2.0 ** -31 * (p * u.transpose(1, 2)).amax(-1, keepdim=True)
        tol = a * (f + 2 * (n + 16) * 2.0 ** -23) + end
        if gate is not None:
            w = torch.sigmoid(gate[i].double().unflatten(0, (kv, group)))
            y, tol = y * w, tol * w + y.abs() * w * 8 * 2.0 ** -24
        tol = tol + (y.abs() + tol) * 2.0 ** -8 + 1e-38
        err = (got[i].double().unflatten(0, (kv, group)) - y).abs()
        assert bool((err <= tol).all()), (i, float((err / tol).max()))


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 500, 1000]


def filled(qcache, lens, kv, dim, seed, fill=0, kstd=1.0, vstd=1.0):
    g = gen(seed)
    pool = Pool(qcache, len(lens), max(1, -(-max(lens) // PAGE)), kv, dim, fill=fill, seed=seed)
    k, v = rows_of(g, sum(lens), kv, dim, kstd), rows_of(g, sum(lens), kv, dim, vstd)
    if sum(lens):
        pool.write([0] * len(lens), lens, k, v)
        k, v = pool.read([0] * len(lens), lens)
    return pool, list(zip(k.split(lens), v.split(lens))), g


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kv,group,dim", [(4, 4, 256), (2, 1, 256), (1, 8, 256), (3, 5, 128), (2, 4, 128), (8, 2, 64),
                                          (1, 7, 64), (1, 3, 64)])
def test_attention_ragged_batch(qcache, kv, group, dim, gated):
    """Every edge length in one batch, garbage (NaN scales) behind the tokens."""
    pool, kvs, g = filled(qcache, LENS, kv, dim, seed=dim + group, fill=0xFF)
    qg = rows_of(g, len(LENS), kv * group, 2 * dim, 2.0)
    q, gate = (qg[:, :, :dim], qg[:, :, dim:]) if gated else (qg[:, :, :dim].contiguous(), None)
    got = attend(qcache, pool.cache, pool.table, LENS, q, gate)
    check_attention(got, q, gate, kvs, dim ** -0.5)
    qcache.kv8_check()
    again = attend(qcache, pool.cache, pool.table, LENS, q, gate)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))       # the same bits on every call


@pytest.mark.parametrize("n,length,kv,group,dim", [(1, 1, 4, 4, 256), (1, 16, 1, 1, 64), (1, 5000, 4, 4, 256),
                                                   (1, 70001, 2, 4, 128), (64, 777, 4, 4, 256), (300, 90, 2, 8, 64),
                                                   (1024, 20, 1, 4, 64), (2, 33333, 1, 6, 256)])
def test_attention_batches_and_long_contexts(qcache, n, length, kv, group, dim):
    lens = [length] * n
    pool, kvs, g = filled(qcache, lens, kv, dim, seed=n)
    q = rows_of(g, n, kv * group, dim)
    check_attention(attend(qcache, pool.cache, pool.table, lens, q), q, None, kvs, dim ** -0.5)
    qcache.kv8_check()


@pytest.mark.parametrize("lens,kv,group,dim", [
    ([16000] * 5, 4, 4, 256), ([90000], 4, 4, 256), ([20000] * 16, 2, 8, 128), ([700] * 9 + [0, 1] + [30011] * 12, 2, 2, 128),
    ([5] * 60 + [65536] * 4, 4, 1, 64), ([40] * 200 + [9000] * 30, 8, 4, 64)])
def test_attention_large_batches_repeat_their_bits(qcache, lens, kv, group, dim):
    """Enough blocks for the small ranges that CTAs draw as they get ready: the
    results are right, and the same bits whoever drew what."""
    pool, kvs, g = filled(qcache, lens, kv, dim, seed=len(lens))
    q = rows_of(g, len(lens), kv * group, dim)
    got = attend(qcache, pool.cache, pool.table, lens, q)
    qcache.kv8_check()
    check_attention(got, q, None, kvs, dim ** -0.5)
    for _ in range(5):
        again = attend(qcache, pool.cache, pool.table, lens, q)
        assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    qcache.kv8_check()


def test_attention_one_long_among_short(qcache):
    lens = [3, 20000, 0, 1, 640, 64, 0, 2]
    pool, kvs, g = filled(qcache, lens, 4, 256, seed=9)
    q = rows_of(g, len(lens), 16, 256)
    check_attention(attend(qcache, pool.cache, pool.table, lens, q), q, None, kvs, 1 / 16)


@pytest.mark.parametrize("group", [4, 8])
@pytest.mark.parametrize("case", ["peaked", "block scales", "constant", "large values", "small values", "rising"])
def test_attention_distributions(qcache, case, group):
    """Scores that leave one token, blocks whose scales are far apart (also the
    block that holds nearly all the weight being the smallest), equal scores,
    and scores that rise along the context, so that the maximum keeps moving."""
    kv, dim, length = 2, 128, 900
    g = gen(group)
    pool = Pool(qcache, 1, 15, kv, dim)
    k, v, q = rows_of(g, length, kv, dim), rows_of(g, length, kv, dim), rows_of(g, 1, kv * group, dim)
    scale = dim ** -0.5
    if case == "peaked":
        q = q * 30
    if case == "block scales":
        f = torch.exp2(torch.randint(-30, 30, (length // 16 + 1, 1, 1), generator=g, device="cuda").float())
        v = (v * f.repeat_interleave(16, 0)[:length]).bfloat16()
        k = (k / 4).bfloat16()
        k[320:336] = q[0, ::group] * 4    # the weight is there, at the smallest values
        v[320:336] = (v[320:336] / f[20] * 2.0 ** -40).bfloat16()
    if case == "constant":
        k[:] = k[0]
    if case == "large values":
        k, v = (k * 2.0 ** 60).bfloat16(), (v * 2.0 ** 90).bfloat16()
        q = (q * 2.0 ** -61).bfloat16()
    if case == "small values":
        k, v = (k * 2.0 ** -60).bfloat16(), (v * 2.0 ** -90).bfloat16()
        q = (q * 2.0 ** 60).bfloat16()
    if case == "rising":
        k = (q[0, ::group] * torch.linspace(-3, 3, length, device="cuda")[:, None, None]).bfloat16()
    q = q.bfloat16()
    pool.write([0], [length], k, v)
    k, v = pool.read([0], [length])
    check_attention(attend(qcache, pool.cache, pool.table, [length], q), q, None, [(k, v)], scale)


def test_attention_scale_argument(qcache):
    pool, kvs, g = filled(qcache, [200, 40], 2, 64, seed=2)
    q = rows_of(g, 2, 8, 64)
    for scale in (0.0, 1.0, -0.25, 0.01):
        check_attention(attend(qcache, pool.cache, pool.table, [200, 40], q, scale=scale), q, None, kvs, scale)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_non_finite_query_stays_in_its_head(qcache, bad):
    pool, kvs, g = filled(qcache, [300, 17], 2, 128, seed=3)
    q = rows_of(g, 2, 8, 128)
    clean = attend(qcache, pool.cache, pool.table, [300, 17], q)
    q2 = q.clone()
    q2[0, 5, 77] = bad
    got = attend(qcache, pool.cache, pool.table, [300, 17], q2)
    assert bool(torch.isnan(got[0, 5]).all())
    got[0, 5] = clean[0, 5]
    assert torch.equal(got.view(torch.int16), clean.view(torch.int16))


def test_attention_output_rows_and_strides(qcache):
    """out inside wider rows, q rows with gaps: neighbours keep their bits, the
    rows behind the last sequence too."""
    lens = [70, 0, 5]
    pool, kvs, g = filled(qcache, lens, 2, 64, seed=4)
    wide = rows_of(g, 3, 8, 64 * 3 + 8)
    q = wide[:, :, 64:128]
    buf = torch.full((5, 8 * 64 + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:3, :512].unflatten(1, (8, 64))
    attend(qcache, pool.cache, pool.table, lens, q, out=out)
    check_attention(out, q, None, kvs, 64 ** -0.5)
    assert bool((buf[3:] == 7.0).all()) and bool((buf[:, 512:] == 7.0).all())


@pytest.mark.parametrize("what", ["page", "negative page", "length", "negative length"])
def test_attention_out_of_range_is_reported(qcache, what):
    """The bad page's tokens are left out, the other sequence's result stands."""
    lens = [100, 150]
    pool, kvs, g = filled(qcache, lens, 2, 128, seed=5)
    q = rows_of(g, 2, 8, 128)
    want = attend(qcache, pool.cache, pool.table, lens, q)
    ids, ln = pool.ids.copy(), list(lens)
    if what == "page":
        ids[1, 1] = pool.pages + 5
    if what == "negative page":
        ids[1, 1] = -2
    if what == "length":
        ln[1] = 64 * pool.width + 1
    if what == "negative length":
        ln[1] = -5
    got = attend(qcache, pool.cache, i32(ids), ln, q)
    with pytest.raises(qcache.QCacheError) as e:
        qcache.kv8_check()
    assert e.value.code == 5
    qcache.kv8_check()
    assert torch.equal(got[0].view(torch.int16), want[0].view(torch.int16))
    if "page" in what:
        k, v = kvs[1]
        rest = [i for i in range(150) if not 64 <= i < 128]
        check_attention(got[1:], q[1:], None, [(k[rest], v[rest])], 128 ** -0.5)
    if what == "negative length":
        assert bool((got[1] == 0).all())


def test_workspace_and_host_memory_are_refused(qcache):
    pool, _, g = filled(qcache, [20], 2, 64, seed=6)
    q, ln = rows_of(g, 1, 8, 64), i32([20])
    out = torch.empty_like(q)
    need = pool.cache.attn_workspace_bytes(1, 8)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    host = torch.empty(need + 4096, dtype=torch.uint8).pin_memory()

    def call(ws_ptr, size, q_ptr=q.data_ptr()):
        pool.cache.attn_decode(pool.table.data_ptr(), 1, ln.data_ptr(), 1, 8, q_ptr, 512, 64, 0, 0.125, out.data_ptr(),
                               512, ws_ptr, size)

    call(ws.data_ptr(), need)
    for args, text in (((ws.data_ptr(), need - 1), "workspace"), ((0, need), "workspace is null"),
                       ((host.data_ptr(), need), "device memory"), ((ws.data_ptr(), need, host.data_ptr()), "device memory")):
        with pytest.raises(qcache.QCacheError) as e:
            call(*args)
        assert e.value.code == qcache.QC_ERR_ARG and text in str(e.value)


def test_captured_steps_and_two_graphs_at_once(qcache):
    """A decode step (write, then attend) captured once and replayed while the
    positions advance on the device, and two such graphs with a workspace each
    replayed side by side on two streams."""
    kv, group, dim, n, lens = 2, 4, 128, 3, [60, 5, 200]
    sets = []
    for seed in (1, 2):
        pool, kvs, g = filled(qcache, lens, kv, dim, seed=seed)
        pool2 = Pool(qcache, n, 6, kv, dim, seed=seed)        # room to grow
        pool2.write([0] * n, lens, torch.cat([a for a, _ in kvs]), torch.cat([b for _, b in kvs]))
        s = dict(pool=pool2, g=g, pos=i32(lens), len=i32([x + 1 for x in lens]), k=rows_of(g, n, kv, dim),
                 v=rows_of(g, n, kv, dim), q=rows_of(g, n, kv * group, dim), kvs=[(a, b) for a, b in kvs])
        s["out"] = torch.empty(n, kv * group, dim, dtype=torch.bfloat16, device="cuda")
        s["ws"] = torch.empty(pool2.cache.attn_workspace_bytes(n, kv * group), dtype=torch.uint8, device="cuda")
        s["graph"], s["stream"] = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(s["graph"], stream=s["stream"]):
            st = torch.cuda.current_stream().cuda_stream
            c, t = pool2.cache, pool2.table
            c.write(t.data_ptr(), 6, s["pos"].data_ptr(), 0, n, n, s["k"].data_ptr(), kv * dim, s["v"].data_ptr(), kv * dim, st)
            c.attn_decode(t.data_ptr(), 6, s["len"].data_ptr(), n, kv * group, s["q"].data_ptr(), kv * group * dim, dim, 0,
                          dim ** -0.5, s["out"].data_ptr(), kv * group * dim, s["ws"].data_ptr(), s["ws"].numel(), st)
            s["pos"].add_(1)
            s["len"].add_(1)
        sets.append(s)
    for step in range(20):
        for s in sets:
            s["k"].copy_(rows_of(s["g"], n, kv, dim, 1.0 + step))
            s["q"].copy_(rows_of(s["g"], n, kv * group, dim))
        torch.cuda.synchronize()
        for s in sets:
            with torch.cuda.stream(s["stream"]):
                s["graph"].replay()
        torch.cuda.synchronize()
        for s in sets:
            now = [x + step + 1 for x in lens]
            k, v = s["pool"].read([0] * n, now)
            check_attention(s["out"], s["q"], None, list(zip(k.split(now), v.split(now))), dim ** -0.5)
    qcache.kv8_check()


def test_first_calls_of_a_process_may_be_captured(qcache):
    """Kernel attributes, occupancy and module loading on the first call of a
    process, all inside a capture."""
    import os
    import subprocess
    import sys

    code = """
import importlib.util, torch
spec = importlib.util.spec_from_file_location("qcache", PATH)
qc = importlib.util.module_from_spec(spec)
spec.loader.exec_module(qc)
pool = torch.zeros(4 * qc.kv8_page_bytes(2, 128), dtype=torch.uint8, device="cuda")
c = qc.Kv8Cache(pool.data_ptr(), 4, 2, 128)
table, pos, ln = torch.zeros(3, 1, dtype=torch.int32, device="cuda").unbind(0)
ln = ln + 1
k, q = torch.ones(1, 2, 128, device="cuda").bfloat16(), torch.ones(1, 8, 128, device="cuda").bfloat16()
out = torch.zeros_like(q)
ws = torch.empty(c.attn_workspace_bytes(1, 8), dtype=torch.uint8, device="cuda")
rope, g = qc.Rope(64), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g):
    st = torch.cuda.current_stream().cuda_stream
    rope.apply(128, pos.data_ptr(), 1, [qc.RopePart(k.data_ptr(), k.data_ptr(), 2, 256, 128, 256, 128)], 1e-6, st)
    c.write(table.data_ptr(), 1, pos.data_ptr(), 0, 1, 1, k.data_ptr(), 256, k.data_ptr(), 256, st)
    c.attn_decode(table.data_ptr(), 1, ln.data_ptr(), 1, 8, q.data_ptr(), 1024, 128, 0, 0.1, out.data_ptr(), 1024,
                  ws.data_ptr(), ws.numel(), st)
g.replay()
qc.kv8_check(st)
assert bool((out == 1).all())
"""
    code = code.replace("PATH", repr(os.path.abspath(qcache.__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
