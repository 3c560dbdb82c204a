"""The 8-bit cache's page tables: rewritten on the device between calls, and kept beside
a context whose pages are shared."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from gpu_util import empty_u16  # noqa: E402
from test_gpu_kv8 import attend, check_attention, filled, gen, i32, rows_of  # noqa: E402


def test_table_rewritten_by_the_kernel_before(qcache):
    """A captured chain in which the table changes between two attention calls, and
    between a write and a read of the same length: each sees the table of its turn."""
    lens = [200, 200, 200]
    pool, kvs, g = filled(qcache, lens, 2, 128, seed=3)
    q, ln, zero, start = rows_of(g, 1, 8, 128), i32([200]), i32([0]), i32([0, 200])
    tables = [i32(pool.ids[i:i + 1]) for i in range(3)]
    table = torch.zeros_like(tables[0])
    outs = [torch.zeros_like(q) for _ in range(3)]
    reads = [torch.zeros(2, 200, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    ws = torch.empty(pool.cache.attn_workspace_bytes(1, 8), dtype=torch.uint8, device="cuda")
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        st = torch.cuda.current_stream().cuda_stream
        for turn in range(3):
            table.copy_(tables[turn])
            pool.cache.attn_decode(table.data_ptr(), pool.width, ln.data_ptr(), 1, 8, q.data_ptr(), 1024, 128, 0, 128 ** -0.5,
                                   outs[turn].data_ptr(), 1024, ws.data_ptr(), ws.numel(), st)
            pool.cache.read(table.data_ptr(), pool.width, zero.data_ptr(), start.data_ptr(), 1, 200, reads[turn][0].data_ptr(),
                            256, reads[turn][1].data_ptr(), 256, st)
    for _ in range(10):
        graph.replay()
    torch.cuda.synchronize()
    qcache.kv8_check()
    for (k, v), out, r in zip(kvs, outs, reads):
        assert torch.equal(r[0], k) and torch.equal(r[1], v)
        check_attention(out, q, None, [(k, v)], 128 ** -0.5)


class Beside:
    """A context of one attention layer and an 8-bit pool under its page ids."""

    KV, D, WIDTH = 4, 256, 8

    def __init__(self, qcache, pages=16):
        self.ctx = qcache.QCache(n_attn_layers=1, n_gdn_layers=1, max_seqs=3, max_pages=pages, max_ctx=512, max_batch=3,
                                 max_snapshots=2, device=0)
        self.pool = torch.full((pages * qcache.kv8_page_bytes(self.KV, self.D),), 0xFF, dtype=torch.uint8, device="cuda")
        self.cache = qcache.Kv8Cache(self.pool.data_ptr(), pages, self.KV, self.D)

    def table(self, seq):
        ids = self.ctx.seq_pages(seq)
        return i32([ids + [0] * (self.WIDTH - len(ids))])

    def rows(self, call, seq, pos, n, k, v):
        p, start, t = i32([pos]), i32([0, n]), self.table(seq)
        call(t.data_ptr(), self.WIDTH, p.data_ptr(), start.data_ptr(), 1, n, k.data_ptr(), 1024, v.data_ptr(), 1024)
        torch.cuda.synchronize()

    def move(self, seq, lo, hi):
        """Positions lo .. hi-1 from the context's pages into the 8-bit ones."""
        k, v = empty_u16(hi - lo, self.KV, self.D), empty_u16(hi - lo, self.KV, self.D)
        self.ctx.kv_read(seq, 0, lo, hi - lo, k.data_ptr(), v.data_ptr())
        self.rows(self.cache.write, seq, lo, hi - lo, k, v)

    def put_back(self, seq, lo, hi):
        k, v = self.read(seq, lo, hi)
        self.ctx.kv_write(seq, 0, lo, hi - lo, k.data_ptr(), v.data_ptr())
        torch.cuda.synchronize()

    def read(self, seq, lo, hi):
        k = torch.zeros(hi - lo, self.KV, self.D, dtype=torch.bfloat16, device="cuda")
        v = torch.zeros_like(k)
        self.rows(self.cache.read, seq, lo, hi - lo, k, v)
        return k, v

    def step(self, qcache, seq, k, v, q):
        """One decoded token of one sequence, over the 8-bit pool alone."""
        at = self.ctx.seq_len(seq)
        self.ctx.decode_begin([seq])
        self.rows(self.cache.write, seq, at, 1, k, v)
        out = attend(qcache, self.cache, self.table(seq), [at + 1], q)
        self.ctx.decode_end()
        now = self.read(seq, 0, at + 1)
        check_attention(out, q, None, [now], self.D ** -0.5)
        return now


@pytest.mark.parametrize("prompt", [128, 150, 5])
def test_prefix_entry_beside_the_8_bit_pool(qcache, prompt):
    """A prompt moved over, decoded in 8 bits, put back and inserted; a second
    sequence restored from it: both go on from the same tokens.  The restored tail is
    quantised from values that were quantised at most twice before (when written and as
    a block's scale grew), each time by at most half a scale, which is u / 127 for a
    block's largest magnitude u; its own step adds as much: together under 4 u / 127."""
    b, g = Beside(qcache), gen(prompt)
    a = b.ctx.seq_alloc()
    b.ctx.seq_reserve(a, prompt)
    k, v = rows_of(g, prompt, 4, 256), rows_of(g, prompt, 4, 256)
    b.ctx.kv_write(a, 0, 0, prompt, k.data_ptr(), v.data_ptr())
    b.move(a, 0, prompt)
    for _ in range(9):
        b.step(qcache, a, rows_of(g, 1, 4, 256), rows_of(g, 1, 4, 256), rows_of(g, 1, 16, 256))
    n = prompt + 9
    b.put_back(a, prompt, n)
    entry = b.ctx.prefix_insert(a, list(range(n)))
    c = b.ctx.seq_alloc()
    b.ctx.prefix_restore([entry], [c])
    full = n // 64 * 64
    assert b.ctx.seq_pages(c)[:full // 64] == b.ctx.seq_pages(a)[:full // 64]
    if full < n:
        assert b.ctx.seq_pages(c)[full // 64] != b.ctx.seq_pages(a)[full // 64]
        b.move(c, full, n)
    mine, theirs = b.read(c, 0, n), b.read(a, 0, n)
    for x, y in zip(mine, theirs):
        assert torch.equal(x[:full], y[:full])
        x, y = x.double(), y.double()
        for lo in range(full, n, 16):
            u = y[lo:lo + 16].abs().amax((0, 2), keepdim=True)
            assert bool(((x[lo:lo + 16] - y[lo:lo + 16]).abs() <= 4 * u / 127).all())
    for _ in range(3):
        k, v, q = rows_of(g, 1, 4, 256), rows_of(g, 1, 4, 256), rows_of(g, 1, 16, 256)
        b.step(qcache, a, k, v, q)
        b.step(qcache, c, k, v, q)
    b.ctx.check_device()
    qcache.kv8_check()
    b.ctx.close()
