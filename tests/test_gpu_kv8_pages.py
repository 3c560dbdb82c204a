"""The 8-bit cache's page tables: rewritten on the device between calls, and kept beside
a context whose pages are shared."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_kv8 import check_attention, filled, i32, rows_of  # noqa: E402


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
