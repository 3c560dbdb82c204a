"""Failed calls on the caller's buffers (rotary, 8-bit cache) leave nothing behind."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from gpu_util import empty_u16  # noqa: E402
from test_gpu_kv8 import filled, i32, rows_of  # noqa: E402


def test_a_refused_launch_does_not_fail_the_next_call(qcache):
    """Launches into a capture that another call has made invalid are refused with
    QC_ERR_CUDA; calls on other streams go on as if nothing had been."""
    cu = C.CDLL("libcuda.so.1")
    pool, kvs, g = filled(qcache, [70], 2, 64, seed=1)
    q, k, pos, ln = rows_of(g, 1, 4, 64), rows_of(g, 1, 2, 64), i32([70]), i32([70])
    out, ws = torch.zeros_like(q), torch.empty(pool.cache.attn_workspace_bytes(1, 4), dtype=torch.uint8, device="cuda")
    rope = qcache.Rope(64)
    ctx = qcache.QCache(n_attn_layers=1, n_gdn_layers=1, max_seqs=1, max_pages=2, max_ctx=64, max_batch=1, max_snapshots=1,
                        device=0)
    seq = ctx.seq_alloc()
    ctx.seq_reserve(seq, 1)
    row = empty_u16(1, 1024)
    torch.cuda.synchronize()

    def calls(st):
        t = pool.table.data_ptr()
        yield lambda: rope.apply(64, pos.data_ptr(), 1, [qcache.RopePart(q.data_ptr(), out.data_ptr(), 4, 256, 64, 256, 64)], 1e-6, st)
        yield lambda: pool.cache.write(t, pool.width, pos.data_ptr(), 0, 1, 1, k.data_ptr(), 128, k.data_ptr(), 128, st)
        yield lambda: pool.cache.read(t, pool.width, pos.data_ptr(), 0, 1, 1, k.data_ptr(), 128, k.data_ptr(), 128, st)
        yield lambda: pool.cache.attn_decode(t, pool.width, ln.data_ptr(), 1, 4, q.data_ptr(), 256, 64, 0, 0.125,
                                             out.data_ptr(), 256, ws.data_ptr(), ws.numel(), st)
        yield lambda: qcache.kv8_check(st)

    for i in range(5):
        stream = torch.cuda.Stream()
        h, graph = C.c_void_p(stream.cuda_stream), C.c_void_p()
        assert cu.cuStreamBeginCapture_v2(h, 2) == 0            # relaxed: no other stream is concerned
        assert cu.cuStreamSynchronize(h) != 0                   # not allowed meanwhile: the capture is invalid now
        with pytest.raises(qcache.QCacheError) as e:
            list(calls(stream.cuda_stream))[i]()
        assert e.value.code == qcache.QC_ERR_CUDA
        assert cu.cuStreamEndCapture(h, C.byref(graph)) != 0 and not graph.value
        ctx.kv_write(seq, 0, 0, 1, row.data_ptr(), row.data_ptr())
        for call in calls(0):
            call()
        torch.cuda.synchronize()
    ctx.check_device()
    ctx.close()
