"""qc_kv8_check beside other streams and other threads."""
import ctypes as C
import threading

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_kv8 import Pool, gen, i32, rows_of  # noqa: E402


def driver(name, *args):
    rc = getattr(C.CDLL("libcuda.so.1"), name)(*args)
    assert rc == 0, (name, rc)


@pytest.fixture
def blocking_stream():
    """A stream that the legacy default stream waits for (torch's are not)."""
    torch.cuda.current_stream().synchronize()
    h = C.c_void_p()
    driver("cuStreamCreate", C.byref(h), 0)
    yield torch.cuda.ExternalStream(h.value)
    driver("cuStreamSynchronize", h)
    driver("cuStreamDestroy_v2", h)


def bad_write(pool, g, stream):
    """A write whose position is out of range: skipped and recorded."""
    k, pos = rows_of(g, 1, 2, 64), i32([-1])
    torch.cuda.synchronize()
    pool.cache.write(pool.table.data_ptr(), 1, pos.data_ptr(), 0, 1, 1, k.data_ptr(), 128, k.data_ptr(), 128, stream)
    torch.cuda.synchronize()


def test_check_waits_for_its_own_stream_alone(qcache, blocking_stream):
    pool, g, side = Pool(qcache, 1, 1, 2, 64), gen(1), torch.cuda.Stream()
    qcache.kv8_check(side.cuda_stream)           # the driver loads a kernel once, for which it may wait for all
    bad_write(pool, g, side.cuda_stream)
    done = torch.cuda.Event()
    with torch.cuda.stream(blocking_stream):
        torch.cuda._sleep(2_000_000_000)         # about a second
        done.record()
    with pytest.raises(qcache.QCacheError) as e:
        qcache.kv8_check(side.cuda_stream)
    assert e.value.code == qcache.QC_ERR_BOUNDS
    assert not done.query()
    qcache.kv8_check(side.cuda_stream)
    assert not done.query()


def test_an_error_is_reported_to_one_of_several_threads(qcache):
    pool, g = Pool(qcache, 1, 1, 2, 64), gen(2)
    threads, rounds = 3, 200
    streams = [torch.cuda.Stream() for _ in range(threads)]
    start, end = threading.Barrier(threads + 1), threading.Barrier(threads + 1)
    seen = [[] for _ in range(rounds)]

    def ask(stream):
        for r in range(rounds):
            start.wait()
            try:
                qcache.kv8_check(stream.cuda_stream)
            except qcache.QCacheError as e:
                seen[r].append(e.code)
            end.wait()

    ts = [threading.Thread(target=ask, args=(s,), daemon=True) for s in streams]
    for t in ts:
        t.start()
    for r in range(rounds):
        bad_write(pool, g, 0)
        start.wait()
        end.wait()
    for t in ts:
        t.join()
    assert all(s == [qcache.QC_ERR_BOUNDS] for s in seen), [s for s in seen if len(s) != 1][:3]
    qcache.kv8_check()
