"""CPU tests of what include/qrope.h and include/qkv8.h refuse beyond test_kv8_abi.py:
index arrays that a kernel could not read (the refusal comes before any pointer is
looked up on a device)."""
import pytest


def refused(qcache, fn, text):
    with pytest.raises(qcache.QCacheError) as e:
        fn()
    assert e.value.code == qcache.QC_ERR_ARG, str(e.value)
    assert text in str(e.value), str(e.value)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_index_arrays_are_aligned(qcache, off):
    at, odd = 1 << 12, (1 << 12) + off
    part = qcache.RopePart(at, at, 4, 1024, 256, 1024, 256)
    refused(qcache, lambda: qcache.Rope(64).apply(256, odd, 1, [part]), "4-byte aligned")
    c = qcache.Kv8Cache(at, 8, 4, 256)
    for table, pos, start in ((odd, at, at), (at, odd, at), (at, at, odd), (at, odd, 0)):
        for call in (c.write, c.read):
            refused(qcache, lambda: call(table, 4, pos, start, 2, 2, at, 1024, at, 1024), "4-byte aligned")
    for table, ln in ((odd, at), (at, odd)):
        refused(qcache, lambda: c.attn_decode(table, 4, ln, 2, 16, at, 8192, 512, 0, 0.0625, at, 4096, at, 1 << 30),
                "4-byte aligned")
