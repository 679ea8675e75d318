"""Sizes that the page operators refuse before anything reaches a GPU."""
import ctypes

import pytest

b2 = pytest.importorskip("b2gguf")


@pytest.mark.parametrize("n_head,n_kv,n_tok", [(1 << 29, 2, 2), (1 << 20, 1, 1), (4, 1 << 30, 1), (4, 2, 2 ** 31 - 1)])
def test_store_refuses_sizes_it_cannot_count(n_head, n_kv, n_tok):
    c = b2._PageCacheC(1 << 20, 1 << 24, 1, 1, 16, n_kv, 64, b2.F16, b2.F16)
    b = b2.PageBatch(1 << 12, 1 << 12, 1 << 12, n_seq=1, max_pages=1, n_tok=n_tok, max_q=1)
    rc = b2.lib.b2_page_rope_store(ctypes.addressof(c), 0, b.ref, n_head, 1 << 12, b2.F32, 1 << 12, b2.F32, 1 << 12, 1,
                                   1 << 12, 1 << 12, 10, 64, 0, None)
    assert rc == b2.ERR_INVALID and b"page" in b2.lib.b2_last_error()


def test_cache_refuses_heads_that_cannot_be_counted():
    with pytest.raises(b2.B2Error):
        b2.PageCache(1, 1, 16, (1 << 20) + 1, 64, k=1 << 20, v=1 << 24)
    c = b2._PageCacheC(1 << 20, 1 << 24, 1, 1, 16, 1 << 27, 64, b2.F16, b2.F16)
    assert b2.lib.b2_page_gather(ctypes.addressof(c), 1, 16, 16, 1, 16, 16, 4, None) == b2.ERR_INVALID
