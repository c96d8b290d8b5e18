"""Page calls with more requests than are taken are refused before anything runs."""

import ctypes

from sparseflow_amd import _lib


def test_more_requests_than_are_taken():
    """Each request looks through those before it for its row: 2^20 of them come to 2^39 looks, 2^24 to minutes."""
    L = _lib.lib()
    one, at = ctypes.c_void_p(16), ctypes.addressof
    d = _lib.PagesDesc(4, 2, 2, (1 << 20) + 1, 4, 0)
    for fn in (L.sf_pages_resize, L.sf_pages_fork):
        assert fn(at(d), one, one, one, one, one, one, one, 1 << 40, None) == _lib.SF_ERR_UNSUPPORTED
    d.requests = 1 << 20
    for fn in (L.sf_pages_resize, L.sf_pages_fork):
        assert fn(at(d), one, one, one, one, one, one, None, 0, None) == _lib.SF_ERR_WORKSPACE
    d.requests = (1 << 24) + 1
    assert L.sf_pages_copy(at(d), one, one, None) == _lib.SF_ERR_UNSUPPORTED
