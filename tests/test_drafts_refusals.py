"""What the native entries around drafted tokens and pages refuse on the host, before any launch (no GPU)."""
import ctypes as C

import pytest

from safetyraise_lmengine_b200.kernels import ops

BAD_ALIGN = -3


@pytest.mark.parametrize("address", [1001, 4097])
def test_pools_at_odd_addresses_are_refused(address):
    """The narrowest access is of two bytes: a pool of one-byte numbers that starts on an odd address has none that fits."""
    src, dst = (C.c_longlong * 1)(0), (C.c_longlong * 1)(1)
    for page_bytes in (2, 16, 4096):
        assert ops._entry("srlm_copy_pages")(address, 1, 4, page_bytes, src, dst, 1, 148, None) == BAD_ALIGN
    assert ops._entry("srlm_keep_drafts")(address, 2, 4, 1, 16, 128, 4096, 1, 4096, 4096, 4096, 3, 4096, 1, 4096, None) == BAD_ALIGN
