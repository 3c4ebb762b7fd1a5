"""The paged cache's later checks, without a GPU: what the host refuses before anything is launched."""
import ctypes as C

import pytest

from test_paged_cpu import A, cache
from xalm_b200 import capi


@pytest.mark.parametrize("bad,taken", [(dict(), 0), (dict(status=0), A), (dict(page_size=24, status=A), A), (dict(k=0, status=A), A)])
def test_a_status_that_cannot_be_taken_is_refused(bad, taken):
    c = cache(**{"status": A, **bad})
    assert capi.lib().xalm_cuda_paged_status(C.byref(c), taken, None) == 1
    assert capi.lib().xalm_cuda_last_error()
    assert capi.lib().xalm_cuda_paged_status(None, taken, None) == 1
