"""The paged cache's later checks, without a GPU: what the host refuses before anything is launched."""
import ctypes as C

import pytest

from test_paged_cpu import A, ALL, batch, cache, calls
from xalm_b200 import capi


@pytest.mark.parametrize("bad,taken", [(dict(), 0), (dict(status=0), A), (dict(page_size=24, status=A), A), (dict(k=0, status=A), A), (dict(status=A + 2), A), (dict(), A + 1)])
def test_a_status_that_cannot_be_taken_is_refused(bad, taken):
    c = cache(**{"status": A, **bad})
    assert capi.lib().xalm_cuda_paged_status(C.byref(c), taken, None) == 1
    assert capi.lib().xalm_cuda_last_error()
    assert capi.lib().xalm_cuda_paged_status(None, taken, None) == 1


@pytest.mark.parametrize("off", [1, 2, 3])
def test_numbers_that_lie_across_their_boundaries_are_refused(off):
    """Arrays of 4-byte numbers: a kernel that reads one elsewhere faults."""
    for name in ALL:
        assert calls(cache(status=A + off), batch())[name]() == 1, name
        for what in ("starts", "lens", "table"):
            assert calls(cache(), batch(**{what: A + off}))[name]() == 1, (name, what)
        for what in ("group_bounds", "group_shared"):
            assert calls(cache(), batch(**{"groups": 1, "group_bounds": A, "group_shared": A, what: A + off}))[name]() == 1, (name, what)
    assert calls(cache(), batch(), freq=A + off)["append"]() == 1
    assert calls(cache(), batch(), lists=A + off)["attend_selected"]() == 1
    assert calls(cache(), batch(), out=A + off)["select"]() == 1
    c, b = cache(), batch()
    L, p, w = capi.lib(), C.byref(c), C.byref(b)
    assert L.xalm_cuda_paged_attend(p, w, A, 512, 8, 0.1, A, 512, A + off, A, 1 << 40, None) == 1
    assert L.xalm_cuda_paged_attend_selected(p, w, A, 512, 8, A, 4, 0.1, A, 512, A + off, A, 1 << 40, None) == 1
    assert b"4-byte" in L.xalm_cuda_last_error()
