"""The paged cache's entry points without a GPU, at the edges: sizes of the workspace and what Python passes on. The
handles are test_paged_host.py's stand-ins."""
import ctypes

import pytest

from test_paged_host import CACHE


class _Ctx(ctypes.Structure):  # the fields that the workspace's size is worked out from
    _fields_ = [("device", ctypes.c_int), ("stream", ctypes.c_void_p), ("sms", ctypes.c_int)]


def _workspace(T, heads, S=1, G=0, sms=148, cache=CACHE):
    from decision_js_b200._lib import lib
    ctx, n = _Ctx(0, None, sms), ctypes.c_size_t()
    assert lib().dc_attention_paged_workspace(ctypes.addressof(ctx), ctypes.addressof(cache), T, heads, S, G, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("T,heads", [(1, 2), (7, 4), (64, 16), (5000, 24)])
def test_the_workspace_may_start_at_any_multiple_of_16(pkg, T, heads):
    """The header asks for 16 bytes, parts are stored 32 at a time: the layout (whole multiples of 256 bytes) starts at the
    next multiple of 256, up to 240 bytes behind the address given."""
    assert _workspace(T, heads) % 256 == 240
