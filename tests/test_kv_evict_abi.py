"""Eviction's C entry point on a machine without a GPU: buffers that may not be shared."""
import ctypes as C

from shear_amd import _native as N
from test_kv_abi import good


def test_new_lengths_are_not_the_lengths():
    # every head's workgroup reads a sequence's length, one of them writes the new one
    a = good()
    a["evict"].new_lengths = a["seq"].lengths
    st = N.load().tessa_kv_evict(C.byref(a["cache"]), C.byref(a["seq"]), C.byref(a["evict"]), None)
    assert st.code == 1 and "new_lengths" in st.msg.decode()
