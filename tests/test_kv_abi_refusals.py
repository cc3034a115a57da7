"""The key-value cache's C entry points on a machine without a GPU: buffers that may not be shared, tokens that no
sequence has."""
import ctypes as C

from shear_amd import _native as N
from test_kv_abi import good


def test_new_lengths_are_not_the_lengths():
    # every head's workgroup reads a sequence's length, one of them writes the new one
    a = good()
    a["evict"].new_lengths = a["seq"].lengths
    st = N.load().tessa_kv_evict(C.byref(a["cache"]), C.byref(a["seq"]), C.byref(a["evict"]), None)
    assert st.code == 1 and "new_lengths" in st.msg.decode()


def test_prompt_tokens_of_no_sequence():
    # nothing would write their rows of out
    a = good()
    a["seq"].batch = 0
    a["attend"].offsets = 0x10
    size = C.c_uint64(7)
    args = C.byref(a["cache"]), C.byref(a["seq"]), C.byref(a["attend"])
    st = N.load().tessa_kv_attend_prompt_scratch(*args, C.byref(size))
    assert st.code == 1 and "no sequence" in st.msg.decode() and size.value == 0
    assert N.load().tessa_kv_attend_prompt(*args, None, 0, None).code == 1
    a["attend"].tokens = 0
    assert N.load().tessa_kv_attend_prompt(*args, None, 0, None).code == 0
