"""Where the rotated append's queries may go: to q's own rows, but not over k's or v's, nor over q's in another order."""
import ctypes as C

import pytest

from shear_amd import _native as N
from test_kv_abi_step import good4


def refusal(**change):
    a = good4()
    t = a["rotated"]
    t.tokens = 3
    for name, value in change.items():
        setattr(t, name, value)
    st = N.load().tessa_kv_append_rotated(C.byref(a["cache"]), C.byref(t), None)
    return st.code, st.msg.decode()


@pytest.mark.parametrize("change", [dict(out=0x2000), dict(out=0x3000), dict(out=0x1000, out_strides=(512, 64)),
                                    dict(out=0x1000, out_strides=(256, 128))])
def test_out_that_is_refused(change):
    code, text = refusal(**change)
    assert code == 1 and "out" in text and "q" in text


def test_out_that_is_q():
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("made-up pointers: only where nothing can run")
    assert refusal(out=0x1000)[0] != 1
    assert refusal(out=0x1000, q_heads=1, q_strides=(256, 64), out_strides=(256, 128))[0] != 1
    assert refusal()[0] != 1
