"""Reads of keys and values into one another's memory are refused."""
import ctypes as C

import pytest

from shear_amd import _native as N
from test_kv_abi_step import good4


def refusal(v, kind):
    a = good4()
    rows = N.KvRows(0x1000, 0x20000, v, 3, kind, 0)  # 3 rows of 2 heads x 64 dims
    st = N.load().tessa_kv_read(C.byref(a["cache"]), C.byref(rows), None)
    return st.code, st.msg.decode()


@pytest.mark.parametrize("kind,size", [(N.KV_BF16, 768), (N.KV_F16, 768), (N.KV_F32, 1536)])
def test_values_over_keys(kind, size):
    for v in (0x20000, 0x20000 + size - 16, 0x20000 - size + 16):
        code, text = refusal(v, kind)
        assert code == 1 and "overlap" in text, hex(v)


@pytest.mark.parametrize("kind,size", [(N.KV_BF16, 768), (N.KV_F16, 768), (N.KV_F32, 1536)])
def test_values_beside_keys(kind, size):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("made-up pointers: only where nothing can run")
    for v in (0x20000 + size, 0x20000 - size, None):
        assert refusal(v, kind)[0] != 1
