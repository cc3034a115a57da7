"""The C entry points of 4-bit caches, of a step's plan, of the rotated append and of reads, on a machine without a GPU:
struct layouts, and arguments that are refused before any device work."""
import ctypes as C
import shutil
import subprocess

import numpy as np
import pytest

from kv4_reference import GRID, mx4_rule, mx4_values, pack
from shear_amd import _native as N
from test_kv_abi import HEADER, good

STRUCTS = {"tessa_kv_rotated": N.KvRotated, "tessa_kv_rows": N.KvRows, "tessa_kv_step": N.KvStep}


def test_struct_layouts_match_the_c_compiler(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for f, _ in cls._fields_:
            lines.append(f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));')
    src = tmp_path / "layout.c"
    src.write_text("\n".join([*lines, "return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True,
                                                       check=True).stdout.splitlines())
    for name, cls in STRUCTS.items():
        assert int(got[name]) == C.sizeof(cls), name
        for f, _ in cls._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, f"{name}.{f}"


def good4():
    a = good()
    strides = (2 * 16 * 64, 16 * 64, 64)
    a["cache"] = N.KvCache(0x1000, 0x2000, 0x3000, 0x4000, strides, strides, (64, 32, 2), (64, 32, 2), N.KV_MX4, 8, 2, 16,
                           64, 0)
    a["rotated"] = N.KvRotated(0x1000, 0x2000, 0x3000, 0x4000, (256, 64), (128, 64), (128, 64), (256, 64), 0x5000, 0x6000,
                               0x7000, 0x8000, 0x9000, 0, N.KV_BF16, N.KV_BF16, 4, 64, 0, 1e-6)
    a["rows"] = N.KvRows(0x1000, 0x2000, 0x3000, 0, N.KV_BF16, 0)
    a["step"] = N.KvStep(0x1000, 4, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, 0x7000, 0x8000, 0x9000, 0xA000, 0xB000, 0xC000,
                         0xD000, 0xE000, 5, 2, 4, 8, 16)
    return a


def scratch(a):
    size = C.c_uint64(7)
    st = N.load().tessa_kv_attend_token_scratch(C.byref(a["cache"]), C.byref(a["seq"]), C.byref(a["attend"]),
                                                C.byref(size))
    return st.code, st.msg.decode()


@pytest.mark.parametrize("field,value,code,text", [
    ("head_dim", 48, 4, "multiple of 32"), ("head_dim", 16, 4, "multiple of 32"), ("head_dim", 288, 4, "head_dim"),
    ("key_scales", None, 1, "scales"), ("value_scales", None, 1, "scales"), ("key_strides", (2048, 1024, 48), 1, "16 bytes"),
    ("value_strides", (2**41, 1024, 64), 1, "stride"), ("value_scale_strides", (2**40, 32, 2), 1, "scale stride"),
    ("key_strides", (2**39, 1024, 64), 4, "64 GiB"), ("type", 7, 1, "unknown type"), ("type", 4, 1, "unknown type"),
    ("type", 6, 1, "unknown type")])
def test_caches_that_are_refused(field, value, code, text):
    a = good4()
    assert scratch(a) == (0, "")
    for kind in (N.KV_BF16, N.KV_F16):
        a["attend"].type = kind
        assert scratch(a)[0] == 0
    setattr(a["cache"], field, value)
    got = scratch(a)
    assert got[0] == code and text in got[1]


@pytest.mark.parametrize("field,value,code,text", [
    ("type", N.KV_SQ8, 1, "neither"), ("type", N.KV_F32, 1, "neither"), ("q_heads", 0, 1, "query heads"),
    ("rotated", 8, 1, "rotated"), ("rotated", 80, 1, "rotated"), ("rotated", 1 << 31, 1, "rotated"),
    ("frequencies", None, 1, "frequencies"), ("frequencies", 0x7004, 1, "frequencies"),
    ("weight_type", N.KV_F16, 1, "weights"), ("weight_type", 0, 1, "weights"), ("q_weight", 0x8008, 1, "weights"),
    ("k_weight", 0x8008, 1, "weights"), ("eps", -1.0, 1, "eps"), ("eps", float("nan"), 1, "eps"),
    ("eps", float("inf"), 1, "eps"), ("q", None, 1, "null q"), ("k", 0x2008, 1, "aligned"), ("v", None, 1, "null v"),
    ("out", None, 1, "null out"), ("out_strides", (256, 60), 1, "aligned"), ("positions", None, 1, "positions"),
    ("slots", None, 1, "slots"), ("tokens", 2**40, 4, "tokens"), ("tokens", 2**29, 4, "tokens")])
def test_rotated_append_refuses(field, value, code, text):
    a = good4()["rotated"]
    a.tokens = 3
    setattr(a, field, value)
    st = N.load().tessa_kv_append_rotated(C.byref(good4()["cache"]), C.byref(a), None)
    assert st.code == code and text in st.msg.decode()


def test_rotated_append_of_another_type_and_of_nothing():
    a = good4()
    lib = N.load()
    assert lib.tessa_kv_append_rotated(C.byref(a["cache"]), C.byref(a["rotated"]), None).code == 0  # no tokens
    plain = good()["cache"]
    a["rotated"].type = a["rotated"].weight_type = N.KV_F16
    st = lib.tessa_kv_append_rotated(C.byref(plain), C.byref(a["rotated"]), None)
    assert st.code == 1 and "type" in st.msg.decode()
    assert lib.tessa_kv_append_rotated(C.byref(plain), None, None).code == 1
    assert lib.tessa_kv_append_rotated(None, C.byref(a["rotated"]), None).code == 1


@pytest.mark.parametrize("field,value,code,text", [
    ("type", N.KV_SQ8, 1, "neither"), ("type", 0, 1, "neither"), ("slots", None, 1, "null"), ("k", None, 1, "null"),
    ("k", 0x2008, 1, "aligned"), ("v", 0x2008, 1, "aligned"), ("count", 2**30, 4, "rows"), ("count", 2**50, 4, "rows")])
def test_read_refuses(field, value, code, text):
    a = good4()
    lib = N.load()
    assert lib.tessa_kv_read(C.byref(a["cache"]), C.byref(a["rows"]), None).code == 0  # no rows
    a["rows"].count = 3
    setattr(a["rows"], field, value)
    st = lib.tessa_kv_read(C.byref(a["cache"]), C.byref(a["rows"]), None)
    assert st.code == code and text in st.msg.decode()
    assert lib.tessa_kv_read(C.byref(a["cache"]), None, None).code == 1


@pytest.mark.parametrize("field,value,code,text", [
    ("page_rows", 0, 1, "page_rows"), ("page_rows", 24, 1, "page_rows"), ("page_rows", 1 << 17, 1, "page_rows"),
    ("batch", 70000, 4, "batch"), ("pages", 1 << 31, 4, "pages"), ("columns", 1 << 31, 4, "columns"),
    ("tokens", 1 << 31, 4, "tokens"), ("table", None, 1, "null"), ("lengths", None, 1, "null"), ("held", None, 1, "null"),
    ("fresh", None, 1, "null"), ("free", None, 1, "null"), ("count", None, 1, "null"), ("new_lengths", None, 1, "null"),
    ("new_held", None, 1, "null"), ("new_count", None, 1, "null"), ("granted", None, 1, "null"),
    ("offsets", None, 1, "null"), ("positions", None, 1, "null"), ("sequences", None, 1, "null"),
    ("slots", None, 1, "null"), ("table_stride", 3, 1, "stride"), ("new_lengths", 0x2000, 1, "arguments"),
    ("new_held", 0x3000, 1, "arguments"), ("new_count", 0x6000, 1, "arguments")])
def test_plan_refuses(field, value, code, text):
    a = good4()["step"]
    setattr(a, field, value)
    st = N.load().tessa_kv_plan(C.byref(a), None)
    assert st.code == code and text in st.msg.decode()
    assert N.load().tessa_kv_plan(None, None).code == 1


def test_the_rule_of_4_bit_rows():
    """The tests' own rule, at values whose codes can be said."""
    x = np.zeros((1, 32))
    x[0, :12] = [6, 0.25, 0.75, -1.25, 1.75, 2.5, -3.5, 5, 0.2500001, 0.2499999, -0.1, 7 - 1e-9]
    code, e = mx4_rule(x)
    assert e[0, 0] == 127
    assert list(code[0, :12]) == [7, 0, 2, 10, 4, 4, 14, 6, 1, 0, 8, 7]
    x[0, 0] = 7.0  # rounds to 8 of the next binade: half as fine, 4
    code, e = mx4_rule(x)
    assert e[0, 0] == 128 and code[0, 0] == 6 and code[0, 7] == 4
    x[0, 3] = np.inf
    code, e = mx4_rule(x)
    assert e[0, 0] == 255 and (code == 0).all()
    code, e = mx4_rule(np.zeros((2, 64)))
    assert (e == 2).all() and (code == 0).all()
    code, e = mx4_rule(np.full((1, 32), 1.99 * 2.0**127))
    assert e[0, 0] == 252 and (code == 7).all()
    g = np.random.default_rng(1).standard_normal((50, 64))
    code, e = mx4_rule(g)
    v = mx4_values(pack(code), e)
    top = np.abs(g).reshape(50, 2, 32).max(-1).repeat(32, -1).reshape(50, 64)
    # half a step at most: between 4 and 6 it is 2 units, a unit at most top / 3.5
    assert (np.abs(v - g) <= top / 3.5 + 1e-12).all() and (np.abs(v) <= 12 / 7 * top + 1e-12).all()
