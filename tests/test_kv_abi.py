"""The paged key-value cache's C entry points on a machine without a GPU: struct
layouts, and arguments that are refused before any device work."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

from shear_amd import _native as N

HEADER = Path(__file__).resolve().parent.parent / "include" / "tessa_hip.h"
STRUCTS = {"tessa_kv_cache": N.KvCache, "tessa_kv_sequences": N.KvSequences, "tessa_kv_tokens": N.KvTokens,
           "tessa_kv_attend": N.KvAttend, "tessa_kv_eviction": N.KvEviction}


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


def good():
    """Arguments that would be accepted (addresses that nothing reads here)."""
    strides = (2 * 16 * 64, 16 * 64, 64)
    cache = N.KvCache(0x1000, 0x2000, 0x3000, 0x4000, strides, strides, (32, 16, 1), (32, 16, 1), N.KV_BF16, 8, 2, 16,
                      64, 0)
    seq = N.KvSequences(0x5000, 0x6000, 4, 2, 4, 64, 0)
    attend = N.KvAttend(0x7000, 0x8000, 0x9000, (256, 64), (256, 64), N.KV_BF16, 4, 0.125, 0, N.KV_ALL, 0, None, None,
                        (0, 0), None, 2, 0, 0)
    tokens = N.KvTokens(0x7000, 0x8000, (128, 64), (128, 64), None, 2, 1, N.KV_BF16)
    evict = N.KvEviction(0x7000, (128, 64), 0x8000, 0x9000, 0xA000, None, 0, 0, 64, 16, 2, 4, 0)
    return {"cache": cache, "seq": seq, "attend": attend, "tokens": tokens, "evict": evict}


def token_scratch(a):
    size = C.c_uint64(7)
    st = N.load().tessa_kv_attend_token_scratch(C.byref(a["cache"]), C.byref(a["seq"]), C.byref(a["attend"]),
                                                C.byref(size))
    return st, size.value


@pytest.mark.parametrize("what,field,value,code,text", [
    ("cache", "type", 0, 1, "unknown type"),
    ("cache", "type", 4, 1, "unknown type"),
    ("cache", "keys", None, 1, "null keys"),
    ("cache", "values", 0x2008, 1, "16-byte aligned"),
    ("cache", "key_strides", (2048, 1024, 65), 1, "multiple of 16 bytes"),
    ("cache", "value_strides", (2**40, 1024, 64), 1, "stride"),
    ("cache", "value_strides", (2**39, 1024, 64), 4, "64 GiB"),
    ("cache", "pages", 0, 1, "0 pages"),
    ("cache", "heads", 0, 1, "0 heads"),
    ("cache", "heads", 1025, 4, "1025 heads"),
    ("cache", "page_rows", 12, 1, "power of two"),
    ("cache", "page_rows", 0, 1, "power of two"),
    ("cache", "head_dim", 72, 4, "head_dim"),
    ("cache", "head_dim", 272, 4, "head_dim"),
    ("cache", "head_dim", 0, 4, "head_dim"),
    ("seq", "batch", 70000, 4, "batch"),
    ("seq", "lengths", None, 1, "null"),
    ("seq", "table", None, 1, "null"),
    ("seq", "table_stride", 3, 1, "stride"),
    ("seq", "max_length", 65, 1, "max_length"),
    ("attend", "type", N.KV_F16, 1, "type"),
    ("attend", "type", N.KV_SQ8, 1, "neither"),
    ("attend", "q_heads", 3, 1, "query heads"),
    ("attend", "q_heads", 0, 1, "query heads"),
    ("attend", "q_heads", 2 * 257, 4, "share one head"),
    ("attend", "scale", 0.0, 1, "scale"),
    ("attend", "scale", -1.0, 1, "scale"),
    ("attend", "scale", float("nan"), 1, "scale"),
    ("attend", "scale", float("inf"), 1, "scale"),
    ("attend", "q", None, 1, "null q"),
    ("attend", "q", 0x7002, 1, "aligned"),
    ("attend", "out_strides", (256, 60), 1, "aligned"),
    ("attend", "lse", None, 1, "lse"),
    ("attend", "tokens", 3, 1, "3 tokens"),
    ("attend", "listed_count", 5, 1, "go together"),
    ("attend", "offsets", 0x10, 1, "offsets"),
    ("attend", "sinks", 2**31, 1, "sinks"),
])
def test_attend_refuses(what, field, value, code, text):
    a = good()
    setattr(a[what], field, value)
    st, size = token_scratch(a)
    assert st.code == code and text in st.msg.decode() and size == 0


def test_attend_takes_what_is_right_and_wants_its_scratch():
    a = good()
    st, size = token_scratch(a)
    assert st.code == 0 and size == 0  # few rows: one workgroup a head, no partial results
    a["attend"].weights, a["attend"].weight_strides = 0xB000, (128, 64)
    st, size = token_scratch(a)
    assert st.code == 0 and size >= 2 * 4 * 64 * 4
    st = N.load().tessa_kv_attend_token(C.byref(a["cache"]), C.byref(a["seq"]), C.byref(a["attend"]), 0x1000, size - 1, None)
    assert st.code == 1 and "scratch" in st.msg.decode()
    st = N.load().tessa_kv_attend_token(C.byref(a["cache"]), C.byref(a["seq"]), C.byref(a["attend"]), 0x1008, size, None)
    assert st.code == 1 and "scratch" in st.msg.decode()
    a["attend"].listed, a["attend"].listed_count = 0x10, 5
    st, _ = token_scratch(a)
    assert st.code == 1 and "window" in st.msg.decode()
    a = good()
    a["cache"].type, a["cache"].key_scales = N.KV_SQ8, None
    assert "scales" in token_scratch(a)[0].msg.decode()
    for args in ((None, a["seq"], a["attend"]), (a["cache"], None, a["attend"]), (a["cache"], a["seq"], None)):
        st = N.load().tessa_kv_attend_token(*(C.byref(x) if x is not None else None for x in args), None, 0, None)
        assert st.code == 1


def test_prompt_append_and_evict_refuse():
    lib = N.load()
    a = good()

    def call(fn, key, **change):
        b = good()
        for k, v in change.items():
            setattr(b[key], k, v)
        extra = (None, 0, None) if key == "attend" else (None,)
        st = fn(C.byref(b["cache"]), C.byref(b["seq"]), C.byref(b[key]), *extra)
        return st.code, st.msg.decode()

    assert call(lib.tessa_kv_attend_prompt, "attend") == (1, "kv attend: null offsets")
    assert call(lib.tessa_kv_attend_prompt, "attend", offsets=0x10, weights=0x10)[0] == 1
    assert call(lib.tessa_kv_attend_prompt, "attend", offsets=0x10, listed=0x10, listed_count=2)[0] == 1
    for change in ({"type": N.KV_F16}, {"k": None}, {"v": 0x7004}, {"tokens": 3}, {"k_strides": (129, 64)}):
        code, text = call(lib.tessa_kv_append, "tokens", **change)
        assert code == 1 and text, change
    for change in ({"keep": 0}, {"keep": 5}, {"weights": None}, {"kept": None}, {"new_weights": 0x7000},
                   {"weight_rows": 15}, {"into": 0x10, "into_columns": 0, "into_stride": 0},
                   {"into": 0x10, "into_columns": 2, "into_stride": 1}):
        code, text = call(lib.tessa_kv_evict, "evict", **change)
        assert code == 1 and text, change
    # nothing to do: no device work, no error
    a["seq"].batch = 0
    a["tokens"].tokens = 0
    assert lib.tessa_kv_append(C.byref(a["cache"]), C.byref(a["seq"]), C.byref(a["tokens"]), None).code == 0
    assert lib.tessa_kv_evict(C.byref(a["cache"]), C.byref(a["seq"]), C.byref(a["evict"]), None).code == 0


@pytest.mark.parametrize("strides,right", [
    ((128, 64), True), ((64, 128), True), ((200, 70), True), ((0, 64), False), ((128, 0), False), ((64, 64), False),
    ((127, 64), False), ((64, 127), False), ((63, 256), False), ((0, 0), False), ((2**40, 64), False)])
def test_weights_that_share_a_place_are_refused(strides, right):
    # 2 sequences x 2 heads x 64 rows, each of them read, added to and written
    a = good()
    a["attend"].weights, a["attend"].weight_strides = 0xB000, strides
    st, _ = token_scratch(a)
    assert (st.code == 0) == right
    if not right:
        assert st.code == 1 and "weight strides" in st.msg.decode()


def test_weight_strides_of_a_single_sequence_or_head():
    a = good()
    a["attend"].weights, a["attend"].weight_strides = 0xB000, (0, 64)
    a["seq"].batch = a["attend"].tokens = 1
    assert token_scratch(a)[0].code == 0
    a["attend"].weight_strides = (0, 63)
    assert token_scratch(a)[0].code == 1
