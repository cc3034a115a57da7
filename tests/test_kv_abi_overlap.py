"""Arrays of the plan of a step that lie in each other's memory are refused before any device work: workgroups read the
arguments while others write the results."""
import ctypes as C

import pytest

from shear_amd import _native as N
from test_kv_abi_step import good4

# bytes of each array of good4()'s step: 2 sequences, 4 columns, 8 pages, 5 places
READ = {"lengths": 8, "held": 8, "fresh": 8, "count": 4}
WRITTEN = {"table": 32, "free": 32, "new_lengths": 8, "new_held": 8, "new_count": 4, "granted": 8, "offsets": 12, "positions": 20,
           "sequences": 20, "slots": 40}
SIZES = {**READ, **WRITTEN}


def refusal(step):
    """(code, message); nothing runs on a machine without a GPU, where a call that is not refused ends at its launch."""
    st = N.load().tessa_kv_plan(C.byref(step), None)
    return st.code, st.msg.decode()


def refused(step):
    code, text = refusal(step)
    return code == 1 and "arguments" in text


@pytest.mark.parametrize("a", list(WRITTEN))
@pytest.mark.parametrize("b", list(SIZES))
def test_arrays_that_overlap_are_refused(a, b):
    if a == b:
        return
    step = good4()["step"]
    at = getattr(step, b)
    if SIZES[a] <= SIZES[b]:
        places = {at, at + SIZES[b] - SIZES[a], at + SIZES[b] - 4}
    else:
        places = {at, at + SIZES[b] - 4, at - SIZES[a] + 4}
    for place in sorted(places):
        setattr(step, a, place)
        assert refused(step), (a, b, hex(place))


def launched(step):
    """Whether a step passes every check (its launch fails without a GPU; with one it must not run: its pointers are made up)."""
    return refusal(step)[0] != 1


@pytest.fixture
def no_gpu():
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("made-up pointers: only where nothing can run")


def test_arguments_may_share_memory(no_gpu):
    step = good4()["step"]
    step.held = step.fresh = step.count = step.lengths
    assert launched(step)


@pytest.mark.parametrize("a", list(WRITTEN))
@pytest.mark.parametrize("b", list(SIZES))
def test_arrays_side_by_side_are_taken(no_gpu, a, b):
    if a == b:
        return
    for place in (getattr(good4()["step"], b) + SIZES[b], getattr(good4()["step"], b) - SIZES[a]):
        step = good4()["step"]
        setattr(step, a, place)
        assert launched(step), (a, b)


def test_between_the_rows_of_a_table(no_gpu):
    """A table's row may lie in a wider row that holds other arrays too."""
    step = good4()["step"]
    step.table_stride = 16  # 64 bytes, 16 of them the row's
    step.lengths, step.new_lengths, step.granted = step.table + 16, step.table + 24, step.table + 64 + 16
    assert launched(step)
    for place in (step.table + 8, step.table + 12, step.table + 60, step.table + 64, step.table + 76):
        step.new_lengths = place
        assert refused(step), hex(place)


def test_arrays_of_no_size(no_gpu):
    """What is not written or read may be anything."""
    step = good4()["step"]
    step.tokens, step.pages = 0, 0
    step.positions = step.sequences = step.slots = step.free = step.lengths
    assert launched(step)
    step.batch = 0
    step.table = step.lengths = step.held = step.fresh = step.new_lengths = step.new_held = step.granted = step.count
    assert launched(step)
