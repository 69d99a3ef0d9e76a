"""Lists of whole numbers and of f32 that kernels read one by one start on any
multiple of four bytes (the plan's align record); vectors of a tensor's rows need 16."""
import ctypes

import pytest

from tcacomp_amd import _lib, attention
from tcacomp_amd.compiler import TensorDesc
from test_attention import attend_tensors, desc
from test_operators import compiled

PLAN = """tca-plan 1
program p
dim A 0
tensor x f32 in 1 A
tensor n i32 out 1 A
tensor w f32 local 1 A
%s
kernel k 256 0 1 A/256
arg ptr x
arg ptr n
end
"""


def parse(record):
    h = ctypes.c_void_p()
    return _lib.lib().tca_program_parse((PLAN % record).encode(), ctypes.byref(h)), h


def moved(tensors, i, by):
    t = tensors[i]
    return tensors[:i] + [TensorDesc(t.ptr + by, t.shape, t.dtype)] + tensors[i + 1:]


def programs():
    """(program, its tensors, the free dims, which of the tensors are lists)."""
    i = lambda *s: desc("i32", *s)  # noqa: E731
    table = [i(3), i(3), i(5), i(1), i(3, 6), i(4), i(3), i(7), i(7), i(1)]
    yield attention.page_table(), table, (16,), set(range(10))
    for elem in ("f32", "bf16"):
        x, k = desc(elem, 5, 4, 64), desc(elem, 9, 1, 16, 64)
        yield attention.rotary(elem), [x, i(5), desc("f32", 32), x], (), {1, 2}
        yield attention.rotary_cache(elem), [x, i(5), i(5), desc("f32", 32), desc(elem, 5, 1, 2, 64), k, k], (), {1, 2, 3}
    yield attention.paged_attention("bf16", stats=True), attend_tensors(stats=True), (), {3, 4, 5, 7}
    yield attention.paged_attention("f16", window=True), attend_tensors(elem="f16"), (7,), {3, 4, 5}


@pytest.mark.parametrize("n", range(7))
def test_lists_start_on_four_bytes(n):
    op, tensors, free, lists = list(programs())[n]
    p = compiled(op)
    assert p.check(tensors, free) == 0
    for t in range(len(tensors)):
        for by in (4, 8, 12):
            assert p.check(moved(tensors, t, by), free) == (0 if t in lists else _lib.TCA_ERR_INVALID), (op.name, t, by)
            if t not in lists:
                assert "16-byte aligned" in _lib.last_error()
        for by in (1, 2):
            assert p.check(moved(tensors, t, by), free) == _lib.TCA_ERR_INVALID, (op.name, t, by)
            assert ("4-byte aligned" if t in lists else "16-byte aligned") in _lib.last_error()


@pytest.mark.parametrize("bytes_", [4, 8, 16])
def test_record(bytes_):
    rc, h = parse("align n %d" % bytes_)
    assert rc == 0, _lib.last_error()
    text = _lib.lib().tca_program_plan_text(h).decode()
    assert ("align n %d" % bytes_ in text) == (bytes_ != 16) and "align x" not in text
    again = ctypes.c_void_p()
    assert _lib.lib().tca_program_parse(text.encode(), ctypes.byref(again)) == 0 and _lib.lib().tca_program_plan_text(again).decode() == text


@pytest.mark.parametrize("record", ["align", "align n", "align q 4", "align n 2", "align n 3", "align n 12", "align n 32", "align n 0", "align n x",
                                    "align n 4 4", "align w 4"])
def test_refused_records(record):
    rc, _ = parse(record)
    assert rc == _lib.TCA_ERR_INVALID
