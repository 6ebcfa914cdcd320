"""What the Python side hands to the prefix plan builder (no GPU)."""
import ctypes

import numpy as np
import pytest

from paged_decode import _native
from paged_decode.layout import Layout
from paged_decode.prefix import find_prefixes, inspect_prefix_plan

LAYOUT = Layout(5, 8, 2, 64, 16, 40)
TABLE = np.array([[0, 1, 2, 9, 10], [0, 1, 2, 11, 12], [3, 4, 13, 14, 15], [3, 4, 16, 17, 18], [0, 1, 2, 19, 20]])
LENGTHS = np.array([70, 80, 33, 60, 49])
GROUPS = [([0, 1, 4], 3), ([2, 3], 2)]


def described(prefixes, **kw):
    info, groups, items = inspect_prefix_plan(LAYOUT, TABLE, LENGTHS, prefixes=prefixes, **kw)
    return info, [(m.tolist(), p) for m, p in groups], items.tolist()


def test_prefixes_from_any_iterable():
    """The list is walked more than once."""
    want = described(GROUPS)
    assert want[1] == GROUPS
    assert described(iter(GROUPS)) == want
    assert described((m, p) for m, p in GROUPS) == want
    assert described(zip([m for m, _ in GROUPS], [p for _, p in GROUPS])) == want
    assert described((tuple(m), np.int32(p)) for m, p in GROUPS) == want


@pytest.mark.parametrize("pages", [2.7, 2.0, True, "2", None, np.float32(1), 2 + 0j])
def test_page_counts_are_integers(pages):
    """As members are: nothing is truncated."""
    with pytest.raises(TypeError, match="sequence indices, pages"):
        described([([0, 1], pages)])


def test_inspected_plans_check_max_lengths_as_plans_do():
    """Too few or misshapen ones do not reach the library, which reads one per sequence."""
    for bad in (LENGTHS[:3], LENGTHS[None], LENGTHS + 0.5, np.array(80), LENGTHS - 1, LENGTHS + 80,
                np.array([2 ** 32 + 80] * 5)):
        with pytest.raises(ValueError, match="max_lengths"):
            described(GROUPS, max_lengths=bad)
    assert described(GROUPS, max_lengths=[80, 80, 80, 80, 80])[0]["dynamic"] == 1


@pytest.mark.parametrize("three", [np.array(3), np.int64(3), np.uint8(3)])
def test_page_counts_of_any_integer_kind(three):
    assert described([([0, 1], three)])[1] == [([0, 1], 3)]


def test_types_by_name_or_as_torch_has_them():
    torch = pytest.importorskip("torch")
    for name in ("float16", "float32"):
        want = described(GROUPS, dtype=name)
        assert described(GROUPS, dtype=getattr(torch, name)) == want
        assert [(m.tolist(), p) for m, p in find_prefixes(LAYOUT, TABLE, LENGTHS, dtype=getattr(torch, name))] == GROUPS
    for bad in ("bfloat16", torch.bfloat16, None):
        with pytest.raises(TypeError, match="float16 or float32"):
            find_prefixes(LAYOUT, TABLE, LENGTHS, dtype=bad)


def test_group_counts_below_the_two_that_mean_something():
    lib = _native.load()
    layout = _native.Layout(5, 8, 2, 64, 16, 40)
    table, lengths = np.ascontiguousarray(TABLE, np.int32), np.ascontiguousarray(LENGTHS, np.int32)
    for count, status in ((-1, _native.PD_OK), (-2, _native.PD_OK), (-3, _native.PD_ERR_VALUE),
                          (-2 ** 31, _native.PD_ERR_VALUE)):
        handle = ctypes.c_void_p()
        got = lib.pd_prefix_plan_create(ctypes.byref(layout), table.ctypes.data, 5, lengths.ctypes.data, None, count,
                                        None, None, None, 0, -1, ctypes.byref(handle))
        assert got == status and bool(handle) == (status == _native.PD_OK)
        lib.pd_prefix_plan_destroy(handle)
