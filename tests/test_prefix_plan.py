"""Prefix groups and the plans behind them, on the host (no GPU)."""
import ctypes

import numpy as np
import pytest

from paged_decode import _native
from paged_decode.layout import Layout
from paged_decode.prefix import _native_plan, find_prefixes, inspect_prefix_plan
from paged_decode.workload import config2


def saved(groups):
    return sum((len(m) - 1) * p for m, p in groups)


def best_saving(rows, depth=0):
    """The most that disjoint groups save, each of all rows with some leading pages: by trying every depth."""
    classes = {}
    for r in rows:
        if len(r) > depth:
            classes.setdefault(r[depth], []).append(r)
    return sum(max((len(c) - 1) * (depth + 1), best_saving(c, depth + 1)) for c in classes.values())


@pytest.mark.parametrize("seed", range(30))
def test_found_groups_are_valid_and_save_the_most_pages(seed):
    rng = np.random.default_rng(seed)
    B, page, width = int(rng.integers(1, 8)), 16, 6
    # pages from a small alphabet per depth, so that rows share leading pages at several depths
    table = rng.integers(0, 2, (B, width)) + 2 * np.arange(width)
    lengths = rng.integers(0, width * page + 1, B)
    layout = Layout(B, 8, 2, 64, page, 2 * width)
    groups = find_prefixes(layout, table, lengths)
    seen = [int(b) for m, _ in groups for b in m]
    assert len(seen) == len(set(seen))
    for members, pages in groups:
        assert len(members) > 1 and pages >= 1
        assert (lengths[members] >= pages * page).all()
        assert (table[members, :pages] == table[members[0], :pages]).all()
    rows = [tuple(table[b, : lengths[b] // page]) for b in range(B)]
    assert saved(groups) == best_saving(rows)


def test_finds_the_shared_pages_of_the_ragged_workload():
    w = config2()
    groups = find_prefixes(w.layout, w.table, w.lengths)
    assert len(groups) == 1 and groups[0][1] == w.notes["prefix_pages"]
    assert groups[0][0].tolist() == w.notes["shared_prefix"]


def test_native_refusals():
    layout = Layout(3, 8, 2, 64, 16, 8)
    table, lengths = np.array([[0, 1, 2], [0, 1, 3], [4, 5, 6]]), np.array([48, 40, 48])
    for prefixes, message in (([([0, 1], 3)], "longer than"), ([([0, 2], 1)], "share its pages"),
                              ([([0, 1], 1), ([1], 1)], "one prefix group only"), ([([], 1)], "at least one"),
                              ([([0, 1], 4)], "table width"), ([([0, 3], 1)], "outside the batch")):
        with pytest.raises(ValueError, match=message):
            _native_plan(layout, table, lengths, prefixes, None, 0, -1)
    with pytest.raises(ValueError, match="max_lengths"):
        _native_plan(layout, table, lengths, [], lengths - 1, 0, -1)
    with pytest.raises(ValueError, match="outside physical cache"):
        _native_plan(layout, table + 8, lengths, [], None, 0, -1)
    lib = _native.load()
    handle = _native_plan(layout, table, lengths, [([0, 1], 2)], None, 0, -1)
    try:
        assert lib.pd_prefix_plan_bind(handle, 256, 1 << 30, None) == _native.PD_ERR_VALUE
        assert lib.pd_prefix_decode(handle, 16, 16, 16, 0, 16, None) == _native.PD_ERR_VALUE
        assert lib.pd_prefix_decode_dynamic(handle, 16, 16, 16, 0, 16, 16, 16, None) == _native.PD_ERR_VALUE
        word = ctypes.c_uint32(7)
        assert lib.pd_prefix_plan_read_errors(handle, ctypes.byref(word), None) == _native.PD_ERR_UNBOUND
    finally:
        lib.pd_prefix_plan_destroy(handle)
    assert lib.pd_prefix_plan_create(None, None, 0, None, None, -1, None, None, None, 0, -1, None) == _native.PD_ERR_VALUE
    assert lib.pd_prefix_plan_device_bytes(None) == 0
    lib.pd_prefix_plan_destroy(None)


def test_rotary_entry_points_refuse_bad_arguments():
    """Everything that the library checks before it touches a GPU."""
    lib = _native.load()
    rotation = _native.Rotation(64, 64, 0, 1e-6, 16, 4096, None, None)
    rows = _native.Heads(4096, 64, 64, 4096, 64, 64, 1)
    layout = _native.Layout(2, 1, 1, 64, 16, 4)
    V, T = _native.PD_ERR_VALUE, _native.PD_ERR_TYPE

    def rotate(r=rotation, q=rows, tokens=2, positions=4096, dtype=0, error=4096):
        ref = lambda x: None if x is None else ctypes.addressof(x)  # noqa: E731
        return lib.pd_rotate_heads(ref(r), ref(q), None, tokens, positions, dtype, error, 0, None)

    assert rotate(r=None) == V and rotate(dtype=7) == T and rotate(tokens=-1) == V and rotate(error=None) == V
    assert rotate(positions=None) == V and rotate(positions=4097) == V and rotate(tokens=0) == 0 and rotate(error=4098) == V
    for field, value in (("head_dim", 96), ("rotary_dim", 8), ("rotary_dim", 80), ("rotary_dim", 40),
                         ("max_positions", 0), ("table", 4100), ("q_weight", 4100), ("eps", -1.0), ("eps", float("nan"))):
        bad = _native.Rotation.from_buffer_copy(rotation)
        setattr(bad, field, value)
        assert rotate(r=bad) == V, field
    for field, value in (("heads", -1), ("heads", 65536), ("data", None), ("data", 4097), ("out", None)):
        bad = _native.Heads.from_buffer_copy(rows)
        setattr(bad, field, value)
        assert rotate(q=bad) == V, field

    def append(l=layout, k=rows, v=rows, tokens=2, cache=4096, dtype=0, table=4096, width=2, lengths=4096, indptr=None):
        ref = lambda x: None if x is None else ctypes.addressof(x)  # noqa: E731
        return lib.pd_cache_append(ref(l), None, None, ref(k), ref(v), tokens, cache, cache, dtype, table, width,
                                   lengths, indptr, 4096, 0, None)

    two = _native.Heads.from_buffer_copy(rows)
    two.heads = 2
    assert append(l=None) == V and append(k=None) == V and append(k=two) == V and append(v=two) == V
    assert append(tokens=3) == V and append(cache=None) == V and append(cache=4100) == V and append(dtype=2) == T
    assert append(table=None) == V and append(width=0) == V and append(lengths=4098) == V and append(indptr=4098) == V
    assert append(tokens=0, indptr=4096) == 0
    for field, value in (("batch", 0), ("page_size", 8), ("head_dim", 80), ("physical_pages", 0), ("kv_heads", 0)):
        bad = _native.Layout.from_buffer_copy(layout)
        setattr(bad, field, value)
        assert append(l=bad) == V, field


def shared_batch(counts, others, heads, kv, page, D=64):
    """A table of groups with (members, pages) and other sequences of one page."""
    rows, lengths, members, pool = [], [], [], 0
    for n, pages in counts:
        shared = list(range(pool, pool + pages))
        pool += pages
        members.append((list(range(len(rows), len(rows) + n)), pages))
        for _ in range(n):
            rows.append(shared)
            lengths.append(pages * page)
    for _ in range(others):
        rows.append([pool])
        pool += 1
        lengths.append(3)
    width = max(map(len, rows))
    table = np.full((len(rows), width), -1, dtype=np.int32)
    for b, r in enumerate(rows):
        table[b, :len(r)] = r
    return Layout(len(rows), heads, kv, D, page, max(pool, 1)), table, np.array(lengths), members


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("heads,kv,page", [(32, 8, 16), (32, 1, 32), (40, 8, 32), (64, 2, 16), (6, 6, 32)])
@pytest.mark.parametrize("counts,others", [([(1, 1)], 0), ([(4, 64)], 3), ([(3, 5), (70, 33), (2, 200)], 1),
                                           ([(400, 20)], 0), ([(64, 512)], 0), ([(2, 4000)], 5)])
def test_work_items_cover_every_row_and_page_once(dtype, heads, kv, page, counts, others):
    layout, table, lengths, members = shared_batch(counts, others, heads, kv, page)
    info, groups, items = inspect_prefix_plan(layout, table, lengths, prefixes=members, dtype=dtype)
    assert len(items) == info["items"] and info["members"] == sum(n for n, _ in counts)
    rows_per_tile, seen, slots = info["tile_rows"], {}, []
    first_member, first_page = 0, 0
    starts = {}                                      # the group of a first member
    for g, (n, pages) in enumerate(counts):
        starts[first_member] = (g, first_page)
        first_member, first_page = first_member + n, first_page + pages
    streams = []                                     # (group, head, tile, first, end, slot)
    for it in items:
        it = [int(x) for x in it]
        g, page0 = starts[it[0]]
        assert it[1] == counts[g][0] and it[4] == page0
        if info["item_words"] == 8:
            streams.append((g, it[2], it[3], it[5], it[6], it[7]))
            continue
        a, b = it[8:12], it[12:16]
        if it[3] == 1:                               # two tiles, one run
            assert b[0] == a[0] + 1 and a[1:3] == b[1:3]
        else:                                        # one tile, the longer run first
            assert a[0] == b[0] and a[2] - a[1] >= b[2] - b[1]
        streams += [(g, it[2], *x) for x in (a, b) if x[2] > x[1]]
    for g, head, tile, first, end, slot in streams:
        assert 0 <= first < end <= counts[g][1] and 0 <= head < kv
        for p in range(first, end):
            key = (g, head, tile, p)
            assert key not in seen
            seen[key] = 1
        slots.append(slot)
    want = sum(kv * -(-n * (heads // kv) // rows_per_tile) * pages for n, pages in counts)
    assert len(seen) == want
    assert sorted(slots) == list(range(len(slots)))
    if info["suffix_ctas"]:                          # the two kernels' CTAs are all resident at once
        assert info["suffix_launch"] and info["suffix_ctas"] + info["items"] <= 148


def test_sharing_is_left_out_where_it_saves_little():
    layout, table, lengths, members = shared_batch([(8, 64)], 2, 32, 8, 16, D=128)
    assert inspect_prefix_plan(layout, table, lengths)[0]["groups"] == 0
    assert inspect_prefix_plan(layout, table, lengths, prefixes=members)[0]["groups"] == 1
    layout, table, lengths, members = shared_batch([(64, 256)], 2, 32, 8, 16, D=128)     # 63 * 256 * 64 KiB saved
    info, groups, _ = inspect_prefix_plan(layout, table, lengths)
    assert info["groups"] == 1 and groups[0][1] == 256 and info["shared_pages"] == 63 * 256
