"""Which of the found groups a plan uses (no GPU)."""
import numpy as np
import pytest

from paged_decode.layout import Layout
from paged_decode.prefix import find_prefixes, inspect_prefix_plan


def batch(counts, own, heads=32, kv=8, D=128, page=16):
    """counts: (groups, members of each, shared pages); every sequence has `own` pages behind its prefix."""
    rows, pool = [], 0
    for groups, members, pages in counts:
        for _ in range(groups):
            shared = list(range(pool, pool + pages))
            pool += pages
            for _ in range(members):
                rows.append(shared + list(range(pool, pool + own)))
                pool += own
    width = max(map(len, rows))
    table = np.array([r + [-1] * (width - len(r)) for r in rows], dtype=np.int32)
    lengths = np.array([len(r) * page for r in rows], dtype=np.int32)
    return Layout(len(rows), heads, kv, D, page, pool), table, lengths


@pytest.mark.parametrize("pairs", [1, 8, 64, 80, 500])
@pytest.mark.parametrize("dtype,members,pages", [("float16", 64, 256), ("float16", 256, 64), ("float16", 8, 4096),
                                                 ("float32", 64, 256), ("float32", 256, 64)])
def test_short_shared_runs_do_not_cost_a_long_one(dtype, pairs, members, pages):
    """Pairs of sequences with one page in common, beside a group that saves thousands of page reads."""
    layout, table, lengths = batch([(1, members, pages)], 3)
    alone, groups, _ = inspect_prefix_plan(layout, table, lengths, dtype=dtype)
    assert alone["groups"] == 1 and groups[0][1] == pages
    layout, table, lengths = batch([(1, members, pages), (pairs, 2, 1)], 3)
    assert len(find_prefixes(layout, table, lengths)) == 1 + pairs
    info, groups, items = inspect_prefix_plan(layout, table, lengths, dtype=dtype)
    assert any(len(m) == members and p == pages for m, p in groups)
    assert info["shared_pages"] >= (members - 1) * pages
    if dtype == "float16":
        # one-page pairs are not worth a CTA per KV head: the SMs stay with the suffixes
        assert info["items"] < alone["items"] + 8 * 8 and (info["suffix_ctas"] > 0) == (alone["suffix_ctas"] > 0)


def test_several_long_groups_are_all_used():
    layout, table, lengths = batch([(4, 48, 256), (60, 2, 1)], 2)
    info, groups, _ = inspect_prefix_plan(layout, table, lengths)
    assert sum(len(m) == 48 and p == 256 for m, p in groups) == 4


def test_nothing_is_shared_where_nothing_pays():
    layout, table, lengths = batch([(60, 2, 1)], 2)
    assert inspect_prefix_plan(layout, table, lengths)[0]["groups"] == 0
    assert len(find_prefixes(layout, table, lengths)) == 60
