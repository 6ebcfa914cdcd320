"""A NaN or an infinite score in a live row, wherever the row's work was cut: the row is NaN, others are untouched.

A row's tokens are cut over CTAs, over the sub-pipelines of a CTA and between a shared prefix and the rest;
no cut may lose a part that holds a NaN.  Expected: attention in 64 bits, where a score of +infinity or NaN
makes the softmax NaN and one of -infinity has weight 0.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("NVIDIA GPU required", allow_module_level=True)

from paged_decode.layout import Layout
from paged_decode.prefix import SharedPrefixPlan
from paged_decode.runtime import DecodePlan

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
SHAPES = [(32, 8, 128, 16), (8, 2, 64, 32), (6, 6, 64, 16), (32, 1, 128, 32), (32, 1, 64, 16), (12, 1, 128, 16)]


def batch(lengths, shared, heads, kv, D, page, dtype):
    """Sequences whose first `shared` pages are the same, pages at random."""
    rng = np.random.default_rng(3)
    lengths = np.array(lengths, dtype=np.int32)
    need = -(-lengths // page)
    pool = list(rng.permutation(int(np.maximum(need - shared, 0).sum()) + shared))
    first = [pool.pop() for _ in range(shared)]
    table = np.full((len(lengths), int(need.max())), -1, dtype=np.int32)
    for b, n in enumerate(need):
        row = (first + [pool.pop() for _ in range(n - shared)]) if n > shared else first[:n]
        table[b, :n] = row
    pages = shared + int(np.maximum(need - shared, 0).sum())
    gen = torch.Generator("cuda").manual_seed(3)
    q = torch.randn((len(lengths), heads, D), device="cuda", dtype=dtype, generator=gen)
    k, v = (torch.randn((pages, page, kv, D), device="cuda", dtype=dtype, generator=gen) for _ in range(2))
    return Layout(len(lengths), heads, kv, D, page, pages), table, lengths, q, k, v


def nan_rows(q, k, table, b, n):
    """Which heads of sequence b are NaN in 64 bits, [heads]."""
    kv, page = k.shape[2], k.shape[1]
    pages = torch.tensor(table[b, : -(-n // page)].astype(np.int64), device="cuda")
    kk = k[pages].flatten(0, 1)[:n].double().transpose(0, 1)
    scores = (q[b].double().view(kv, -1, q.shape[2])[:, :, None] * kk[:, None]).sum(-1)
    return torch.softmax(scores, -1).isnan().any(-1).flatten()


def check(plan, q, k, v, table, lengths, where, value):
    """`value` into one key element of (sequence, token) at a time."""
    clean = plan.run(q, k, v).clone()
    assert not clean.isnan().any()
    for b, t in where:
        row = (int(table[b, t // k.shape[1]]), t % k.shape[1], k.shape[2] - 1, 5)
        kept = k[row].item()
        k[row] = value
        out = plan.run(q, k, v)
        for s, n in enumerate(int(x) for x in lengths):
            want = nan_rows(q, k, table, s, n)
            got = out[s].isnan()
            assert torch.equal(got.all(-1), want) and torch.equal(got.any(-1), want), (b, t, s)
        k[row] = kept
    assert torch.equal(plan.run(q, k, v), clean) and plan.read_errors() == 0


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,kv,D,page", SHAPES)
@pytest.mark.parametrize("lengths", [[2900, 333, 1], [40, 17, 9, 1], [3000]])
def test_in_a_decode_plan(value, dtype, heads, kv, D, page, lengths):
    layout, table, lengths, q, k, v = batch(lengths, 0, heads, kv, D, page, dtype)
    where = [(0, t) for t in sorted({int(x) for x in np.linspace(0, lengths[0] - 1, 14)})]
    check(DecodePlan(layout, table, lengths), q, k, v, table, lengths, where, value)


@pytest.mark.parametrize("heads,kv,D,page", [(32, 1, 128, 32), (32, 1, 64, 16)])
def test_in_a_pair_plan(heads, kv, D, page):
    """Sequences about equally long, two CTAs each."""
    layout, table, lengths, q, k, v = batch([700] * 64, 0, heads, kv, D, page, F16)
    plan = DecodePlan(layout, table, lengths)
    check(plan, q, k, v, table, lengths, [(0, 0), (9, 340), (30, 500), (63, 699)], float("nan"))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,kv,D,page", SHAPES)
@pytest.mark.parametrize("share", [True, False])
def test_in_a_shared_prefix_plan(value, dtype, heads, kv, D, page, share):
    shared = 12
    first = shared * page
    layout, table, lengths, q, k, v = batch([first + 2500, first + 60, first, first + 1], shared, heads, kv, D, page, dtype)
    plan = SharedPrefixPlan(layout, table, lengths, dtype=dtype, prefixes=[(range(4), shared)] if share else [])
    where = [(0, t) for t in sorted({int(x) for x in np.linspace(first, lengths[0] - 1, 10)})]
    where += [(0, 0), (0, first - 1), (1, first), (1, first + 59), (3, first)]
    check(plan, q, k, v, table, lengths, where, value)


def test_in_one_shard_of_several():
    """The merge of sequence shards: row 0 is NaN in one shard, row 1 empty in another, row 2 empty in all."""
    from paged_decode import _native
    lib, shards, rows, D = _native.load(), 3, 3, 128
    packed = torch.rand((shards, rows * (D + 2)), device="cuda")
    out, stats = packed[:, : rows * D].view(shards, rows, D), packed[:, rows * D:].view(shards, rows, 2)
    stats[..., 1] += 1
    out[1, 0], stats[1, 0, 1] = float("nan"), float("nan")
    for s, r in ((0, 1), (0, 2), (1, 2), (2, 2)):
        out[s, r], stats[s, r] = 0.0, torch.tensor([float("-inf"), 0.0])
    merged = torch.empty((rows, D), device="cuda")
    _native.check(lib.pd_merge_shards(packed.data_ptr(), packed.data_ptr() + rows * D * 4, shards, rows * (D + 2), rows,
                                      D, merged.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert merged[0].isnan().all() and (merged[2] == 0).all()
    w = (torch.exp2(stats[1:, 1, 0].double()) * stats[1:, 1, 1])[:, None]
    torch.testing.assert_close(merged[1].double(), (w * out[1:, 1]).sum(0) / w.sum(), atol=1e-6, rtol=0)
