"""Dynamic shared-prefix launches: live lengths and tables that are not the ones planned with."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("NVIDIA GPU required", allow_module_level=True)

from paged_decode import _native
from paged_decode.layout import Layout
from paged_decode.prefix import SharedPrefixPlan

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def cuda(x):
    return torch.tensor(np.asarray(x, dtype=np.int32), device="cuda")


def tensors(layout, dtype, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    shape = (layout.physical_pages, layout.page_size, layout.kv_heads, layout.head_dim)
    q = torch.randn((layout.batch, layout.query_heads, layout.head_dim), device="cuda", dtype=dtype, generator=gen)
    return q, *(torch.randn(shape, device="cuda", dtype=dtype, generator=gen) for _ in range(2))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("others", [0, 2])
def test_a_length_past_a_plan_that_ends_with_its_prefixes_is_flagged(dtype, others):
    """No sequence has room behind its prefix (others: no room at all): one more live token is flagged, and
    the launch attends to the planned ones."""
    page, shared, sharers = 16, 2, 3
    batch = sharers + others
    table = np.full((batch, shared + 1), -1, dtype=np.int32)
    table[:sharers] = [0, 1, 2]
    lengths = np.array([shared * page] * sharers + [0] * others, dtype=np.int32)
    layout = Layout(batch, 8, 2, 64, page, 3)
    q, k, v = tensors(layout, dtype)
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=[(range(sharers), shared)], dtype=dtype,
                            max_lengths=lengths)
    want = plan.run(q, k, v).clone()
    assert plan.read_errors() == 0
    for b in range(batch):
        live = lengths.copy()
        live[b] += 1
        out = plan.run_dynamic(q, k, v, cuda(table), cuda(live))
        assert plan.read_errors() == _native.PD_DEVERR_LENGTH
        assert torch.equal(out, want)
    assert torch.equal(plan.run_dynamic(q, k, v, cuda(table), cuda(lengths)), want) and plan.read_errors() == 0


def exact(q, k, v, table, lengths):
    """Attention in 64 bits and the weights' average of |v|; tokens on pages outside the cache are left out."""
    B, H, D = q.shape
    P, page, kv = k.shape[:3]
    out, size = (torch.zeros((B, H, D), dtype=torch.float64) for _ in range(2))
    for b, n in enumerate(int(x) for x in lengths):
        at = np.arange(n)
        ids = np.asarray(table)[b, at // page].astype(np.int64)
        slots = torch.tensor((ids * page + at % page)[(ids >= 0) & (ids < P)], device="cuda")
        if len(slots) == 0:
            continue
        kk, vv = (x.flatten(0, 1)[slots].double().transpose(0, 1) for x in (k, v))
        w = torch.softmax(q[b].double().view(kv, -1, D) @ kk.mT / D ** 0.5, -1)
        out[b], size[b] = (w @ vv).view(H, D).cpu(), (w @ vv.abs()).view(H, D).cpu()
    return out, size


def close(got, want, size):
    """FP16: weights rounded to 2^-11 of themselves in numerator and denominator, one rounding at the store;
    scores and sums are FP32."""
    tol = 2e-5 * (size + want.abs()) + 1e-6
    if got.dtype == F16:
        tol = tol + 2.0 ** -11 * (1.05 * size + 2.1 * want.abs()) + 2.0 ** -24
    worst = ((got.cpu().double() - want).abs() - tol).max().item()
    assert worst <= 0, f"{worst:.3g} over the tolerance"     # NaN fails too


def serving_batch(sharers, shared, others, heads, kv, D, page, dtype, own=3, spare=60):
    """Sequences behind `shared` common pages with room for `own` pages more, others apart, and spare pages."""
    rng = np.random.default_rng(11)
    batch = sharers + others
    pages = shared + (batch * own + others * shared) + spare
    pool = list(rng.permutation(pages))
    common = [pool.pop() for _ in range(shared)]
    table = np.zeros((batch, shared + own), dtype=np.int32)
    for b in range(batch):
        head = common if b < sharers else [pool.pop() for _ in range(shared)]
        table[b] = head + [pool.pop() for _ in range(own)]
    lengths = (shared * page + rng.integers(0, own * page + 1, batch)).astype(np.int32)
    layout = Layout(batch, heads, kv, D, page, pages)
    return layout, table, lengths, np.array(pool, dtype=np.int32), *tensors(layout, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,kv,D,page", [(32, 8, 128, 16), (6, 6, 64, 32), (1, 1, 64, 16), (32, 1, 128, 32)])
def test_pages_that_move_under_a_plan(dtype, heads, kv, D, page):
    """The live table counts, as in DecodePlan.run_dynamic, also where a sequence no longer starts with the
    plan's shared pages: a page copied elsewhere, another sequence in the slot, a page outside the cache."""
    shared, sharers = 9, 12
    layout, table, lengths, spare, q, k, v = serving_batch(sharers, shared, 3, heads, kv, D, page, dtype)
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=[(range(sharers), shared)], dtype=dtype,
                            max_lengths=np.full(layout.batch, table.shape[1] * page))

    def run(live_table, live, flags=0):
        out = plan.run_dynamic(q, k, v, cuda(live_table), cuda(live))
        close(out, *exact(q, k, v, live_table, live))
        assert plan.read_errors() == flags
        return out.clone()

    before = run(table, lengths)
    for moved in ([0], [shared - 1], [4], [2, 7], list(range(shared))):
        live = table.copy()
        live[5, moved] = spare[: len(moved)]
        after = run(live, lengths)
        same = [b for b in range(layout.batch) if b != 5]
        assert torch.equal(after[same], before[same]) and not torch.equal(after[5], before[5])
    slot = table.copy()                              # other sequences in two slots, one longer, one shorter
    slot[3], slot[8] = spare[:shared + 3], spare[12:12 + shared + 3]
    live = lengths.copy()
    live[3], live[8], live[1], live[2] = table.shape[1] * page, 2 * page + 5, 0, shared * page
    run(slot, live)
    slot[1] = -1                                     # not in use: its row may hold anything
    run(slot, live)
    everyone = table.copy()                          # the whole group behind another prefix
    everyone[:sharers, :shared] = spare[20:20 + shared]
    run(everyone, lengths)
    for bad in (-1, layout.physical_pages, np.iinfo(np.int32).max):
        broken = table.copy()
        broken[4, 3] = bad
        run(broken, lengths, _native.PD_DEVERR_BAD_PAGE)
    assert torch.equal(run(table, lengths), before)


def test_found_groups_follow_the_live_table_too():
    """The caller named no groups: a slot that another sequence took over still gets its own attention."""
    sharers, shared, page = 48, 128, 16
    layout, table, lengths, spare, q, k, v = serving_batch(sharers, shared, 0, 32, 8, 128, page, F16, spare=200)
    plan = SharedPrefixPlan(layout, table, lengths, max_lengths=lengths)
    assert len(plan.prefixes) == 1
    live = table.copy()
    live[7, :shared + 3] = spare[: shared + 3]
    out = plan.run_dynamic(q, k, v, cuda(live), cuda(lengths))
    close(out, *exact(q, k, v, live, lengths))
    assert plan.read_errors() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("sharers,shared", [(6, 700), (40, 70)])
def test_lengths_at_every_cut_of_a_prefix(dtype, sharers, shared):
    """Live lengths around the ends of pieces, steps and pages, a sequence each."""
    page = 16
    layout, table, lengths, _, q, k, v = serving_batch(sharers, shared, 1, 8, 2, 64, page, dtype)
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=[(range(sharers), shared)], dtype=dtype,
                            max_lengths=np.full(layout.batch, table.shape[1] * page))
    rng = np.random.default_rng(5)
    for _ in range(6):
        live = lengths.copy()
        cuts = rng.integers(0, shared + 1, sharers) * page + rng.choice([-17, -3, -1, 0, 1, 5, 15], sharers)
        live[:sharers] = np.clip(cuts, 0, table.shape[1] * page)
        moved = table.copy()
        moved[rng.integers(0, sharers), rng.integers(0, shared)] = table[sharers, 0]       # and a page that moved
        out = plan.run_dynamic(q, k, v, cuda(moved), cuda(live))
        close(out, *exact(q, k, v, moved, live))
        assert plan.read_errors() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_length_inside_a_long_prefix_costs_a_piece_of_it(dtype):
    """One sequence a token short of 49152: the pieces before its last one serve it too.  (Token by token over
    the whole prefix the step took more than a hundred times as long as planned.)"""
    page, shared = 32, 1536
    layout, table, lengths, _, q, k, v = serving_batch(8, shared, 0, 32, 8, 128, page, dtype)
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=[(range(8), shared)], dtype=dtype, max_lengths=lengths)
    short = lengths.copy()
    short[2] = shared * page - 1
    times = {}
    for name, live in (("planned", cuda(lengths)), ("short", cuda(short))):
        live_table, begin, end = cuda(table), *(torch.cuda.Event(enable_timing=True) for _ in range(2))
        plan.run_dynamic(q, k, v, live_table, live)
        times[name] = 1e9
        for _ in range(5):
            begin.record()
            out = plan.run_dynamic(q, k, v, live_table, live)
            end.record()
            end.synchronize()
            times[name] = min(times[name], begin.elapsed_time(end))
    close(out[2:3], *exact(q[2:3], k, v, table[2:3], short[2:3]))
    assert times["short"] < 25 * times["planned"], times


@pytest.mark.parametrize("heads,kv,sharers", [(10, 2, 60), (4, 4, 140), (2, 1, 67), (21, 7, 45)])
@pytest.mark.parametrize("page", [16, 32])
def test_every_page_of_every_row_tile_is_looked_at(heads, kv, sharers, page):
    """Members with few rows, and ones whose rows lie in two tiles: one page at a time moves for one of them."""
    shared, D = 11, 64
    layout, table, lengths, spare, q, k, v = serving_batch(sharers, shared, 0, heads, kv, D, page, F16)
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=[(range(sharers), shared)],
                            max_lengths=np.full(layout.batch, table.shape[1] * page))
    before = plan.run_dynamic(q, k, v, cuda(table), cuda(lengths)).clone()
    group = heads // kv
    edges = {m for m in range(sharers) if m * group // 128 != ((m + 1) * group - 1) // 128}
    for m in sorted(edges | {0, sharers - 1}):
        for p in range(shared):
            live = table.copy()
            live[m, p] = spare[p]
            out = plan.run_dynamic(q, k, v, cuda(live), cuda(lengths))
            close(out[m:m + 1], *exact(q[m:m + 1], k, v, live[m:m + 1], lengths[m:m + 1]))
            same = np.arange(sharers) != m
            assert torch.equal(out[same], before[same]) and not torch.equal(out[m], before[m])
    assert plan.read_errors() == 0
