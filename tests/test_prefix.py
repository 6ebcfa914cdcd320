"""Shared-prefix decode against attention in 64 bits.

Tolerances, from the arithmetic: with A = sum p |v| (the weights' average of
|v|), rounding each weight to FP16 moves a row by at most 2^-11 (A + |o|), and
the FP16 store by 2^-11 |o| more; scores and sums are FP32 (below 2e-5 of A
here).  FP32 plans have only the latter: products of D terms are off by a few
2^-24 of their terms' sum, which reaches the weights through the exponential.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("NVIDIA GPU required", allow_module_level=True)

from paged_decode.layout import Layout
from paged_decode.prefix import SharedPrefixPlan
from paged_decode.rotary import CacheAppend, HeadRotation, rotation_table
from paged_decode.runtime import DecodePlan

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def case(groups, others, heads, kv, D, page, dtype, seed=0, reserve=0, spare=3, extra_columns=0):
    """groups: [(prefix pages, [suffix lengths])], others: lengths.  Sequences in a shuffled order, pages
    at random, rows that no sequence sees filled with NaN and infinities."""
    rng = np.random.default_rng(seed)
    seqs = [(g, p * page + n) for g, (p, ns) in enumerate(groups) for n in ns] + [(-1, n) for n in others]
    seqs = [seqs[i] for i in rng.permutation(len(seqs))]
    lengths = np.array([n for _, n in seqs], dtype=np.int32)
    need = -(-(lengths + reserve) // page)
    width = max(1, int(need.max())) + extra_columns
    first = np.array([groups[g][0] if g >= 0 else 0 for g, _ in seqs])
    pages = sum(p for p, _ in groups) + int(np.maximum(need - first, 0).sum()) + spare
    pool = list(rng.permutation(pages))
    shared = [[pool.pop() for _ in range(p)] for p, _ in groups]
    table = np.full((len(seqs), width), -1, dtype=np.int32)
    live = torch.zeros((pages, page), dtype=torch.bool)
    for b, (g, n) in enumerate(seqs):
        if g >= 0:
            table[b, :first[b]] = shared[g]
        for i in range(first[b], need[b]):
            table[b, i] = pool.pop()
        for t in range(n):
            live[table[b, t // page], t % page] = True
    layout = Layout(len(seqs), heads, kv, D, page, pages)
    gen = torch.Generator("cuda").manual_seed(seed)
    q = torch.randn((len(seqs), heads, D), device="cuda", dtype=dtype, generator=gen)
    k, v = (torch.randn((pages, page, kv, D), device="cuda", dtype=dtype, generator=gen) for _ in range(2))
    dead = (~live).cuda()
    k[dead], v[dead] = float("nan"), float("inf")
    members = [([b for b, (h, _) in enumerate(seqs) if h == g], p) for g, (p, _) in enumerate(groups)]
    return layout, table, lengths, members, q, k, v


def exact(q, k, v, table, lengths):
    """(attention in 64 bits, the weights' average of |v|)."""
    B, H, D = q.shape
    kv, page = k.shape[2], k.shape[1]
    out, size = torch.zeros((B, H, D), dtype=torch.float64), torch.zeros((B, H, D), dtype=torch.float64)
    for b, n in enumerate(int(x) for x in lengths):
        if n == 0:
            continue
        pages = torch.tensor(table[b, : -(-n // page)].astype(np.int64), device="cuda")
        kk, vv = (x[pages].flatten(0, 1)[:n].double().transpose(0, 1) for x in (k, v))
        w = torch.softmax(q[b].double().view(kv, -1, D) @ kk.mT / D ** 0.5, -1)
        out[b], size[b] = (w @ vv).view(H, D).cpu(), (w @ vv.abs()).view(H, D).cpu()
    return out, size


def close(got, want, size):
    tol = 2e-5 * (size + want.abs()) + 1e-6
    if got.dtype == F16:
        tol = tol + 2.0 ** -11 * (1.05 * size + 2.1 * want.abs()) + 2.0 ** -24
    worst = ((got.cpu().double() - want).abs() - tol).max().item()
    assert worst <= 0, f"{worst:.3g} over the tolerance"     # NaN fails too


SHAPES = [(32, 8, 128, 16), (8, 1, 64, 32), (40, 8, 128, 32), (6, 6, 64, 16), (64, 2, 128, 16), (3, 1, 128, 32)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,kv,D,page", SHAPES)
@pytest.mark.parametrize("groups,others", [
    ([(1, [0])], []),                                            # one token block, one member, nothing behind
    ([(3, [0, 0, 0])], []),                                      # no suffix at all
    ([(9, [0, 1, 17, 64, 5])], []),
    ([(8, [3, 40]), (1, [0, 2, 9]), (17, [100])], [0, 1, 77]),   # several groups, others, an empty sequence
    ([(5, list(range(45)))], [4]),                               # many rows, odd counts
])
def test_matches_attention_in_64_bits(dtype, heads, kv, D, page, groups, others):
    layout, table, lengths, members, q, k, v = case(groups, others, heads, kv, D, page, dtype)
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=members, dtype=dtype)
    out = plan.run(q, k, v)
    assert out.dtype == dtype
    close(out, *exact(q, k, v, table, lengths))
    first = out.clone()
    mine = torch.empty_like(out)
    assert plan.run(q, k, v, out=mine) is mine and torch.equal(mine, first)     # repeats bit for bit
    assert plan.read_errors() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
def test_long_prefix_split_over_many_ctas(dtype):
    layout, table, lengths, members, q, k, v = case([(700, [0, 33, 5])], [], 8, 2, 128, 16, dtype)
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=members, dtype=dtype)
    close(plan.run(q, k, v), *exact(q, k, v, table, lengths))
    assert plan.read_errors() == 0


@pytest.mark.parametrize("D,page", [(64, 16), (64, 32), (128, 16), (128, 32)])
@pytest.mark.parametrize("tokens", [16384, 12000])
def test_many_steps_per_cta(D, page, tokens):
    """Enough tiles that a CTA walks many 128-token steps, in pairs of tiles and (odd tile counts) in halves."""
    groups = [(tokens // page, list(range(70))), (tokens // 2 // page, [3] * 33)]
    layout, table, lengths, members, q, k, v = case(groups, [], 64, 8, D, page, F16)
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=members)
    out = plan.run(q, k, v)
    some = np.r_[0:103:17]
    close(out[some], *exact(q[some], k, v, table[some], lengths[some]))
    assert plan.read_errors() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("scale", [0.0, 30.0])
def test_flat_and_peaked_scores(dtype, scale):
    """All scores equal, and scores hundreds apart whose maximum moves along the prefix."""
    layout, table, lengths, members, q, k, v = case([(40, [0, 7, 30])], [], 8, 2, 128, 16, dtype, seed=4)
    k.mul_(scale)
    k[k.isnan()] = 0.0
    if scale:
        ramp = torch.linspace(0.1, 1, 40, device="cuda")           # later pages score higher
        for i in range(40):
            k[table[members[0][0][0], i]] *= ramp[i]
    out = SharedPrefixPlan(layout, table, lengths, prefixes=members, dtype=dtype).run(q, k, v)
    want, size = exact(q, k, v, table, lengths)
    if scale:      # |s| reaches ~30 |q k| / sqrt(D): its FP32 rounding grows with it
        size = size * 20
    close(out, want, size)


def test_scores_far_below_the_first_steps_maximum_and_above():
    """The first tokens score lowest by far, then highest: the running maximum moves every way."""
    for sign in (1.0, -1.0):
        layout, table, lengths, members, q, k, v = case([(64, [0, 3])], [], 4, 1, 128, 16, F16, seed=9)
        row = table[members[0][0][0]]
        q.copy_(torch.randn_like(q).abs())
        for i in range(64):
            k[row[i]] = sign * (i - 32) * 0.25 * torch.ones_like(k[0]) + 0.1 * torch.randn_like(k[0])
        out = SharedPrefixPlan(layout, table, lengths, prefixes=members).run(q, k, v)
        want, size = exact(q, k, v, table, lengths)
        close(out, want, size * 20)


def test_found_prefixes_and_none_agree_with_the_decode_plan():
    layout, table, lengths, members, q, k, v = case([(200, [1, 5, 90, 17])], [30, 0], 32, 8, 128, 16, F16)
    want = DecodePlan(layout, table, lengths).run(q, k, v)
    for prefixes in (None, [], members):
        plan = SharedPrefixPlan(layout, table, lengths, prefixes=prefixes)
        torch.testing.assert_close(plan.run(q, k, v).float(), want, atol=2e-3, rtol=2e-3)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,kv", [(32, 8), (32, 1)])
def test_dynamic_plan_with_live_lengths(dtype, heads, kv):
    """Lengths grow, end inside the prefix, or are zero; dead rows hold NaN."""
    layout, table, lengths, members, q, k, v = case([(10, [4, 0, 9, 20])], [12, 0], heads, kv, 128, 16, dtype,
                                                    reserve=24, extra_columns=2)
    k[k.isnan()], v[v.isinf()] = 0.25, 0.5
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=members, dtype=dtype, max_lengths=lengths + 24)
    dev_table = torch.tensor(table, device="cuda")
    a, b, c, d = members[0][0]
    for change in ({}, {a: 24}, {a: -100, b: -160, c: -1}, {a: -164, b: -143, c: -30, d: 3}):
        live = lengths.copy()
        for s, n in change.items():
            live[s] += n
        assert (live >= 0).all()
        out = plan.run_dynamic(q, k, v, dev_table, torch.tensor(live, device="cuda"))
        close(out, *exact(q, k, v, table, live))
        assert plan.read_errors() == 0
    close(plan.run(q, k, v), *exact(q, k, v, table, lengths))       # the plan's own lengths
    over = lengths.copy()
    over[a] += 25
    plan.run_dynamic(q, k, v, dev_table, torch.tensor(over, device="cuda"))
    assert plan.read_errors() == 8


def test_dead_rows_of_a_live_length_inside_the_prefix():
    layout, table, lengths, members, q, k, v = case([(10, [4, 9])], [], 8, 2, 64, 16, F16)
    a, b = members[0][0]
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=members, max_lengths=lengths)
    live = lengths.copy()
    live[a], live[b] = 37, 37
    for i in range(10):                                             # tokens 37.. are dead for both
        for t in range(16):
            if 16 * i + t >= 37:
                k[table[a, i], t], v[table[a, i], t] = float("nan"), float("nan")
    out = plan.run_dynamic(q, k, v, torch.tensor(table, device="cuda"), torch.tensor(live, device="cuda"))
    close(out, *exact(q, k, v, table, live))


@pytest.mark.parametrize("members,pages,heads,kv", [
    (400, 32, 64, 8),      # more row tiles than SMs, an odd one among them
    (200, 32, 64, 8),
    (64, 512, 32, 1),      # pairs of tiles in pieces
    (40, 700, 8, 2)])      # odd tile counts in pieces
def test_every_way_to_cut_the_work(members, pages, heads, kv):
    layout, table, lengths, groups, q, k, v = case([(pages, [i % 40 for i in range(members)])], [7, 0], heads, kv, 128,
                                                   16, F16)
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=groups)
    out = plan.run(q, k, v)
    some = np.r_[0:members + 2:9, members, members + 1]
    close(out[some], *exact(q[some], k, v, table[some], lengths[some]))
    first = out.clone()
    assert all(torch.equal(plan.run(q, k, v), first) for _ in range(5)) and plan.read_errors() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
def test_live_lengths_inside_a_long_prefix(dtype):
    """As above where the prefix is cut in many pieces."""
    layout, table, lengths, members, q, k, v = case([(600, [4, 0, 9, 20])], [12, 0], 8, 2, 128, 16, dtype)
    k[k.isnan()], v[v.isinf()] = 0.25, 0.5
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=members, dtype=dtype, max_lengths=lengths)
    live = lengths.copy()
    a, b, c, _ = members[0][0]
    live[a], live[b], live[c] = 0, 1, 9000
    out = plan.run_dynamic(q, k, v, torch.tensor(table, device="cuda"), torch.tensor(live, device="cuda"))
    close(out, *exact(q, k, v, table, live))
    assert plan.read_errors() == 0


def test_another_stream_and_interleaved_plans():
    """Two plans of different shapes taking turns on a stream of their own."""
    sets = [case([(30, [3, 9])], [4], 8, 2, 128, 16, F16, seed=1), case([(12, list(range(40)))], [], 32, 1, 64, 32, F16, seed=2)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        plans = [SharedPrefixPlan(s[0], s[1], s[2], prefixes=s[3]) for s in sets]
        for _ in range(20):
            outs = [p.run(*s[4:]) for p, s in zip(plans, sets)]
    stream.synchronize()
    for s, out, plan in zip(sets, outs, plans):
        close(out, *exact(*s[4:], s[1], s[2]))
        assert plan.read_errors() == 0


def test_pages_past_32_bit_offsets():
    page, kv, D = 32, 8, 128
    pages = (1 << 31) // (page * kv * D) + 40
    k, v = (torch.empty((pages, page, kv, D), device="cuda", dtype=F16) for _ in range(2))
    lengths = np.array([32 * 6 + 20, 32 * 6 + 3], dtype=np.int32)
    table = np.stack([np.arange(pages - 7, pages), np.arange(pages - 7, pages)]).astype(np.int32)
    table[1, 6] = pages - 20
    for p in set(table.reshape(-1).tolist()):
        k[p].normal_(), v[p].normal_()
    q = torch.randn((2, 16, D), device="cuda", dtype=F16)
    out = SharedPrefixPlan(Layout(2, 16, kv, D, page, pages), table, lengths, prefixes=[([0, 1], 6)]).run(q, k, v)
    close(out, *exact(q, k, v, table, lengths))


def test_a_nan_in_a_live_row_reaches_its_sequences_only():
    layout, table, lengths, members, q, k, v = case([(6, [4, 9])], [50], 8, 2, 64, 16, F32)
    k[table[members[0][0][0], 2], 3, 1, 5] = float("nan")
    out = SharedPrefixPlan(layout, table, lengths, prefixes=members, dtype=F32).run(q, k, v)
    other = [b for b in range(3) if b not in members[0][0]]
    assert torch.isnan(out[members[0][0], 4:]).all() and not torch.isnan(out[members[0][0], :4]).any()
    assert not torch.isnan(out[other]).any()


def test_append_and_shared_prefix_steps_in_a_graph():
    """A decode loop: append with rotation, then attention behind a shared prefix, captured once."""
    layout, table, lengths, members, q, k, v = case([(12, [0, 5, 30, 2])], [9], 32, 8, 128, 16, F16, reserve=12)
    k[k.isnan()], v[v.isinf()] = 0.0, 0.0
    rope = rotation_table(512, 128)
    append = CacheAppend(layout, HeadRotation(128, rope))
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=members, max_lengths=lengths + 12)
    dev_table, live = torch.tensor(table, device="cuda"), torch.tensor(lengths, device="cuda")
    qkv = torch.randn((5, 48, 128), device="cuda", dtype=F16)
    rotated = torch.empty((5, 32, 128), device="cuda", dtype=F16)

    def step():
        live.add_(1)
        append.run(qkv[:, 32:40], qkv[:, 40:], k, v, dev_table, live, q=qkv[:, :32], q_out=rotated)
        return plan.run_dynamic(rotated, k, v, dev_table, live)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(10):
        qkv.copy_(torch.randn_like(qkv))
        graph.replay()
    torch.cuda.synchronize()
    assert live.tolist() == (lengths + 11).tolist()
    close(out, *exact(rotated, k, v, table, lengths + 11))
    assert append.read_errors() == 0 and plan.read_errors() == 0


def test_refusals():
    layout, table, lengths, members, q, k, v = case([(3, [4, 9])], [50], 8, 2, 64, 16, F16)
    a, b = members[0][0]
    other = 3 - a - b
    for prefixes in ([([a, b], 0)], [([a, b], 99)], [([a, b], 4)], [([a, other], 1)], [([a, b], 1), ([b], 2)],
                     [([a, 7], 1)], [([a, -1], 1)], [([], 1)], [([a, a], 1)]):
        with pytest.raises(ValueError):
            SharedPrefixPlan(layout, table, lengths, prefixes=prefixes)
    with pytest.raises(TypeError):
        SharedPrefixPlan(layout, table, lengths, prefixes=[([0.5], 1)])
    with pytest.raises(TypeError):
        SharedPrefixPlan(layout, table, lengths, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        SharedPrefixPlan(layout, table, lengths, device="cpu")
    with pytest.raises(ValueError):
        SharedPrefixPlan(layout, table, lengths, max_lengths=lengths - 1)
    plan = SharedPrefixPlan(layout, table, lengths, prefixes=members)
    for args, error in (((q[:1], k, v), ValueError), ((q.float(), k.float(), v.float()), TypeError),
                        ((q, k[1:], v), ValueError), ((q.cpu(), k, v), ValueError),
                        ((q.clone().requires_grad_(), k, v), ValueError)):
        with pytest.raises(error):
            plan.run(*args)
    with pytest.raises(ValueError):
        plan.run(q, k, v, out=torch.empty_like(q, dtype=F32))
    with pytest.raises(ValueError):
        plan.run_dynamic(q, k, v, torch.tensor(table, device="cuda"), torch.tensor(lengths, device="cuda"))
    dynamic = SharedPrefixPlan(layout, table, lengths, prefixes=members, max_lengths=lengths)
    with pytest.raises(ValueError):
        dynamic.run_dynamic(q, k, v, torch.tensor(table, device="cuda").long(), torch.tensor(lengths, device="cuda"))


@pytest.mark.parametrize("batch,prompt,steps", [(3, 100, 20), (33, 1024, 5)])
def test_the_example_runs(batch, prompt, steps):
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parents[1] / "paged-decode-lab_b200" / "examples" / "shared_prefix_loop.py"
    spec = importlib.util.spec_from_file_location("shared_prefix_loop", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    result = module.run(batch=batch, prompt=prompt, steps=steps)
    # values of the projection are about N(0, 1): the FP16 bounds above with |v| <= 6
    assert result["shared_error"] < 6 * 2.0 ** -10 and result["apart_error"] < 6 * 2.0 ** -10
