"""Head norm + rotation and the cache append against their formulas in 64 bits.

Tolerances, from the formulas: with u = 2^-24 the FP32 norm is off by at most
(D/2 + 4) u of an element (a sum of D squares, halved by the square root, three
more products), the rotation by 3u of |a cos| + |b sin|, and the store rounds
once (2^-11 relative for FP16, half a spacing of 2^-24 below its normal range).
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("NVIDIA GPU required", allow_module_level=True)

from oracle.paged_oracle import dense_attention
from paged_decode.layout import Layout
from paged_decode.rotary import CacheAppend, HeadRotation, rotation_table
from paged_decode.runtime import DecodePlan

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
BAD_PAGE, LENGTH, POSITION = 2, 8, 16


def exact(x, weight, positions, table, interleaved, eps=1e-6):
    """(the head rows in 64 bits, the bound of the FP32 computation's error before the store)."""
    x = x.detach().cpu().double()
    D = x.shape[-1]
    y = x.clone()
    if weight is not None:
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.cpu().double()
    size = y.abs()
    if table is not None:
        r = table.shape[1]
        at = table.cpu().double()[positions.cpu().long()]
        c, s = at[:, None, :r // 2], at[:, None, r // 2:]
        i, j = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
        a, b = y[..., i].clone(), y[..., j].clone()
        y[..., i], y[..., j] = a * c - b * s, b * c + a * s
        size[..., i], size[..., j] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size * (D / 2 + 8) * 2.0 ** -24


def close(got, want, bound):
    got16 = got.dtype == F16
    got = got.cpu().double()
    if got16:
        bound = bound + (want.abs() + bound) * 2.0 ** -11 + 2.0 ** -25
    worst = ((got - want).abs() - bound).max().item()
    assert worst <= 0, f"{worst:.3g} over the bound"


def packed(tokens, heads, kv, D, dtype, form, seed=0):
    """q, k, v with the strides of one packed projection ("packed"), one element off 16-byte
    alignment ("odd"), heads before tokens ("swapped"), or dense."""
    gen = torch.Generator("cuda").manual_seed(seed)
    width = (heads + 2 * kv) * D
    if form == "swapped":
        x = torch.randn((heads + 2 * kv, tokens, D), device="cuda", dtype=dtype, generator=gen).mul_(2).transpose(0, 1)
    else:
        pad = 3 if form == "odd" else 0
        x = torch.randn((tokens, width + pad), device="cuda", dtype=dtype, generator=gen).mul_(2)
        x = x[:, pad and 1: width + (pad and 1)].unflatten(1, (heads + 2 * kv, D))
    parts = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    return tuple(p.contiguous() for p in parts) if form == "dense" else parts


def weights(D, dtype):
    return (1 + 0.2 * torch.randn(D, device="cuda", dtype=dtype), 1 + 0.2 * torch.randn(D, device="cuda", dtype=dtype))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,rotary", [(64, 64), (64, 16), (128, 128), (128, 32), (128, 48), (128, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("form,heads,kv,tokens", [("packed", 32, 8, 5), ("odd", 3, 1, 1), ("swapped", 7, 7, 33),
                                                  ("dense", 130, 2, 3)])
def test_rotate_matches_the_formula(dtype, D, rotary, interleaved, form, heads, kv, tokens):
    q, k, _ = packed(tokens, heads, kv, D, dtype, form)
    table = rotation_table(300, rotary) if rotary else None
    qw, kw = weights(D, dtype) if heads != 7 else (None, None)
    if heads == 130:
        kw = None                                   # queries normed, keys not
    op = HeadRotation(D, table, interleaved=interleaved, q_weight=qw, k_weight=kw)
    positions = torch.randint(0, 300, (tokens,), device="cuda", dtype=torch.int32)
    positions[0] = 299
    q_out, k_out = op.run(q, k, positions)
    close(q_out, *exact(q, qw, positions, table, interleaved))
    close(k_out, *exact(k, kw, positions, table, interleaved))
    assert op.read_errors() == 0
    # one operand alone, into strided outputs, and in place: the same bits
    out = torch.full((tokens, heads + 1, D + 8), float("nan"), device="cuda", dtype=dtype)
    alone, none = op.run(q, None, positions, q_out=out[:, 1:, :D])
    assert none is None and torch.equal(alone, q_out) and torch.isnan(out[:, 0]).all() and torch.isnan(out[..., D:]).all()
    op.run(q, k, positions, q_out=q, k_out=k)
    assert torch.equal(q, q_out) and torch.equal(k, k_out)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,heads,kv,rotary,interleaved", [(128, 32, 8, 128, False), (128, 5, 1, 32, True),
                                                           (64, 33, 33, 64, True), (64, 4, 0, 16, False)])
@pytest.mark.parametrize("tokens", [900, 4099])
def test_rotate_many_tokens(dtype, D, heads, kv, rotary, interleaved, tokens):
    """Enough tokens for a persistent grid; the same bits as a few tokens at a time, and as strided heads."""
    q, k, _ = packed(tokens, heads, kv, D, dtype, "packed")
    k = k if kv else None
    qw, kw = weights(D, dtype)
    op = HeadRotation(D, rotation_table(300, rotary), interleaved=interleaved, q_weight=qw, k_weight=kw if kv != 1 else None)
    positions = torch.randint(0, 300, (tokens,), device="cuda", dtype=torch.int32)
    positions[[3, tokens - 2]] = 300                 # outside the table
    got = op.run(q, k, positions)
    assert op.read_errors() == POSITION
    for x, y, w in zip((q, k), got, (qw, kw if kv != 1 else None)):
        if x is not None:
            live = positions < 300
            close(y[live], *exact(x[live], w, positions[live], op.table, interleaved))
            assert not y[~live].any()
    few = [op.run(q[i:i + 50], None if k is None else k[i:i + 50], positions[i:i + 50]) for i in range(0, tokens, 50)]
    swapped = op.run(q.transpose(0, 1).contiguous().transpose(0, 1), k, positions)
    for i in range(1 + (k is not None)):
        assert torch.equal(got[i], torch.cat([f[i] for f in few])) and torch.equal(got[i], swapped[i])
    op.run(q, k, positions, q_out=q, k_out=k)
    assert torch.equal(q, got[0]) and (k is None or torch.equal(k, got[1]))


def test_rotation_table_is_exact_to_fp32():
    t = rotation_table(131072, 128, base=500000.0)
    p, i = 131071, 1
    angle = p * 500000.0 ** (-2 * i / 128)
    assert abs(t[p, i].item() - np.cos(angle)) < 1e-7 and abs(t[p, 64 + i].item() - np.sin(angle)) < 1e-7


def test_zero_tokens_and_zero_heads():
    op = HeadRotation(64, rotation_table(4, 64))
    empty = torch.empty((0, 8, 64), device="cuda", dtype=F16)
    q, k = op.run(empty, empty[:, :2], torch.empty(0, device="cuda", dtype=torch.int32))
    assert q.shape == (0, 8, 64) and k.shape == (0, 2, 64)
    q, k = op.run(torch.empty((2, 0, 64), device="cuda", dtype=F16), None, torch.zeros(2, device="cuda", dtype=torch.int32))
    assert q.shape == (2, 0, 64)


def test_positions_outside_the_table_give_zero_rows_and_a_flag():
    op = HeadRotation(128, rotation_table(8, 128))
    q = torch.randn(4, 2, 128, device="cuda", dtype=F16)
    positions = torch.tensor([7, 8, -1, 0], device="cuda", dtype=torch.int32)
    out, _ = op.run(q, None, positions)
    assert op.read_errors() == POSITION and op.read_errors() == 0
    assert not out[1].any() and not out[2].any() and out[0].any() and out[3].any()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_infinities_and_nans_stay_in_their_head(dtype):
    op = HeadRotation(128, rotation_table(8, 64), q_weight=torch.ones(128, device="cuda"))
    x = torch.randn(3, 5, 128, device="cuda", dtype=dtype)
    k = x.clone()
    clean, clean_k = op.run(x, k, torch.arange(3, device="cuda", dtype=torch.int32))
    x[1, 2, 5] = float("nan")
    k[1, 3, 100] = float("inf")                     # past the rotation: passes
    k[2, 0, 3] = -float("inf")                      # inside it: its pair's two elements
    got, got_k = op.run(x, k, torch.arange(3, device="cuda", dtype=torch.int32))
    assert torch.isnan(got[1, 2]).all()
    got[1, 2] = clean[1, 2]
    assert torch.equal(got, clean)
    assert got_k[1, 3, 100] == float("inf") and not torch.isfinite(got_k[2, 0, [3, 35]]).any()
    got_k[1, 3, 100], got_k[2, 0, 3], got_k[2, 0, 35] = clean_k[1, 3, 100], clean_k[2, 0, 3], clean_k[2, 0, 35]
    assert torch.equal(got_k, clean_k)


# ------------------------------------------------------------------ append
def cache_case(lengths, page, kv, D, dtype, seed=1, spare=2):
    rng = np.random.default_rng(seed)
    width = max(1, -(-max(lengths) // page)) + 1
    pages = len(lengths) * width + spare
    table = rng.permutation(pages)[: len(lengths) * width].reshape(len(lengths), width).astype(np.int32)
    for b, n in enumerate(lengths):
        table[b, -(-n // page):] = -1
    caches = [torch.randn((pages, page, kv, D), device="cuda", dtype=dtype) for _ in range(2)]
    return table, caches


def appended(table, lengths, counts, page):
    """(token, page, offset, position) of every appended token."""
    out, i = [], 0
    for b, (n, m) in enumerate(zip(counts, lengths)):
        for t in range(m - n, m):
            out.append((i, int(table[b, t // page]), t % page, t))
            i += 1
    return out


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,page,heads,kv,form", [(128, 16, 32, 8, "packed"), (64, 32, 5, 5, "odd"),
                                                  (128, 32, 32, 1, "swapped"), (64, 16, 12, 4, "dense")])
@pytest.mark.parametrize("lengths,counts", [
    ([1], None), ([5, 0, 33, 48, 1], None), ([40, 16, 17, 70], [40, 16, 0, 37]), ([0, 0, 3], [0, 0, 3]),
    ([64, 100], [1, 65])])
def test_append_matches_the_formula(dtype, D, page, heads, kv, form, lengths, counts):
    n = [int(m > 0) for m in lengths] if counts is None else counts
    tokens = len(lengths) if counts is None else sum(counts)
    table, (kc, vc) = cache_case(lengths, page, kv, D, dtype)
    q, k, v = packed(tokens, heads, kv, D, dtype, form, seed=3)
    rope = rotation_table(128, D // 2 if D == 128 else D)
    qw, kw = weights(D, dtype)
    interleaved = page == 32
    layout = Layout(len(lengths), heads, kv, D, page, kc.shape[0])
    op = CacheAppend(layout, HeadRotation(D, rope, interleaved=interleaved, q_weight=qw, k_weight=kw))
    indptr = None if counts is None else torch.tensor(np.concatenate(([0], np.cumsum(counts))), device="cuda",
                                                      dtype=torch.int32)
    before = kc.clone(), vc.clone()
    out = op.run(k, v, kc, vc, torch.tensor(table, device="cuda"),
                 torch.tensor(lengths, device="cuda", dtype=torch.int32), q=q, indptr=indptr)
    assert op.read_errors() == 0
    where = appended(table, lengths, n, page)
    if counts is None:                               # token b belongs to sequence b
        live = [b for b, m in enumerate(lengths) if m]
        where = [(b, *w[1:]) for b, w in zip(live, where)]
        dead = [b for b, m in enumerate(lengths) if not m]
        assert not out[dead].any()
    i, pg, off, pos = (torch.tensor(x, dtype=torch.int64) for x in zip(*where))
    close(out[i], *exact(q[i], qw, pos, rope, interleaved))
    close(kc[pg, off], *exact(k[i], kw, pos, rope, interleaved))
    assert torch.equal(vc[pg, off], v[i])
    kc[pg, off], vc[pg, off] = before[0][pg, off], before[1][pg, off]
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])      # nothing else was touched


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,page,heads,kv", [(128, 16, 32, 8), (64, 32, 4, 4), (128, 32, 6, 1)])
@pytest.mark.parametrize("with_q", [True, False])
def test_append_many_tokens(dtype, D, page, heads, kv, with_q):
    """A long ragged prompt batch with padding behind it, a page that is missing and a sequence that is too long."""
    counts = [700, 0, 1, 333, 64, 1025]
    lengths = [700, 5, 900, 400, 64, 1030]
    tokens, padded = sum(counts), sum(counts) + 19
    table, (kc, vc) = cache_case(lengths, page, kv, D, dtype)
    table[3, 200 // page] = -1                       # positions of one page of sequence 3
    q, k, v = packed(padded, heads, kv, D, dtype, "packed", seed=3)
    rope = rotation_table(1029, D)                   # the last position of sequence 5 is outside
    qw, kw = weights(D, dtype)
    op = CacheAppend(Layout(6, heads, kv, D, page, kc.shape[0]), HeadRotation(D, rope, q_weight=qw, k_weight=kw))
    before = kc.clone(), vc.clone()
    out = op.run(k, v, kc, vc, torch.tensor(table, device="cuda"),
                 torch.tensor(lengths, device="cuda", dtype=torch.int32), q=q if with_q else None,
                 indptr=torch.tensor(np.concatenate(([0], np.cumsum(counts))), device="cuda", dtype=torch.int32))
    assert op.read_errors() == BAD_PAGE | POSITION
    where = appended(table, lengths, counts, page)
    dead = [w[0] for w in where if w[1] < 0 or w[3] >= 1029]
    assert len(dead) == page + 1
    where = [w for w in where if w[0] not in dead]
    i, pg, off, pos = (torch.tensor(x, dtype=torch.int64) for x in zip(*where))
    if with_q:
        close(out[i], *exact(q[i], qw, pos, rope, False))
        assert not out[tokens:].any() and not out[dead].any()
    close(kc[pg, off], *exact(k[i], kw, pos, rope, False))
    assert torch.equal(vc[pg, off], v[i])
    kc[pg, off], vc[pg, off] = before[0][pg, off], before[1][pg, off]
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


def test_append_without_rotation_copies_bits():
    table, (kc, vc) = cache_case([9, 4], 16, 2, 64, F16)
    k = torch.randint(-32768, 32768, (2, 2, 64), device="cuda", dtype=torch.int16).view(F16)   # NaNs with payloads
    v = torch.randint(-32768, 32768, (2, 2, 64), device="cuda", dtype=torch.int16).view(F16)
    k.view(torch.int16)[k.isnan()] = 0               # an FP32 pass may quiet a NaN; values are copied whole
    op = CacheAppend(Layout(2, 4, 2, 64, 16, kc.shape[0]))
    assert op.run(k, v, kc, vc, torch.tensor(table, device="cuda"),
                  torch.tensor([9, 4], device="cuda", dtype=torch.int32)) is None
    for b, n in enumerate((9, 4)):
        page, off = int(table[b, (n - 1) // 16]), (n - 1) % 16
        assert torch.equal(kc[page, off].view(torch.int16), k[b].view(torch.int16))
        assert torch.equal(vc[page, off].view(torch.int16), v[b].view(torch.int16))


def test_append_skips_and_flags_what_has_no_place():
    page, kv, D = 16, 2, 64
    layout = Layout(4, 4, kv, D, page, 8)
    kc, vc = (torch.zeros((8, page, kv, D), device="cuda", dtype=F16) for _ in range(2))
    op = CacheAppend(layout, HeadRotation(D, rotation_table(20, D)))
    q, k, v = packed(4, 4, kv, D, F16, "packed")
    table = torch.tensor([[0, 1], [2, -1], [8, 3], [4, 5]], device="cuda", dtype=torch.int32)

    def run(lengths, **kw):
        kc.zero_(), vc.zero_()
        out = op.run(k, v, kc, vc, table, torch.tensor(lengths, device="cuda", dtype=torch.int32), q=q, **kw)
        return [bool(r.any()) for r in out], int(kc.flatten(0, 1).any(-1).any(-1).sum()), op.read_errors()

    assert run([17, 16, 18, 20]) == ([True] * 4, 4, 0)
    assert run([17, 17, 18, 20]) == ([True, False, True, True], 3, BAD_PAGE)       # page -1
    assert run([17, 16, 16, 20]) == ([True, True, False, True], 3, BAD_PAGE)       # page 8 of 8
    assert run([33, 16, 18, 20]) == ([False, True, True, True], 3, LENGTH)         # past the table row
    assert run([17, 16, 18, 21]) == ([True, True, True, False], 3, POSITION)       # past the rotation table
    assert run([17, 16, 18, -3]) == ([True, True, True, False], 3, LENGTH)
    # ragged: more tokens than the length counts; padding behind the last sequence is silent
    ends = torch.tensor([0, 2, 2, 2, 3], device="cuda", dtype=torch.int32)
    assert run([1, 0, 0, 5], indptr=ends) == ([False, True, True, False], 2, LENGTH)


def test_append_past_32_bit_offsets():
    page, kv, D = 32, 8, 128
    pages = (1 << 31) // (page * kv * D) + 8         # elements past 2^31, bytes past 2^32
    kc, vc = (torch.empty((pages, page, kv, D), device="cuda", dtype=F16) for _ in range(2))
    layout = Layout(2, 8, kv, D, page, pages)
    table = torch.tensor([[pages - 1], [pages - 3]], device="cuda", dtype=torch.int32)
    _, k, v = packed(2, 8, kv, D, F16, "packed")
    CacheAppend(layout).run(k, v, kc, vc, table, torch.tensor([32, 7], device="cuda", dtype=torch.int32))
    assert torch.equal(kc[pages - 1, 31], k[0]) and torch.equal(vc[pages - 3, 6], v[1])


def test_append_then_decode_in_a_graph_on_another_stream():
    """A captured step (lengths + 1, append with rotation, decode) replayed along a sequence's growth."""
    heads, kv, D, page, steps = 8, 2, 128, 16, 20
    start = np.array([3, 15, 0], dtype=np.int32)
    width = 4
    layout = Layout(3, heads, kv, D, page, 3 * width)
    table = np.random.default_rng(2).permutation(3 * width).reshape(3, width).astype(np.int32)
    kc, vc = (torch.randn((3 * width, page, kv, D), device="cuda", dtype=F16) for _ in range(2))
    rope = rotation_table(64, D)
    op = CacheAppend(layout, HeadRotation(D, rope))
    plan = DecodePlan(layout, table, start, max_lengths=start + steps)
    dev_table, lengths = torch.tensor(table, device="cuda"), torch.tensor(start, device="cuda")
    qkv = torch.randn((3, heads + 2 * kv, D), device="cuda", dtype=F16)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    rotated = torch.empty((3, heads, D), device="cuda", dtype=F16)

    def step():
        lengths.add_(1)
        op.run(k, v, kc, vc, dev_table, lengths, q=q, q_out=rotated)
        return plan.run_dynamic(rotated, kc, vc, dev_table, lengths)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        lengths.copy_(torch.tensor(start + 1))
        for i in range(2, steps):
            qkv.copy_(torch.randn((3, heads + 2 * kv, D), device="cuda", dtype=F16))
            graph.replay()
    torch.cuda.synchronize()
    assert lengths.tolist() == (start + steps - 1).tolist()
    want, bound = exact(q, None, lengths - 1, rope, False)
    close(rotated, want, bound)
    oracle = dense_attention(rotated.cpu().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table, start + steps - 1)
    np.testing.assert_allclose(out.cpu().numpy(), oracle, atol=2e-3, rtol=1e-3)
    assert op.read_errors() == 0 and plan.read_errors() == 0


# ------------------------------------------------------------------ refusals
def test_refusals():
    rope = rotation_table(16, 64)
    op = HeadRotation(64, rope)
    q = torch.randn(2, 4, 64, device="cuda", dtype=F16)
    at = torch.zeros(2, device="cuda", dtype=torch.int32)
    for bad in (dict(head_dim=96), dict(head_dim=64, table=rope[:, :24]), dict(head_dim=64, table=rope[:, ::2]),
                dict(head_dim=64, eps=-1.0), dict(head_dim=64, q_weight=torch.ones(32, device="cuda")),
                dict(head_dim=64, table=rope.cpu()), dict(head_dim=64, device="cpu")):
        with pytest.raises(ValueError):
            HeadRotation(**bad)
    with pytest.raises(TypeError):
        HeadRotation(64, rope.half())
    for args, error in (((q.bfloat16(), None, at), TypeError), ((q, q.float(), at), TypeError),
                        ((None, None, at), ValueError), ((q, None, at.long()), ValueError),
                        ((q, None, at[:1]), ValueError), ((q[..., :32], None, at), ValueError),
                        ((q.transpose(1, 2), None, at), ValueError), ((q.cpu(), None, at), ValueError),
                        ((q, q[:1], at), ValueError), ((q.clone().requires_grad_(), None, at), ValueError)):
        with pytest.raises(error):
            op.run(*args)
    with pytest.raises(ValueError):
        op.run(q, None, at, q_out=q[:1])
    with pytest.raises(ValueError):
        op.run(q, None, at, k_out=q)
    layout = Layout(2, 4, 4, 64, 16, 4)
    cache = torch.zeros(4, 16, 4, 64, device="cuda", dtype=F16)
    table, lengths = torch.zeros(2, 2, device="cuda", dtype=torch.int32), torch.ones(2, device="cuda", dtype=torch.int32)
    append = CacheAppend(layout, op)
    good = (q, q, cache, cache.clone(), table, lengths)
    for i, bad, error in ((0, q[:1], ValueError), (1, q.float(), TypeError), (2, cache[:3], ValueError),
                          (3, cache.transpose(1, 2).contiguous().transpose(1, 2), ValueError),
                          (2, cache.float(), TypeError), (4, table.long(), ValueError), (4, table[:1], ValueError),
                          (5, lengths.cpu(), ValueError)):
        args = list(good)
        args[i] = bad
        with pytest.raises(error):
            append.run(*args)
    with pytest.raises(ValueError):
        append.run(*good, indptr=torch.zeros(2, device="cuda", dtype=torch.int32))
    with pytest.raises(ValueError):
        append.run(*good, q_out=q)
    with pytest.raises(ValueError):
        append.run(q[:1], q[:1], *good[2:])          # one token per sequence without indptr
    with pytest.raises(ValueError):
        CacheAppend(Layout(2, 4, 4, 128, 16, 4), op)
    with pytest.raises(ValueError):
        CacheAppend(Layout(2, 4, 4, 64, 8, 4))
