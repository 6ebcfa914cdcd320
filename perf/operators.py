"""Cases for the operators around a paged decode step, with their plain forms.

Three operators that meet at the paged cache of the decode attention:

* ``rotate``: RMS norm of each query and key head and the position rotation, in one pass;
* ``append``: a step's (or a prompt's) keys and values into the paged cache, normed and rotated on
  the way, with the queries normed and rotated beside them;
* ``prefix``: decode attention of a batch whose sequences share leading pages, the shared part
  computed once for all of them.

With ``own`` false, ``run`` computes them in elementary torch operations in 32 bits, rounded once at
the end; with ``own`` true it calls the framework.  A case is a dict of plain values; lengths follow
from the case alone, tensors and page numbers from the seed.
"""
import math

import numpy as np
import torch

own = False

_HALF, _FULL = "float16", "float32"


def listed():
    return [
        # one new token for each of four sequences, Llama-3-8B heads: the latency of a small decode step
        dict(name="append_decode_b4", op="append", dtype=_HALF, batch=4, heads=32, kv_heads=8, dim=128, page=16,
             chunk=1, ragged=False, context=4096, rotary=128, interleaved=False, norm=True),
        # prompts of eight sequences in one ragged batch, Llama-3-70B heads: prefill throughput
        dict(name="append_prefill", op="append", dtype=_HALF, batch=8, heads=64, kv_heads=8, dim=128, page=16,
             chunk=4096, ragged=True, context=4096, rotary=128, interleaved=False, norm=True),
        # short chunks of many FP32 sequences with as many KV heads as query heads: half of each head
        # rotated in neighbouring pairs, no norm, a chunk that ends inside a page
        dict(name="append_fp32_chunks", op="append", dtype=_FULL, batch=64, heads=32, kv_heads=32, dim=64, page=32,
             chunk=37, ragged=True, context=2048, rotary=32, interleaved=True, norm=False),
        # queries and keys of one decode step, one shared KV head
        dict(name="rotate_decode_b64", op="rotate", dtype=_HALF, tokens=64, heads=32, kv_heads=1, dim=128,
             positions=8192, rotary=128, interleaved=False, norm=True),
        # a long prompt's queries and keys
        dict(name="rotate_prefill", op="rotate", dtype=_HALF, tokens=16384, heads=32, kv_heads=8, dim=128,
             positions=16384, rotary=128, interleaved=False, norm=True),
        # an odd number of FP32 tokens, half of a narrow head rotated
        dict(name="rotate_fp32_odd", op="rotate", dtype=_FULL, tokens=4099, heads=32, kv_heads=32, dim=64,
             positions=8192, rotary=32, interleaved=False, norm=True),
        # a few chats right behind one system prompt: latency
        dict(name="prefix_b4", op="prefix", dtype=_HALF, batch=4, sharers=4, heads=32, kv_heads=8, dim=128, page=16,
             prefix=1024, low=0, high=64),
        # 32 ragged sequences of which a quarter share 64 pages
        dict(name="prefix_quarter_shared", op="prefix", dtype=_HALF, batch=32, sharers=8, heads=32, kv_heads=8,
             dim=128, page=16, prefix=1024, low=0, high=7168),
        # one KV head for all query heads, pages of 32
        dict(name="prefix_mqa_b64", op="prefix", dtype=_HALF, batch=64, sharers=64, heads=32, kv_heads=1, dim=128,
             page=32, prefix=2048, low=1, high=256),
        # a large serving batch, Llama-3-70B heads, behind a long instruction
        dict(name="prefix_b256", op="prefix", dtype=_HALF, batch=256, sharers=256, heads=64, kv_heads=8, dim=128,
             page=16, prefix=4096, low=1, high=1024),
        # questions to one long document
        dict(name="prefix_long", op="prefix", dtype=_HALF, batch=8, sharers=8, heads=32, kv_heads=8, dim=128,
             page=32, prefix=131072 - 512, low=1, high=512),
        # FP32 cache, as many KV heads as query heads
        dict(name="prefix_fp32", op="prefix", dtype=_FULL, batch=16, sharers=16, heads=32, kv_heads=32, dim=64,
             page=32, prefix=2048, low=0, high=128),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], uniform in its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _heads(rng):
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (32, 32), (32, 1), (8, 2), (12, 4), (40, 8), (28, 4), (16, 1),
                                  (24, 8), (6, 6)])
    return heads, kv_heads


def draw(rng):
    op = rng.choice(["append", "rotate", "prefix", "prefix"])
    top = {o: [work(c) for c in listed() if c["op"] == o] for o in ("append", "rotate", "prefix")}[op]
    top = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    while True:
        heads, kv_heads = _heads(rng)
        dim, page = rng.choice([64, 128]), rng.choice([16, 32])
        dtype = _FULL if rng.random() < 0.25 else _HALF
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        case = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim)
        if op == "append":
            chunk = 1 if rng.random() < 0.4 else _spread(rng, 2, 4096)
            case.update(batch=_spread(rng, 1, 256), page=page, chunk=chunk,
                        ragged=chunk > 1 and rng.random() < 0.7, context=_spread(rng, max(chunk, 16), 8192),
                        rotary=rotary, interleaved=rng.random() < 0.4, norm=rng.random() < 0.6)
            if case["batch"] * case["context"] > 65536:      # the cache that is compared
                continue
        elif op == "rotate":
            case.update(tokens=_spread(rng, 1, 16384), positions=_spread(rng, 1024, 131072), rotary=rotary,
                        interleaved=rng.random() < 0.4, norm=rng.random() < 0.6)
        else:
            batch = _spread(rng, 2, 256)
            case.update(batch=batch, sharers=batch if rng.random() < 0.7 else rng.randint(2, batch), page=page,
                        prefix=page * _spread(rng, 1, 131072 // page), low=rng.choice([0, 1]),
                        high=_spread(rng, 1, 2048))
            span = case["prefix"] + case["high"]
            if batch * span * kv_heads * dim > 1.4e9 or batch * heads * span > 2e8:
                continue                                      # the plain form's gathered rows and scores
            if dtype == _FULL and work(case)["flops"] > work(listed()[-1])["flops"]:
                continue
        w = work(case)
        if all(w[k] <= top[k] for k in top):
            return case


def _plan_rng(case):
    """The generator of a case's lengths: the same for every seed of its tensors."""
    words = [case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]]
    words += [case[k] for k in ("chunk", "context", "sharers", "prefix", "low", "high") if k in case]
    return np.random.default_rng([int(w) for w in words])


def _append_lengths(case):
    """New tokens n[b] and lengths[b] after the append."""
    rng, B = _plan_rng(case), case["batch"]
    n = rng.integers(0, case["chunk"] + 1, B) if case["ragged"] else np.full(B, case["chunk"])
    if case["ragged"]:
        n[0] = case["chunk"]
    lengths = n + rng.integers(0, np.maximum(case["context"] - n, 0) + 1)
    return n.astype(np.int64), lengths.astype(np.int64)


def _prefix_lengths(case):
    """lengths[b] and whether sequence b shares the prefix."""
    rng, B = _plan_rng(case), case["batch"]
    shares = np.zeros(B, dtype=bool)
    shares[rng.permutation(B)[: case["sharers"]]] = True
    lengths = rng.integers(case["low"], case["high"] + 1, B) + np.where(shares, case["prefix"], 0)
    return lengths.astype(np.int64), shares


def work(case):
    elt = 2 if case["dtype"] == _HALF else 4
    D, H, K = case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "prefix":
        lengths, shares = _prefix_lengths(case)
        rows = int(lengths.sum()) - (int(shares.sum()) - 1) * case["prefix"]      # distinct cache rows
        pages = int((-(-lengths // case["page"])).sum())
        return {"bytes": 2 * rows * K * D * elt + 2 * case["batch"] * H * D * elt + 4 * pages,
                "flops": 4 * H * D * int(lengths.sum())}
    n = case["tokens"] if case["op"] == "rotate" else int(_append_lengths(case)[0].sum())
    heads = H + K if case["op"] == "rotate" else H + 2 * K
    turned = case["rotary"] + (D if case["norm"] else 0)
    return {"bytes": 2 * n * heads * D * elt + n * (4 * case["rotary"] + 4), "flops": 3 * n * (H + K) * turned}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rotation(case, positions):
    """cos | sin of every position, [positions, rotary] in 32 bits."""
    r = case["rotary"]
    freq = 10000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _package():
    import sys
    from pathlib import Path
    root = str(Path(__file__).resolve().parents[1] / "paged-decode-lab_b200")
    if root not in sys.path:
        sys.path.insert(0, root)


def prepare(case, seed):
    gen = _generator(seed)
    dtype = getattr(torch, case["dtype"])
    D, H, K = case["dim"], case["heads"], case["kv_heads"]
    s = {"case": case}

    def randn(*shape, std=1.0):
        return torch.randn(shape, device="cuda", dtype=dtype, generator=gen).mul_(std)

    if case["op"] != "prefix":
        # projections leave one packed row per token: queries, keys, values
        n = case["tokens"] if case["op"] == "rotate" else int(_append_lengths(case)[0].sum())
        packed = randn(n, (H + 2 * K) * D, std=2.0)
        s["q"] = packed[:, :H * D].view(n, H, D)
        s["k"] = packed[:, H * D:(H + K) * D].view(n, K, D)
        s["v"] = packed[:, (H + K) * D:].view(n, K, D)
        s["q_weight"] = (1 + 0.2 * randn(D)) if case["norm"] else None
        s["k_weight"] = (1 + 0.2 * randn(D)) if case["norm"] else None
        s["rotation"] = _rotation(case, case["positions"] if case["op"] == "rotate" else case["context"])
        s["q_out"] = torch.empty((n, H, D), device="cuda", dtype=dtype)
    if case["op"] == "rotate":
        s["positions"] = torch.randint(0, case["positions"], (n,), device="cuda", dtype=torch.int32, generator=gen)
        s["k_out"] = torch.empty((n, K, D), device="cuda", dtype=dtype)
    elif case["op"] == "append":
        counts, lengths = _append_lengths(case)
        B, T = case["batch"], case["page"]
        width = -(-case["context"] // T)
        pages = B * width
        s["table"] = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32).view(B, width)
        s["lengths"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
        indptr = np.concatenate(([0], np.cumsum(counts)))
        s["indptr"] = None if case["chunk"] == 1 and not case["ragged"] else \
            torch.tensor(indptr, device="cuda", dtype=torch.int32)
        s["k_cache"], s["v_cache"] = randn(pages, T, K, D), randn(pages, T, K, D)
    else:
        lengths, shares = _prefix_lengths(case)
        B, T, P = case["batch"], case["page"], case["prefix"]
        rng = np.random.default_rng(seed)
        total = -(-lengths // T)
        first = np.where(shares, P // T, 0)                  # pages of its own start here
        mine = total - first
        pool = rng.permutation(int(mine.sum()) + P // T).astype(np.int32)
        width = max(1, int(total.max()))
        table = np.full((B, width), -1, dtype=np.int32)
        table[shares, :P // T] = pool[:P // T]
        column = np.arange(width)[None, :]
        table[(column >= first[:, None]) & (column < total[:, None])] = pool[P // T:]
        s["q"] = randn(B, H, D)
        s["k"], s["v"] = randn(pool.size, T, K, D), randn(pool.size, T, K, D)
        s["host_table"], s["host_lengths"] = table, lengths.astype(np.int32)
        s["table"] = torch.tensor(table, device="cuda")
        s["lengths"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    if own:
        _package()
        from paged_decode.layout import Layout
        if case["op"] == "prefix":
            from paged_decode.prefix import SharedPrefixPlan
            layout = Layout(case["batch"], H, K, D, case["page"], s["k"].shape[0])
            s["plan"] = SharedPrefixPlan(layout, s["host_table"], s["host_lengths"], dtype=dtype)
        else:
            from paged_decode.rotary import CacheAppend, HeadRotation
            rotation = HeadRotation(D, s["rotation"], interleaved=case["interleaved"], q_weight=s["q_weight"],
                                    k_weight=s["k_weight"])
            s["plan"] = rotation
            if case["op"] == "append":
                layout = Layout(case["batch"], H, K, D, case["page"], s["k_cache"].shape[0])
                s["plan"] = CacheAppend(layout, rotation)
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"append": _plain_append, "rotate": _plain_rotate, "prefix": _plain_prefix}[s["case"]["op"]](s)


def _run_own(s):
    op, plan = s["case"]["op"], s["plan"]
    if op == "prefix":
        return plan.run(s["q"], s["k"], s["v"])
    if op == "rotate":
        q, k = plan.run(s["q"], s["k"], s["positions"], q_out=s["q_out"], k_out=s["k_out"])
        return {"q": q, "k": k}
    q = plan.run(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], q=s["q"],
                 indptr=s["indptr"], q_out=s["q_out"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _norm_rotate(x, weight, cos_sin, interleaved):
    """x [n, heads, D]; cos_sin [n, rotary]."""
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
    r = cos_sin.shape[1]
    c, s = cos_sin[:, None, :r // 2], cos_sin[:, None, r // 2:]
    turn, rest = y[..., :r], y[..., r:]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = turn[..., :r // 2], turn[..., r // 2:]
        turn = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turn, rest), -1).to(x.dtype)


def _plain_rotate(s):
    cos_sin = s["rotation"][s["positions"].long()]
    inter = s["case"]["interleaved"]
    return {"q": _norm_rotate(s["q"], s["q_weight"], cos_sin, inter),
            "k": _norm_rotate(s["k"], s["k_weight"], cos_sin, inter)}


def _plain_append(s):
    case, T = s["case"], s["case"]["page"]
    i = torch.arange(s["q"].shape[0], device="cuda")
    if s["indptr"] is None:
        seq, position = i, s["lengths"].long() - 1
    else:
        indptr = s["indptr"].long()
        seq = torch.searchsorted(indptr[1:].contiguous(), i, right=True)
        position = s["lengths"].long()[seq] - indptr[seq + 1] + i
    page = s["table"][seq, position // T].long()
    cos_sin = s["rotation"][position]
    s["k_cache"][page, position % T] = _norm_rotate(s["k"], s["k_weight"], cos_sin, case["interleaved"])
    s["v_cache"][page, position % T] = s["v"]
    return {"q": _norm_rotate(s["q"], s["q_weight"], cos_sin, case["interleaved"]),
            "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_prefix(s):
    case = s["case"]
    B, H, K, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    pages = s["table"].clamp(min=0).long()
    k = s["k"][pages].float().view(B, -1, K, D).permute(0, 2, 3, 1)          # [B, K, D, L]
    q = s["q"].float().view(B, K, H // K, D) / math.sqrt(D)
    scores = torch.matmul(q, k)
    del k
    live = torch.arange(scores.shape[-1], device="cuda") < s["lengths"][:, None]
    live = live[:, None, None, :]
    top = scores.masked_fill(~live, -math.inf).amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.where(live, torch.exp(scores - top), 0.0)
    total = p.sum(-1, keepdim=True)
    v = s["v"][pages].float().view(B, -1, K, D).permute(0, 2, 1, 3)          # [B, K, L, D]
    out = torch.matmul(p, v) / total.clamp(min=1e-30)                        # an empty sequence gives zeros
    return out.view(B, H, D).to(s["q"].dtype)


# ---------------------------------------------------------------- 64 bits, from the definitions
def _exact_heads(x, weight, positions, case):
    """Each pair of a head row as one complex number, turned by its position's angle row."""
    r, x = case["rotary"], x.double().clone()
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * weight.double()
    table = case["table"].double()
    turn = torch.complex(table[positions, :r // 2], table[positions, r // 2:]).unsqueeze(1)
    step = slice(0, r, 2) if case["interleaved"] else slice(0, r // 2)
    mate = slice(1, r, 2) if case["interleaved"] else slice(r // 2, r)
    z = torch.complex(x[..., step].contiguous(), x[..., mate].contiguous()) * turn
    x[..., step], x[..., mate] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prefix":
        K, D = case["kv_heads"], case["dim"]
        out = torch.zeros((case["batch"], case["heads"], D), device="cuda", dtype=torch.float64)
        for b, length in enumerate(s["host_lengths"].tolist()):
            if length == 0:
                continue
            pages = s["table"][b, : -(-length // case["page"])].long()
            k = s["k"][pages].flatten(0, 1)[:length].double().transpose(0, 1)        # [K, L, D]
            v = s["v"][pages].flatten(0, 1)[:length].double().transpose(0, 1)
            q = s["q"][b].double().view(K, -1, D)
            weights = torch.softmax(q @ k.mT / D ** 0.5, -1)
            out[b] = (weights @ v).reshape(-1, D)
        return out
    case = dict(case, table=s["rotation"])
    if case["op"] == "rotate":
        at = s["positions"].long()
        return {"q": _exact_heads(s["q"], s["q_weight"], at, case), "k": _exact_heads(s["k"], s["k_weight"], at, case)}
    counts, lengths = _append_lengths(case)
    at = np.concatenate([np.arange(m - n, m) for n, m in zip(counts, lengths)])
    seq = np.repeat(np.arange(case["batch"]), counts)
    at, seq = torch.tensor(at, device="cuda"), torch.tensor(seq, device="cuda")
    slot = s["table"][seq, at // case["page"]].long() * case["page"] + at % case["page"]
    q, k = _exact_heads(s["q"], s["q_weight"], at, case), _exact_heads(s["k"], s["k_weight"], at, case)
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    k_cache.flatten(0, 1)[slot] = k
    v_cache.flatten(0, 1)[slot] = s["v"].double()
    return {"q": q, "k_cache": k_cache, "v_cache": v_cache}
