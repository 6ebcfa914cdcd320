"""A decode loop of sequences behind one prompt: append with rotation, then shared-prefix attention.

    python paged-decode-lab_b200/examples/shared_prefix_loop.py [--batch 64] [--prompt 4096] [--steps 32]

One attention layer with random weights.  The prompt's keys and values go into the
paged cache once; every sequence's page table starts with its pages.  A step
projects the hidden states, norms and rotates queries and keys and appends keys and
values (``CacheAppend``), attends (``SharedPrefixPlan.run_dynamic``) and projects back.
It is captured in one CUDA graph and replayed.  The last step's attention is checked
against a plain FP64 computation, and the step is timed with sharing and without.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

import numpy as np
import torch

from paged_decode.layout import Layout
from paged_decode.prefix import SharedPrefixPlan
from paged_decode.rotary import CacheAppend, HeadRotation, rotation_table


def run(batch=64, prompt=4096, steps=32, heads=32, kv_heads=8, dim=128, page=16, seed=0):
    """Returns the largest error of the last step and the microseconds of a step, shared and not."""
    gen = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return torch.randn(shape, device="cuda", dtype=torch.float16, generator=gen) * scale

    prompt = prompt // page * page                   # whole pages are shared
    shared, own = prompt // page, -(-steps // page)
    pages = shared + batch * own
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table = np.concatenate([np.tile(order[:shared], (batch, 1)), order[shared:].reshape(batch, own)], axis=1)
    layout = Layout(batch, heads, kv_heads, dim, page, pages)
    k_cache, v_cache = (torch.zeros((pages, page, kv_heads, dim), device="cuda", dtype=torch.float16) for _ in range(2))
    width = heads * dim
    w_qkv = randn(width, (heads + 2 * kv_heads) * dim, scale=width ** -0.5)
    w_out = randn(width, width, scale=width ** -0.5)
    rotation = HeadRotation(dim, rotation_table(prompt + steps, dim), q_weight=1 + 0.1 * randn(dim),
                            k_weight=1 + 0.1 * randn(dim))

    def split(qkv):
        rows = qkv.view(qkv.shape[0], heads + 2 * kv_heads, dim)
        return rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]

    # the prompt, once: one sequence whose last `prompt` tokens these are
    _, k, v = split(randn(prompt, width) @ w_qkv)
    filler = CacheAppend(Layout(1, heads, kv_heads, dim, page, pages), rotation)
    filler.run(k, v, k_cache, v_cache, torch.tensor(order[None, :shared], device="cuda"),
               torch.tensor([prompt], device="cuda", dtype=torch.int32),
               indptr=torch.tensor([0, prompt], device="cuda", dtype=torch.int32))

    start = np.full(batch, prompt, dtype=np.int32)
    append = CacheAppend(layout, rotation)
    dev_table = torch.tensor(table, device="cuda")
    result = {}
    for name, prefixes in (("shared", [(np.arange(batch), shared)]), ("apart", [])):
        plan = SharedPrefixPlan(layout, table, start, prefixes=prefixes, max_lengths=start + steps)
        lengths = torch.tensor(start, device="cuda")
        hidden = torch.ones((batch, width), device="cuda", dtype=torch.float16)
        q_rotated = torch.empty((batch, heads, dim), device="cuda", dtype=torch.float16)

        def step():
            lengths.add_(1)
            q, k, v = split(hidden @ w_qkv)
            append.run(k, v, k_cache, v_cache, dev_table, lengths, q=q, q_out=q_rotated)
            out = plan.run_dynamic(q_rotated, k_cache, v_cache, dev_table, lengths)
            hidden.copy_(torch.tanh(out.view(batch, width) @ w_out))
            return out

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(steps - 1):                   # (the capture ran nothing)
            graph.replay()
        end.record()
        torch.cuda.synchronize()
        result[f"{name}_us"] = 1000 * begin.elapsed_time(end) / (steps - 1)
        worst = 0.0
        for b in range(0, batch, max(1, batch // 4)):
            ids = torch.tensor(table[b].astype(np.int64), device="cuda")
            kk, vv = (c[ids].flatten(0, 1)[:prompt + steps].double().transpose(0, 1) for c in (k_cache, v_cache))
            s = q_rotated[b].double().view(kv_heads, -1, dim) @ kk.mT / dim ** 0.5
            want = (torch.softmax(s, -1) @ vv).view(heads, dim)
            worst = max(worst, (out[b].double() - want).abs().max().item())
        result[f"{name}_error"] = worst
        if append.read_errors() or plan.read_errors():
            raise RuntimeError("the device error word is set")
    return result


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for flag, value in (("--batch", 64), ("--prompt", 4096), ("--steps", 32)):
        ap.add_argument(flag, type=int, default=value)
    r = run(**vars(ap.parse_args()))
    print(f"step with a shared prefix {r['shared_us']:.1f} us, without {r['apart_us']:.1f} us; "
          f"largest error {max(r['shared_error'], r['apart_error']):.2g}")
