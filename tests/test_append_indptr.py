"""CacheAppend with token ranges that do not start at token 0."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("NVIDIA GPU required", allow_module_level=True)

from paged_decode import _native
from paged_decode.layout import Layout
from paged_decode.rotary import CacheAppend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("row", [256, 257])                  # whole aligned rows one after another, or not
@pytest.mark.parametrize("first", [0, 1, 5, 40])
def test_tokens_before_the_first_range_belong_to_no_sequence(dtype, row, first):
    """They are skipped and flagged, like other tokens without a place, and sequence 0 keeps its earlier rows."""
    page, kv, heads, D, counts, lengths = 16, 1, 2, 64, [3, 0, 20], [60, 7, 33]
    tokens = first + sum(counts) + 4                         # four padding tokens behind
    packed = torch.randn((tokens, row), device="cuda").to(dtype)
    q, k, v = (packed[:, a: a + 64 * n].view(tokens, n, D) if row % 4 == 0 else
               packed[:, a: a + 64 * n].unflatten(1, (n, D)) for a, n in ((0, 2), (128, 1), (192, 1)))
    table = torch.randperm(12, device="cuda").to(torch.int32).view(3, 4)
    kc, vc = (torch.zeros((12, page, kv, D), device="cuda", dtype=dtype) for _ in range(2))
    op = CacheAppend(Layout(3, heads, kv, D, page, 12))
    ends = torch.tensor(first + np.concatenate(([0], np.cumsum(counts))), device="cuda", dtype=torch.int32)
    out = op.run(k, v, kc, vc, table, torch.tensor(lengths, device="cuda", dtype=torch.int32), q=q, indptr=ends)
    assert op.read_errors() == (_native.PD_DEVERR_LENGTH if first else 0)
    want_k, want_v, want_q, i = torch.zeros_like(kc), torch.zeros_like(vc), torch.zeros_like(out), first
    for b, (n, m) in enumerate(zip(counts, lengths)):
        for t in range(m - n, m):
            at = int(table[b, t // page]), t % page
            want_k[at], want_v[at], want_q[i] = k[i], v[i], q[i]
            i += 1
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v) and torch.equal(out, want_q)
