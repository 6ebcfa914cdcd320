"""Shared-prefix decode: what the sums of a row have to keep."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("NVIDIA GPU required", allow_module_level=True)

from paged_decode.layout import Layout
from paged_decode.prefix import SharedPrefixPlan

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("batch,heads,kv,D,page,pages", [
    (5, 32, 8, 128, 16, 3), (9, 8, 1, 64, 32, 40), (40, 40, 8, 128, 32, 64), (3, 64, 2, 64, 16, 700)])
def test_a_row_is_an_average_of_its_values(dtype, batch, heads, kv, D, page, pages):
    """Equal values come out as they went in, whatever the weights: numerator and denominator hold the
    same weights.  A piece's sums are FP32 chains of fewer than 2^11 terms, off by less than 2^-13 of
    themselves: FP16 rows then round to the value itself, and FP32 rows stay that near."""
    gen = torch.Generator("cuda").manual_seed(batch)
    q = 6 * torch.randn((batch, heads, D), device="cuda", dtype=dtype, generator=gen)   # a few tokens count
    k = torch.randn((pages, page, kv, D), device="cuda", dtype=dtype, generator=gen)
    v = torch.full_like(k, 1.9)
    v[..., 1::2] = -0.95
    table = np.tile(np.random.default_rng(0).permutation(pages), (batch, 1)).astype(np.int32)
    lengths = np.full(batch, pages * page, dtype=np.int32)
    plan = SharedPrefixPlan(Layout(batch, heads, kv, D, page, pages), table, lengths,
                            prefixes=[(np.arange(batch), pages)], dtype=dtype)
    out, want = plan.run(q, k, v), v[0, 0, 0].expand(batch, heads, D)
    if dtype == F16:
        assert torch.equal(out, want), (out - want).abs().max()
    else:
        torch.testing.assert_close(out, want, rtol=2.0 ** -13, atol=0)
    assert plan.read_errors() == 0
