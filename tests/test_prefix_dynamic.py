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
