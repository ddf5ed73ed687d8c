"""The rotation on the way into pages in 8 bits: the same queries as on the way into 16-bit pages, keys rounded once."""

import math

import pytest
import torch

from .paged_support import paged_batch, rotate_bound, spun, within

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("new,heads,kv_heads,d", [([1], 8, 2, 128), ([40, 7], 3, 3, 64), ([900] * 3, 12, 12, 128)])
def test_queries_that_are_not_finite(new, heads, kv_heads, d, layout, dtype):
    """Infinities and NaN of q come out as they do beside 16-bit pages."""
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = torch.Generator(device="cuda").manual_seed(d)
    rope = AxisRope.wan(d, layout=layout)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, new, new, kv_heads, d, 16, dtype)
    packed = [paged.PackedPages.empty(len(k_pages), 16, kv_heads, d, "cuda") for _ in range(2)]
    tokens = sum(new)
    q, k, v = (torch.randn(tokens, h, d, generator=g, device="cuda").to(dtype) for h in (heads, kv_heads, kv_heads))
    where = torch.rand(q.shape, generator=g, device="cuda")
    q[where < 0.05] = math.inf
    q[where > 0.95] = -math.inf
    q[(where > 0.5) & (where < 0.52)] = math.nan
    positions = torch.randint(1, 4000, (tokens, 3), generator=g, device="cuda", dtype=torch.int32)
    got = paged.append(q, k, v, positions, rope, *packed, table, kv_lens, cu_q)
    want = paged.append(q, k, v, positions, rope, k_pages, v_pages, table, kv_lens, cu_q)
    assert bool(want.isinf().any()) and bool(want.isnan().any()) and bool(want.isfinite().any())
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.masked_fill(~got.isinf(), 0.0), want.masked_fill(~want.isinf(), 0.0))
    exact, size = spun(q, positions, rope.sections, 10000.0, layout)
    both = want.isfinite()
    assert within(got[both], exact[both], rotate_bound(exact, size, dtype)[both])
