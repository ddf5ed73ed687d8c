"""The rotation on the way into pages in 8 bits: the same queries as on the way into 16-bit pages, keys rounded once."""

import math

import pytest
import torch

from .paged_support import paged_batch, rotate_bound, spun, within
from .sparse_support import RANGE

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


def _code(x, power):
    """The nearest e4m3 number to ``x * 2^-power`` (64 bits, ties to even)."""
    x = (x * torch.exp2(-power.double())[..., None]).clamp(-448.0, 448.0)
    step = torch.exp2(torch.frexp(x.abs().clamp(min=2.0 ** -6))[1].double() - 4.0)
    return torch.round(x / step) * step


def _power(top, dtype):
    """The exponent of a row's scale for its largest magnitude."""
    low, high = RANGE[dtype]
    part, power = torch.frexp(top)
    return torch.where(top > 0, power - 9 + (part > 0.875), low).clamp(low, high)


def _check_codes(codes, power, want, off, dtype):
    """Codes of the exact rows ``want`` wherever those are further than ``off`` from where rounding changes, and no others than the two
    next to it elsewhere; scales likewise. Returns how many codes are not the exact rows'."""
    top = want.abs().amax(dim=-1)
    edge = off.amax(dim=-1)
    assert bool(((power >= _power((top - edge).clamp(min=0.0), dtype)) & (power <= _power(top + edge, dtype))).all())
    assert bool(((codes >= _code(want - off, power)) & (codes <= _code(want + off, power))).all())
    return int((codes != _code(want, power)).sum())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("tokens,kv_heads,d", [(1, 3, 64), (700, 4, 64), (4680, 12, 128)])
def test_codes_of_rotated_keys(tokens, kv_heads, d, layout, dtype):
    """A rotated number is off by two roundings to FP32 of at most 2^-24 of |a| + |b| each (the sines' two parts hold 2^-48), and
    then rounded to its code once, to no 16-bit type between. So a code can differ from the exact one's only where the exact number
    lies within 2^-23 of |a| + |b| of a border between two codes. Borders are a step apart: of numbers that lie anywhere between
    them, 2 off / step do at most."""
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = torch.Generator(device="cuda").manual_seed(tokens)
    rope = AxisRope.wan(d, layout=layout)
    *_, table, kv_lens, cu_q = paged_batch(g, [tokens], [tokens], 1, 64, 24, BF16)
    pages = [paged.PackedPages.empty(int(table.max()) + 1, 24, kv_heads, d, "cuda") for _ in range(2)]
    q, k, v = (torch.randn(tokens, kv_heads, d, generator=g, device="cuda").to(dtype) for _ in range(3))
    positions = torch.randint(0, 4000, (tokens, 3), generator=g, device="cuda", dtype=torch.int32)
    paged.append(q, k, v, positions, rope, *pages, table, kv_lens, cu_q)
    at = torch.arange(tokens, device="cuda")
    place = table[0].long()[at // 24], at % 24
    codes = pages[0].codes[place].float().double()
    power = pages[0].scales.view(torch.uint8)[:, place[0], place[1]].T.to(torch.int32) - 127
    want, size = spun(k, positions, rope.sections, 10000.0, layout)
    off = size * 2.0 ** -23
    differ = _check_codes(codes, power, want, off, dtype)
    scaled = (want * torch.exp2(-power.double())[..., None]).abs().clamp(min=2.0 ** -6)
    most = float((2.0 * off * torch.exp2(-power.double())[..., None] / torch.exp2(torch.frexp(scaled)[1].double() - 4.0)).sum())
    assert differ <= most + 6.0 * math.sqrt(most) + 6.0
    # what the check is there for: rows rounded to 16 bits first, and sines of 2^-21, would not pass it
    if tokens > 1:
        for wrong in (want.to(dtype).double(), want + size * 2.0 ** -19 * (torch.rand(want.shape, generator=g, device="cuda", dtype=torch.float64) - 0.5)):
            with pytest.raises(AssertionError):
                _check_codes(_code(wrong, power), power, want, off, dtype)
