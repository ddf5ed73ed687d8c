"""Attention of few rows over pages in 8 bits where rows of V differ much in size: the error is that of the probabilities in
fp16, whatever the size of rows of little weight."""

import math

import pytest
import torch

from .paged_support import paged_batch, within
from .sparse_support import held, pack_pages

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _exact(q, k, v, table, kv_lens, new, causal):
    """Output in 64 bits and its bound. A weight is off by half a step of fp16 (2^-11 of it), and by what moves its exponent: the
    scores' FP32 products (2^-22 of the sum of magnitudes a step, as for pages in 16 bits), 2^-17 of the addend log2 scale - unit
    (below 256 in magnitude, half a step of FP32) and the exponential's own 2^-22. Below 2^-14 of fp16's range the step is 2^-24:
    half of it is 2^-32 of the largest weight, which is 2^7 at least, for each key; a code is 448 at most and a row's largest 224 at
    least, so for n keys that is n 2^-31 of the largest (probability x largest magnitude of its row). The output is
    rounded once."""
    page, kv_heads, d = k.shape[1:]
    out_unit = 2.0 ** -11 if q.dtype == FP16 else 2.0 ** -8
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    first = 0
    for s, n in enumerate(new):
        total = int(kv_lens[s])
        at = table[s][:-(-total // page)].long()
        ks, vs = (x[at].flatten(0, 1)[:total].double() for x in (k, v))
        last = torch.arange(total - n, total, device=q.device) if causal else torch.full((n,), total - 1, device=q.device)
        seen = torch.arange(total, device=q.device) <= last[:, None]
        for h in range(q.shape[1]):
            x, kh, vh = q[first:first + n, h].double(), ks[:, h * kv_heads // q.shape[1]], vs[:, h * kv_heads // q.shape[1]]
            p = torch.softmax((x @ kh.T / math.sqrt(d)).masked_fill(~seen, -math.inf), dim=1)
            rows = slice(first, first + n)
            out[rows, h] = p @ vh
            noise = (x.abs() @ kh.abs().T / math.sqrt(d)).amax(dim=1, keepdim=True) * (d / 16 + 8) * 2.0 ** -22 + 2.0 ** -17 + total * 2.0 ** -24
            weight = p @ vh.abs()
            largest = (p * vh.abs().amax(dim=1)).amax(dim=1, keepdim=True)
            bound[rows, h] = (2.0 ** -11 * 1.01 + 2.0 * noise) * weight + total * 2.0 ** -31 * largest + out_unit * 1.01 * out[rows, h].abs()
            if q.dtype == FP16:
                bound[rows, h] += 2.0 ** -25
        first += n
    return out, bound


def _check(new, totals, heads, kv_heads, d, dtype, change, *, causal=True, page=16, seed=0):
    """``change(k, v, table)`` changes the rows (FP32) before they are packed."""
    from reelcache_b200.ops import paged
    g = torch.Generator(device="cuda").manual_seed(seed + sum(totals) + d)
    k, v, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, page, torch.float32)
    q = torch.randn(sum(new), heads, d, generator=g, device="cuda").to(dtype)
    q[..., 0] = 8.0
    k[..., 0] = 0.0  # (so that change can set any score)
    change(k, v, table)
    packed = [pack_pages(x, dtype) for x in (k, v)]
    want, bound = _exact(q, *(held(p, dtype) for p in packed), table, kv_lens, new, causal)
    out = paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=max(new), causal=causal)
    assert within(out, want, bound)
    return q, packed, table, kv_lens, cu_q, out


# up to eight rows clustered and as a line, up to sixteen clustered and as a line of slices, slices clustered
FORMS = [([1], [1000], 4, 1), ([1] * 60, [900 + 7 * i for i in range(60)], 16, 8), ([3, 2], [1000, 777], 8, 2), ([5] * 30, [800 + 9 * i for i in range(30)], 24, 3),
         ([10], [1000], 4, 1)]


@pytest.mark.parametrize("steps,dtype", [(16, BF16), (20, BF16), (26, BF16), (60, BF16), (9, FP16)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,totals,heads,kv_heads", FORMS)
def test_a_large_row_of_no_weight(new, totals, heads, kv_heads, d, steps, dtype):
    """Key 3 has a row of V 2^steps larger and a score that leaves it a weight below e^-60 of the others' sum."""
    def change(k, v, table):
        at = table[:, 0].long()
        k[at, 3] = 0.0
        k[at, 3, :, 0] = -100.0 * math.sqrt(d / 64)
        v[at, 3] *= 2.0 ** steps
    _check(new, totals, heads, kv_heads, d, dtype, change)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,heads", [(2, 4), (4, 4), (4, 12)])
def test_a_large_row_that_only_later_tokens_see(new, heads, d):
    """The last new token's row of V is 2^30 larger: the tokens before it do not see it."""
    at = {}

    def change(k, v, table):
        at["last"] = (int(table[0, -1]), 499 % 16)
        v[at["last"]] *= 2.0 ** 30
    q, packed, table, kv_lens, cu_q, out = _check([new], [500], heads, 1, d, BF16, change)
    from reelcache_b200.ops import paged
    packed[1].codes.view(torch.uint8)[at["last"]] = 0  # without the row: the same within two bounds
    packed[1].scales.view(torch.uint8)[:, at["last"][0], at["last"][1]] = 127
    other = paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=new, causal=True)
    want, bound = _exact(q, *(held(p, BF16) for p in packed), table, kv_lens, [new], True)
    assert within(other, want, bound)
    assert within(out[:-1], other[:-1].double(), 2.0 * bound[:-1])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("new,totals,heads,kv_heads", FORMS)
def test_rows_of_all_sizes(new, totals, heads, kv_heads, causal):
    """Sizes over 2^40, in any order, and rising and falling along the sequence."""
    for kind in ("any", "rising", "falling"):
        def change(k, v, table):
            g = torch.Generator(device="cuda").manual_seed(len(kind))
            size = torch.randint(-20, 21, v.shape[:3], generator=g, device="cuda").float()
            if kind != "any":
                for s in range(table.shape[0]):
                    held_pages = table[s][table[s] >= 0].long()
                    ramp = torch.linspace(-20, 20, len(held_pages) * 16, device="cuda").round().view(-1, 16, 1)
                    size[held_pages] = ramp if kind == "rising" else -ramp
            v *= torch.exp2(size)[..., None]
        _check(new, totals, heads, kv_heads, 64, BF16, change, causal=causal)


@pytest.mark.parametrize("power", [-112, 112])
@pytest.mark.parametrize("new,totals,heads,kv_heads", FORMS)
def test_rows_at_the_ends_of_the_range(new, totals, heads, kv_heads, power):
    """All of V near the smallest and the largest numbers of bf16."""
    def change(k, v, table):
        v *= 2.0 ** power
    _check(new, totals, heads, kv_heads, 128, BF16, change)


@pytest.mark.parametrize("rise", [0.05, 0.5, 3.0])
@pytest.mark.parametrize("new,totals,heads,kv_heads", FORMS[:4])
def test_scores_that_rise_while_sizes_fall(new, totals, heads, kv_heads, rise):
    """Every key's score is higher than the one's before it, its row of V smaller: the maximum moves and the unit need not."""
    def change(k, v, table):
        for s in range(table.shape[0]):
            at = table[s][table[s] >= 0].long()
            step = torch.arange(len(at) * 16, device="cuda", dtype=torch.float32).view(-1, 16, 1)
            k[at] *= 0.1
            k[at, :, :, 0] = ((step - step.amax()) * rise).clamp(min=-200.0)
            v[at] *= torch.exp2(-step / 40.0)[..., None]
    _check(new, totals, heads, kv_heads, 64, BF16, change)


@pytest.mark.parametrize("new,totals,heads,kv_heads", FORMS)
def test_infinite_scores(new, totals, heads, kv_heads):
    """A score of plus infinity makes the log-sum-exp plus infinity and the output NaN; of minus infinity a key that counts for nothing."""
    from reelcache_b200.ops import paged
    g = torch.Generator(device="cuda").manual_seed(len(new))
    k, v, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, 64, 16, torch.float32)
    k[..., 0] = 0.0
    at = table[:, 0].long()
    k[at, 3, :, 0] = -4.0e4 * 64
    q = torch.zeros(sum(new), heads, 64, device="cuda", dtype=BF16)
    packed = [pack_pages(x, BF16) for x in (k, v)]
    below = q.clone()
    below[..., 0] = 2.0 ** 120
    above = q.clone()
    above[..., 0] = -(2.0 ** 120)
    call = lambda x: paged.attention(x, *packed, table, kv_lens, cu_q, max_q_len=max(new), causal=True, return_lse=True)  # noqa: E731
    out, lse = call(above)
    assert bool(out.isnan().all()) and bool((lse == math.inf).all())
    # every key but the one of minus infinity scores zero
    out, lse = call(below)
    values = held(packed[1], BF16).double()
    first = 0
    for s, n in enumerate(new):
        total = totals[s]
        rows = values[table[s][:-(-total // 16)].long()].flatten(0, 1)[:total]
        for i in range(n):
            seen = [p for p in range(total - n + i + 1) if p != 3]
            want = rows[seen].mean(dim=0).repeat_interleave(heads // kv_heads, dim=0)
            size = rows[seen].abs().mean(dim=0).repeat_interleave(heads // kv_heads, dim=0)
            # equal weights, a power of two times V's scales: exact in fp16; sums in FP32 and one rounding
            assert within(out[first + i], want, want.abs() * 2.0 ** -8 + size * (len(seen) + 8) * 2.0 ** -22)
            assert within(lse[first + i], torch.full_like(lse[first + i], math.log(len(seen))).double(), torch.full_like(lse[first + i], 2.0 ** -18).double())
        first += n
