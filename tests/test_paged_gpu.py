"""Multi-axis rotary positions, paged append, paged attention and the page table on sm_100a, against 64-bit forms."""

import math

import pytest
import torch

from .paged_support import ListTable, attend, paged_batch, rotate_bound, spun, within

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _positions(g, tokens, axes, most=4000):
    return torch.randint(0, most, (tokens, axes), generator=g, device="cuda", dtype=torch.int32)


# -- rotation ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("tokens,heads,kv_heads,d,sections", [
    (1, 1, 1, 16, (8,)), (7, 3, 1, 128, (22, 21, 21)), (333, 12, 12, 128, (22, 21, 21)), (129, 5, 2, 64, (12, 10, 10)),
    (65, 8, 2, 80, (10, 10, 10, 10)), (3000, 16, 4, 256, (44, 42, 42)), (2, 1, 1, 128, (0, 64))])
def test_rotate_matches_64_bits(tokens, heads, kv_heads, d, sections, dtype, layout):
    from reelcache_b200.ops.rope import AxisRope, rotate
    g = _gen(tokens + d)
    rope = AxisRope(d, sections, layout=layout)
    q = torch.randn(tokens, heads, d, generator=g, device="cuda").to(dtype)
    k = torch.randn(tokens, kv_heads, d, generator=g, device="cuda").to(dtype)
    positions = _positions(g, tokens, len(sections))
    for got, x in zip(rotate(q, k, positions, rope), (q, k)):
        want, size = spun(x, positions, sections, 10000.0, layout)
        assert got.dtype == dtype and got.is_contiguous()
        assert within(got, want, rotate_bound(want, size, dtype))
    alone, none = rotate(q, None, positions, rope)
    assert none is None and torch.equal(alone, rotate(q, k, positions, rope)[0])


@pytest.mark.parametrize("top,kind", [(1_000_000, torch.int32), (16_000_000, torch.int32), (1_000_000, FP32)])
def test_rotate_far_positions(top, kind):
    """The angle does not lose bits with the position (a product in FP32 radians would be off by tenths of a radian)."""
    from reelcache_b200.ops.rope import AxisRope, rotate
    g = _gen(3)
    rope = AxisRope.wan(128)
    q = torch.randn(64, 2, 128, generator=g, device="cuda")
    positions = (torch.rand(64, 3, generator=g, device="cuda") * top).to(kind)
    got, _ = rotate(q, None, positions, rope)
    want, size = spun(q, positions, rope.sections, 10000.0, "interleaved")
    assert within(got, want, rotate_bound(want, size, FP32))


@pytest.mark.parametrize("layout", ["interleaved", "halves"])
def test_rotate_strided_rows_and_empty(layout):
    from reelcache_b200.ops.rope import AxisRope, rotate
    g = _gen(4)
    rope = AxisRope.wan(64, layout=layout)
    fused = torch.randn(50, 7, 64, generator=g, device="cuda").bfloat16()
    q, k, _ = fused.split([4, 2, 1], dim=1)
    positions = _positions(g, 50, 3)
    got = rotate(q, k, positions, rope)
    dense = rotate(q.contiguous(), k.contiguous(), positions, rope)
    assert all(torch.equal(a, b) for a, b in zip(got, dense))
    by_head = q.contiguous().transpose(0, 1).contiguous().transpose(0, 1)  # heads outside of tokens in memory
    assert torch.equal(rotate(by_head, None, positions, rope)[0], dense[0])
    odd = torch.randn(50, 4, 66, generator=g, device="cuda").bfloat16()[..., 1:65]  # unaligned rows are copied
    assert torch.equal(rotate(odd, None, positions, rope)[0], rotate(odd.contiguous(), None, positions, rope)[0])
    empty, _ = rotate(q[:0], None, positions[:0], rope)
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_rotate_gradient_is_the_formulas(dtype, layout):
    from reelcache_b200.ops.rope import AxisRope, rotate
    g = _gen(5)
    sections = (22, 21, 21)
    rope = AxisRope(128, sections, layout=layout)
    q = torch.randn(97, 6, 128, generator=g, device="cuda").to(dtype).requires_grad_()
    k = torch.randn(97, 2, 128, generator=g, device="cuda").to(dtype).requires_grad_()
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    positions = _positions(g, 97, 3)
    out = rotate(q, k, positions, rope)
    for got, d in zip(torch.autograd.grad(out, (q, k), (dq, dk)), (dq, dk)):
        want, size = spun(d, positions, sections, 10000.0, layout, -1.0)
        assert within(got, want, rotate_bound(want, size, dtype))


@pytest.mark.parametrize("layout", ["interleaved", "halves"])
def test_rotate_gradient_against_differences(layout):
    """f(x) = <w, rotate(x)> is linear: its central difference along a direction is exact up to the FP32 rounding of the
    outputs, 2^-20 of the summed magnitudes (times 1/h for the difference of two values)."""
    from reelcache_b200.ops.rope import AxisRope, rotate
    g = _gen(6)
    rope = AxisRope.wan(64, layout=layout)
    q = torch.randn(31, 3, 64, generator=g, device="cuda", requires_grad=True)
    k = torch.randn(31, 1, 64, generator=g, device="cuda", requires_grad=True)
    positions = _positions(g, 31, 3)
    wq, wk = torch.randn_like(q), torch.randn_like(k)
    tq, tk = torch.randn_like(q), torch.randn_like(k)

    def f(a, b):
        x, y = rotate(a, b, positions, rope)
        return float((x.double() * wq.double()).sum() + (y.double() * wk.double()).sum())

    gq, gk = torch.autograd.grad(rotate(q, k, positions, rope), (q, k), (wq, wk))
    slope = float((gq.double() * tq.double()).sum() + (gk.double() * tk.double()).sum())
    h = 0.5
    with torch.no_grad():
        got = (f(q + h * tq, k + h * tk) - f(q - h * tq, k - h * tk)) / (2 * h)
    size = float((wq.abs() * (q.detach().abs() + tq.abs())).sum() + (wk.abs() * (k.detach().abs() + tk.abs())).sum())
    assert abs(got - slope) <= 4 * size * 2.0 ** -20 / h


def test_rotate_gradient_of_one_output_broadcast_and_twice():
    from reelcache_b200.ops.rope import AxisRope, rotate
    g = _gen(7)
    rope = AxisRope.wan(64)
    positions = _positions(g, 20, 3)
    q = torch.randn(20, 4, 64, generator=g, device="cuda", requires_grad=True)
    shared = torch.randn(20, 1, 64, generator=g, device="cuda", requires_grad=True)
    # a key head shared by four: the gradient adds up over the heads that saw it
    out_q, out_k = rotate(q, shared.expand(20, 4, 64), positions, rope)
    dk = torch.randn(20, 4, 64, generator=g, device="cuda")
    (got,) = torch.autograd.grad(out_k, shared, dk, retain_graph=True)
    want, size = spun(dk, positions, rope.sections, 10000.0, "interleaved", -1.0)
    assert within(got, want.sum(1, keepdim=True), 4 * rotate_bound(want, size, FP32).sum(1, keepdim=True))
    # a gradient that is expanded (stride 0), of q alone
    (gq,) = torch.autograd.grad(out_q.sum(), q, retain_graph=True)
    want, size = spun(torch.ones_like(q), positions, rope.sections, 10000.0, "interleaved", -1.0)
    assert within(gq, want, rotate_bound(want, size, FP32))
    # the gradient's gradient turns forward again
    w = torch.randn_like(q, requires_grad=True)
    (first,) = torch.autograd.grad(out_q, q, w, create_graph=True)
    (second,) = torch.autograd.grad(first, w, torch.ones_like(first))
    want, size = spun(torch.ones_like(q), positions, rope.sections, 10000.0, "interleaved")
    assert within(second, want, rotate_bound(want, size, FP32))


def test_rotate_on_another_stream():
    from reelcache_b200.ops.rope import AxisRope, rotate
    g = _gen(8)
    rope = AxisRope.wan(128)
    q = torch.randn(500, 12, 128, generator=g, device="cuda").bfloat16()
    positions = _positions(g, 500, 3)
    want, _ = rotate(q, None, positions, rope)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got, _ = rotate(q, None, positions, rope)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


def test_rotate_refusals():
    from reelcache_b200.errors import ConfigurationError, UnsupportedError
    from reelcache_b200.ops.rope import AxisRope, rotate
    rope = AxisRope.wan(64)
    q = torch.randn(4, 2, 64, device="cuda")
    positions = torch.zeros(4, 3, dtype=torch.int32, device="cuda")
    with pytest.raises(ConfigurationError):
        rotate(torch.randn(4, 2, 128, device="cuda"), None, positions, rope)
    with pytest.raises(UnsupportedError):
        rotate(q.cpu(), None, positions.cpu(), rope)
    for bad_q, bad_k, bad_p in [(q, None, positions[:3]), (q, None, positions[:, :2].contiguous()), (q, None, positions.long()),
                                (q, q[:3], positions), (q, q.half(), positions), (q.double(), None, positions),
                                (q, None, positions.cpu())]:
        with pytest.raises(RuntimeError):
            rotate(bad_q, bad_k, bad_p, rope)


# -- append -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("pages_layout", ["nhd", "hnd"])
@pytest.mark.parametrize("new,totals,heads,kv_heads,d,page,layout", [
    ([1], [1], 1, 1, 64, 8, "halves"), ([1, 1, 1], [17, 16, 1], 8, 2, 128, 16, "interleaved"),
    ([5, 0, 40], [5, 9, 73], 6, 3, 64, 24, "halves"), ([300, 100], [1600, 3120], 12, 12, 128, 1560, "interleaved"),
    ([2000], [2000], 4, 1, 80, 64, "interleaved")])
def test_append_writes_only_the_new_tokens(new, totals, heads, kv_heads, d, page, layout, dtype, pages_layout):
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = _gen(sum(totals))
    rope = AxisRope.wan(d, layout=layout)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, page, dtype, layout=pages_layout)
    fused = torch.randn(sum(new), heads + 2 * kv_heads, d, generator=g, device="cuda").to(dtype)
    q, k, v = fused.split([heads, kv_heads, kv_heads], dim=1)
    positions = _positions(g, sum(new), 3)
    want_k, want_v = k_pages.clone(), v_pages.clone()
    turned, size = spun(k, positions, rope.sections, 10000.0, layout)
    at = 0
    checked = []
    for s, (n, total) in enumerate(zip(new, totals)):
        for i in range(n):
            place = total - n + i
            checked.append((int(table[s, place // page]), place % page, at + i))
            want_v[checked[-1][0], place % page] = v[at + i]
        at += n
    out = paged.append(q, k, v, positions, rope, k_pages, v_pages, table, kv_lens, cu_q)
    want, qsize = spun(q, positions, rope.sections, 10000.0, layout)
    assert within(out, want, rotate_bound(want, qsize, dtype))
    assert torch.equal(v_pages, want_v)
    page_at, row_at, token_at = (torch.tensor(x, device="cuda") for x in zip(*checked))
    got = k_pages[page_at, row_at]
    assert within(got, turned[token_at], rotate_bound(turned, size, dtype)[token_at])
    want_k[page_at, row_at] = got
    assert torch.equal(k_pages, want_k)  # nothing else moved


def test_append_refusals():
    from reelcache_b200.errors import ConfigurationError, UnsupportedError
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = _gen(20)
    rope = AxisRope.wan(64)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [2], [10], 2, 64, 8, BF16)
    q, k = (torch.randn(2, n, 64, generator=g, device="cuda").bfloat16() for n in (4, 2))
    positions = _positions(g, 2, 3)
    call = lambda q=q, k=k, v=k, p=positions, kp=k_pages, vp=v_pages, t=table, n=kv_lens, c=cu_q, **kw: paged.append(  # noqa: E731
        q, k, v, p, rope, kp, vp, t, n, c, **kw)
    call()
    with pytest.raises(UnsupportedError):
        call(q=q.cpu())
    with pytest.raises(ConfigurationError):
        call(q=torch.randn(2, 4, 128, device="cuda").bfloat16())
    nine = torch.randn(5, 9, 2, 64, device="cuda").bfloat16()
    for wrong in (dict(q=q.float(), k=k.float(), v=k.float()), dict(k=k.half()), dict(k=k[:1]), dict(v=k[:, :1]), dict(p=positions.float()[:1]),
                  dict(p=positions[:, :2]), dict(kp=nine, vp=nine), dict(kp=k_pages[:, :, :1]), dict(vp=v_pages[1:]), dict(t=table.long()),
                  dict(n=kv_lens.cpu()), dict(c=cu_q[:1]), dict(q=q[..., 1:]), dict(out=q[:1].clone()), dict(q=q.clone().requires_grad_())):
        with pytest.raises((RuntimeError, ConfigurationError)):
            call(**wrong)


def test_append_out_of_range_is_reported_and_dropped(cuda_device):
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext, paged
    from reelcache_b200.ops.rope import AxisRope
    g = _gen(9)
    rope = AxisRope.wan(64)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [2, 2], [10, 20], 2, 64, 8, BF16)
    before = k_pages.clone(), v_pages.clone()
    q = torch.randn(4, 2, 64, generator=g, device="cuda").bfloat16()
    positions = _positions(g, 4, 3)
    for bad in (-1, k_pages.shape[0], 1 << 30):
        broken = table.clone()
        broken[0, 1] = bad
        broken[1, 2] = bad
        paged.append(q, q, q, positions, rope, k_pages, v_pages, broken, kv_lens, cu_q)
        with pytest.raises(DeviceStatusError, match="page number"):
            _ext.check_status(cuda_device)
        assert torch.equal(k_pages, before[0]) and torch.equal(v_pages, before[1])
    paged.append(q, q, q, positions, rope, k_pages, v_pages, table, torch.full_like(kv_lens, 10 ** 6), cu_q)
    with pytest.raises(DeviceStatusError):
        _ext.check_status(cuda_device)
    paged.append(q, q, q, positions, rope, k_pages, v_pages, table, torch.zeros_like(kv_lens), cu_q)  # before position 0
    with pytest.raises(DeviceStatusError):
        _ext.check_status(cuda_device)
    assert torch.equal(k_pages, before[0]) and torch.equal(v_pages, before[1])


# -- attention --------------------------------------------------------------------------------------------------------

def _check_attention(new, totals, heads, kv_heads, d, page, dtype, *, seed=0, layout="nhd", fill=None, scale=None, spread=1.0, **mask):
    from reelcache_b200.ops import _ext, paged
    g = _gen(seed + sum(totals) + d)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, page, dtype, layout=layout, fill=fill,
                                                         width_extra=2)
    q = (torch.randn(sum(new), heads, d, generator=g, device="cuda") * spread).to(dtype)
    out, lse = paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=max(max(new), 1), return_lse=True,
                               scale=scale, **mask)
    torch.cuda.synchronize()
    _ext.check_status(q.device)
    want, want_lse, bound, lse_bound = attend(q, k_pages, v_pages, table, kv_lens, new, scale=scale, **mask)
    assert within(out, want, bound), float(((out.double() - want).abs() - bound).max())
    assert within(lse, want_lse, lse_bound), float(((lse.double() - want_lse).abs() - lse_bound).nan_to_num().max())
    return out


TOKENS = [([1], [1]), ([1], [2]), ([1], [63]), ([1], [64]), ([1], [65]), ([1], [2049]), ([1] * 5, [7, 300, 1, 64, 1031]),
          ([1, 0, 1], [40, 50, 0 + 1]), ([1] * 40, [17 * i + 1 for i in range(40)])]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(1, 1, 64, 8), (8, 1, 128, 16), (12, 12, 128, 24), (10, 2, 64, 64), (6, 3, 128, 200)])
@pytest.mark.parametrize("new,totals", TOKENS)
def test_single_tokens(new, totals, heads, kv_heads, d, page, dtype):
    _check_attention(new, totals, heads, kv_heads, d, page, dtype, causal=True)


CHUNKS = [([2], [2]), ([3, 5], [3, 900]), ([17], [100]), ([40, 1, 7], [40, 513, 200]), ([128], [128]), ([129, 300], [700, 300]),
          ([500], [1777])]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads,d,page,dtype", [
    (1, 1, 64, 8, BF16), (4, 4, 128, 16, FP16), (8, 2, 128, 24, BF16), (5, 1, 64, 128, FP16), (6, 2, 128, 200, BF16),
    (40, 1, 64, 64, BF16), (3, 3, 128, 1560, BF16)])
@pytest.mark.parametrize("new,totals", CHUNKS)
def test_chunks(new, totals, heads, kv_heads, d, page, dtype, causal):
    _check_attention(new, totals, heads, kv_heads, d, page, dtype, causal=causal)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("new,totals,heads,kv_heads,d,page", [
    ([1100], [2000], 40, 40, 64, 64), ([900, 10, 333, 700], [3000, 2100, 333, 800], 20, 4, 128, 16),
    ([2900], [2900], 24, 8, 64, 32), ([70] * 30, [200 + 90 * i for i in range(30)], 8, 4, 128, 128)])
def test_more_items_than_sms(new, totals, heads, kv_heads, d, page, causal):
    """Whole rounds of items and items cut between SMs, with group sizes that do not divide a tile."""
    _check_attention(new, totals, heads, kv_heads, d, page, BF16, causal=causal)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (64, 3), (100, 64), (100, 130), (333, 5), (5000, 10)])
@pytest.mark.parametrize("new,totals,heads,kv_heads,d,page", [
    ([1, 1], [700, 90], 8, 2, 128, 16), ([9], [400], 4, 4, 64, 24), ([150, 33], [900, 33], 4, 2, 128, 32), ([260], [3200], 2, 2, 128, 1560)])
def test_windows_and_sinks(new, totals, heads, kv_heads, d, page, window, sinks, causal):
    _check_attention(new, totals, heads, kv_heads, d, page, BF16, causal=causal, window=window, sinks=sinks)


@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf, torch.finfo(BF16).min])
@pytest.mark.parametrize("new,totals,page", [([1, 1], [70, 5], 16), ([1], [33], 64), ([20], [41], 24), ([200, 3], [333, 3], 64), ([200], [1700], 1560)])
def test_what_no_session_holds_may_hold_anything(new, totals, page, fill):
    """Positions past a session's end (recycled or never written pages) are not read into the result."""
    for causal in (False, True):
        out = _check_attention(new, totals, 4, 2, 128, page, BF16, causal=causal, fill=fill)
        assert bool(torch.isfinite(out.float()).all())


@pytest.mark.parametrize("new,totals", [([5], [2]), ([200, 1], [60, 0]), ([3, 4], [0, 4]), ([1, 1], [0, 0])])
def test_rows_that_see_nothing(new, totals):
    """More new tokens than the session holds, or none held: zeros, and minus infinity for the log-sum-exp."""
    from reelcache_b200.ops import paged
    g = _gen(11)
    heads, kv_heads, d, page = 4, 2, 64, 16
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, page, BF16, fill=math.nan)
    q = torch.randn(sum(new), heads, d, generator=g, device="cuda").bfloat16()
    out, lse = paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=max(new), causal=True, return_lse=True,
                               out=torch.full_like(q, 7.0))
    want, want_lse, bound, lse_bound = attend(q, k_pages, v_pages, table, kv_lens, new, causal=True)
    assert within(out, want, bound) and within(lse, want_lse, lse_bound)
    empty = torch.isinf(want_lse)
    assert bool(empty.any()) and bool((out[empty] == 0).all())


def test_peaked_and_growing_scores():
    """Scores of some hundreds, growing along the keys: the running maximum moves in every tile."""
    from reelcache_b200.ops import paged
    for new in (1, 5, 300):
        g = _gen(12)
        k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [new], [1500], 2, 128, 32, BF16)
        ramp = torch.empty(1500, device="cuda")
        for s in range(1500):
            ramp[s] = s / 250
        for b in range(47):
            n = min(32, 1500 - b * 32)
            k_pages[int(table[0, b]), :n] = ramp[b * 32:b * 32 + n, None, None].bfloat16()
        q = torch.ones(new, 4, 128, device="cuda").bfloat16()
        out, lse = paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=new, causal=True, return_lse=True, scale=0.5)
        want, want_lse, bound, lse_bound = attend(q, k_pages, v_pages, table, kv_lens, [new], causal=True, scale=0.5)
        assert within(out, want, bound) and within(lse, want_lse, lse_bound)


@pytest.mark.parametrize("new", [1, 6, 150])
def test_page_layouts_and_strided_queries(new):
    """Heads outside of tokens in memory, one layer of a pool of several, queries out of a fused projection."""
    from reelcache_b200.ops import paged
    _check_attention([new, 2], [new + 300, 80], 8, 2, 128, 16, BF16, causal=True, layout="hnd")
    g = _gen(13)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [new], [new + 77], 2, 64, 32, BF16)
    pool = torch.stack([k_pages, v_pages, v_pages, k_pages]).view(2, 2, *k_pages.shape)
    fused = torch.randn(new, 10, 64, generator=g, device="cuda").bfloat16()
    q = fused[:, 1:9]
    got = paged.attention(q, pool[1, 1], pool[1, 0], table, kv_lens, cu_q, max_q_len=new)
    want = paged.attention(q.contiguous(), k_pages, v_pages, table, kv_lens, cu_q, max_q_len=new)
    assert torch.equal(got, want)
    by_layer = pool.permute(2, 0, 1, 3, 4, 5).contiguous().permute(1, 2, 0, 3, 4, 5)  # a page holds all layers
    assert torch.equal(paged.attention(q, by_layer[1, 1], by_layer[1, 0], table, kv_lens, cu_q, max_q_len=new), want)


@pytest.mark.parametrize("new", [1, 6, 150, 700])
def test_outputs_given_with_strides(new):
    """Outputs inside a larger buffer, on 16 but not on 32 bytes."""
    from reelcache_b200.ops import paged
    g = _gen(21)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [new], [new + 900], 2, 64, 32, BF16)
    q = torch.randn(new, 4, 64, generator=g, device="cuda").bfloat16()
    want = paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=new)
    buffer = torch.zeros(new, 5, 72, dtype=BF16, device="cuda")
    paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=new, out=buffer[:, :4, 8:])
    assert torch.equal(buffer[:, :4, 8:], want)
    assert not bool(buffer[:, 4].any()) and not bool(buffer[:, :, :8].any())


@pytest.mark.parametrize("new", [1, 200])
def test_pages_beyond_32_bit_offsets(new):
    """A pool of more than 2^32 elements: its last pages are read where they are."""
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    pages, page = (1 << 32) // (64 * 128) + 40, 64
    pool = torch.empty(pages, page, 1, 128, dtype=BF16, device="cuda")
    g = _gen(14)
    small_k, small_v, table, kv_lens, cu_q = paged_batch(g, [new], [600], 1, 128, page, BF16)
    held = table[0, :10].long()
    far = pages - 1 - 2 * torch.arange(10, device="cuda")
    pool[far] = small_k[held]
    v_far = far - 1
    pool[v_far] = small_v[held]
    v_pool = torch.as_strided(pool, pool.shape, pool.stride())
    q = torch.randn(new, 2, 128, generator=g, device="cuda").bfloat16()
    # one table serves keys and values: shift the value pool by one page
    got = paged.attention(q, pool[1:], v_pool[:-1], (far - 1).to(torch.int32)[None].contiguous(), kv_lens, cu_q, max_q_len=new)
    want = paged.attention(q, small_k, small_v, table, kv_lens, cu_q, max_q_len=new)
    assert torch.equal(got, want)
    k_new = torch.randn(new, 1, 128, generator=g, device="cuda").bfloat16()
    positions = _positions(g, new, 3)
    v_small = small_v.clone()
    paged.append(q, k_new, k_new, positions, AxisRope.wan(128), pool[1:], v_pool[:-1], (far - 1).to(torch.int32)[None].contiguous(), kv_lens, cu_q)
    paged.append(q, k_new, k_new, positions, AxisRope.wan(128), small_k, v_small, table, kv_lens, cu_q)
    assert torch.equal(pool[far], small_k[held]) and torch.equal(pool[v_far], v_small[held])


@pytest.mark.parametrize("new", [1, 30, 300])
def test_repeated_calls_agree_bit_for_bit_and_streams(new):
    from reelcache_b200.ops import paged
    g = _gen(15)
    totals = [new + 2000, new, new + 700]
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [new] * 3, totals, 4, 128, 32, BF16)
    q = torch.randn(3 * new, 8, 128, generator=g, device="cuda").bfloat16()
    call = lambda: paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=new, causal=True)  # noqa: E731
    first = call()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got += [call(), call()]
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in got)


@pytest.mark.parametrize("new", [1, 300])
def test_attention_in_a_graph(new):
    """Captured once, replayed with other lengths and pages."""
    from reelcache_b200.ops import paged
    g = _gen(16)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [new, new], [new + 500, new + 9], 2, 128, 16, BF16, width_extra=3)
    q = torch.randn(2 * new, 4, 128, generator=g, device="cuda").bfloat16()
    call = lambda: paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=new, causal=True)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    kv_lens[0] -= 123
    table[0, :2] = table[0, :2].flip(0)
    q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call())


def test_attention_page_out_of_range_is_reported(cuda_device):
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext, paged
    g = _gen(17)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [1, 150], [100, 200], 2, 64, 16, BF16)
    q = torch.randn(151, 2, 64, generator=g, device="cuda").bfloat16()
    for bad in (-1, k_pages.shape[0], 1 << 30, -(1 << 30)):
        for s, block in ((0, 3), (1, 0)):
            broken = table.clone()
            broken[s, block] = bad
            for most, ids in ((1, slice(0, 1)), (150, slice(0, 2))):
                if s == 1 and most == 1:
                    continue
                out = paged.attention(q[:1 if most == 1 else 151], k_pages, v_pages, broken[ids], kv_lens[ids],
                                      cu_q[:2 if most == 1 else 3], max_q_len=most)
                assert bool(torch.isfinite(out.float()).all())
                with pytest.raises(DeviceStatusError, match="page number"):
                    _ext.check_status(cuda_device)
    for most in (1, 150):  # a length that the table's row cannot name
        out = paged.attention(q[:most], k_pages, v_pages, table[:1], kv_lens[:1] + 10 ** 6, torch.tensor([0, most], dtype=torch.int32, device="cuda"),
                              max_q_len=most)
        with pytest.raises(DeviceStatusError, match="block table"):
            _ext.check_status(cuda_device)


def test_attention_refusals():
    from reelcache_b200.errors import ConfigurationError, UnsupportedError
    from reelcache_b200.ops import paged
    g = _gen(18)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [1], [100], 2, 64, 16, BF16)
    q = torch.randn(1, 4, 64, generator=g, device="cuda").bfloat16()
    call = lambda q=q, k=k_pages, v=v_pages, t=table, n=kv_lens, c=cu_q, **kw: paged.attention(  # noqa: E731
        q, k, v, t, n, c, **{"max_q_len": 1, **kw})
    call()
    with pytest.raises(UnsupportedError):
        call(q=q.cpu())
    with pytest.raises(ConfigurationError):
        call(window=0)
    nine = torch.randn(5, 9, 2, 64, device="cuda").bfloat16()
    for wrong in (dict(q=q.half()), dict(q=q.float()), dict(q=q[:, :3]), dict(k=k_pages[:, :, :1]), dict(k=nine, v=nine),
                  dict(v=v_pages[1:]), dict(t=table.long()), dict(n=kv_lens[:0]), dict(c=cu_q[:1]), dict(t=table.cpu()),
                  dict(max_q_len=0), dict(sinks=-1, window=5), dict(scale=0.0), dict(scale=-1.0), dict(q=q.clone().requires_grad_()), dict(q=torch.randn(1, 4, 96, device="cuda").bfloat16()),
                  dict(out=torch.empty(2, 4, 64, device="cuda", dtype=BF16)), dict(k=k_pages[..., ::2])):
        with pytest.raises(RuntimeError):
            call(**wrong)


# -- the page table ---------------------------------------------------------------------------------------------------

def _ints(*values):
    return [torch.tensor(v, dtype=torch.int32, device="cuda") for v in values]


def _table(pages, seqs, width, page, planes=3, row=8, seed=0):
    from reelcache_b200.ops.paged import PageTable
    storage = torch.randn(planes, pages, page, row, generator=_gen(seed), device="cuda").bfloat16()
    return PageTable.empty(pages, seqs, width, page, "cuda"), ListTable(pages, seqs, width, page, storage.cpu()), storage


@pytest.mark.parametrize("seed", range(6))
def test_page_table_follows_its_rules(seed):
    """Random calls against the same rules in Python lists."""
    import random
    rng = random.Random(seed)
    page = rng.choice([8, 16, 24])
    seqs, width = rng.choice([(5, 4), (40, 9), (300, 6)])
    pages = seqs * width // 2 + 3
    table, model, storage = _table(pages, seqs, width, page, planes=rng.choice([1, 3]), row=rng.choice([8, 40]), seed=seed)
    for _ in range(30):
        kind = rng.choice(["allocate", "fork", "fork", "release", "compact"])
        if kind == "allocate":
            some = rng.sample(range(seqs), rng.randint(1, seqs))
            lens = [rng.randint(model.lens[s], min(width * page, model.lens[s] + 2 * page)) for s in some]
            if not model.allocate(some, lens):
                continue
            table.allocate(*_ints(some, lens))
        elif kind == "fork":
            empty = [s for s in range(seqs) if model.lens[s] == 0]
            held = [s for s in range(seqs) if model.lens[s]]
            if not empty or not held:
                continue
            children = rng.sample(empty, rng.randint(1, len(empty)))
            parents = [rng.choice(held) for _ in children]
            lens = [rng.randint(0, model.lens[p]) for p in parents]
            if not model.fork(parents, children, lens):
                continue
            table.fork(*_ints(parents, children, lens), storage)
        elif kind == "release":
            some = rng.sample(range(seqs), rng.randint(1, seqs // 2))
            model.release(some)
            table.release(_ints(some)[0])
        else:
            assert int(table.compact(storage)) == model.compact()
        model.check(table, storage)


def test_page_table_large_pool_and_pages():
    """Scans over several blocks of the pool; pages of more than one copy item."""
    table, model, storage = _table(9000, 700, 20, 64, planes=2, row=8, seed=1)
    lens = [(37 * i) % 1280 for i in range(600)]
    assert model.allocate(list(range(600)), lens)
    table.allocate(*_ints(list(range(600)), lens))
    gone = list(range(0, 600, 3))
    model.release(gone)
    table.release(_ints(gone)[0])
    children = list(range(600, 700))
    parents = [1 + 3 * (i % 190) for i in range(100)]
    at = [max(0, lens[p] - i) for i, p in enumerate(parents)]
    assert model.fork(parents, children, at)
    table.fork(*_ints(parents, children, at), storage)
    model.check(table, storage)
    assert int(table.compact(storage)) == model.compact()
    model.check(table, storage)
    table, model, storage = _table(9, 4, 3, 72, planes=2, row=1000, seed=2)  # 144 KB pages
    for op, values in (("allocate", ([3, 0], [150, 100])), ("release", ([3],)), ("fork", ([0], [1], [99])), ("fork", ([0], [2], [72]))):
        assert getattr(model, op)(*values) is not False
        getattr(table, op)(*_ints(*values), *([storage] if op == "fork" else []))
        model.check(table, storage)
    assert int(table.compact(storage)) == model.compact()
    model.check(table, storage)


def test_page_table_refusals_change_nothing(cuda_device):
    from reelcache_b200.errors import ConfigurationError, DeviceStatusError
    from reelcache_b200.ops import _ext
    from reelcache_b200.ops.paged import PageTable
    table, model, storage = _table(10, 6, 8, 8)
    assert model.allocate([0, 1], [20, 33])
    table.allocate(*_ints([0, 1], [20, 33]))
    refused = [("allocate", ([2], [30]), "too few"), ("allocate", ([0, 0], [21, 22]), "invalid"), ("allocate", ([6], [1]), "invalid"),
               ("allocate", ([-1], [1]), "invalid"), ("allocate", ([1], [32]), "invalid"), ("allocate", ([2], [65]), "invalid"),
               ("allocate", ([2, 3], [2 ** 31 - 1, 2 ** 31 - 1]), "invalid"),
               ("fork", ([0], [1], [3]), "invalid"), ("fork", ([0], [2], [21]), "invalid"), ("fork", ([0, 0], [2, 2], [1, 1]), "invalid"),
               ("fork", ([7], [2], [1]), "invalid"), ("fork", ([0], [9], [1]), "invalid"), ("fork", ([0], [2], [-1]), "invalid"),
               ("fork", ([0, 0, 0, 1], [2, 3, 4, 5], [1, 2, 3, 4]), "too few")]
    for op, values, text in refused:
        getattr(table, op)(*_ints(*values), *([storage] if op == "fork" else []))
        with pytest.raises(DeviceStatusError, match=text):
            _ext.check_status(cuda_device)
        model.check(table, storage)
    table.release(_ints([1, 1, 1])[0])  # named thrice, given back once
    model.release([1])
    model.check(table, storage)
    table.release(_ints([8])[0])
    with pytest.raises(DeviceStatusError):
        _ext.check_status(cuda_device)
    model.check(table, storage)
    for call in (lambda: table.allocate(*_ints([0], [30, 31])), lambda: table.release(torch.tensor([0], device="cuda")),
                 lambda: table.release(torch.tensor([0], dtype=torch.int32)), lambda: table.compact(storage[:, :9]),
                 lambda: table.fork(*_ints([0], [1], [3]), storage.transpose(2, 3)), lambda: table.compact(storage[:1].expand(3, -1, -1, -1))):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ConfigurationError):
        PageTable(torch.zeros(10, dtype=torch.int32, device="cuda"), pages=4, seqs=4, page_size=8)
    model.check(table, storage)


def test_copy_pages(cuda_device):
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext, paged
    g = _gen(19)
    storage = torch.randn(3, 20, 16, 4, 24, generator=g, device="cuda").half()
    want = storage.clone()
    source, target, rows = [3, 5, 0, 19, -1], [4, 1, 10, 2, -1], [16, 1, 0, 9, 5]
    for s, t, r in zip(source, target, rows):
        if s >= 0:
            want[:, t, :r] = storage[:, s, :r]
    paged.copy_pages(storage, *_ints(source, target, rows))
    assert torch.equal(storage, want)
    by_page = storage.transpose(0, 1).contiguous().transpose(0, 1)  # a page holds all planes
    paged.copy_pages(by_page, *_ints([7], [8]))
    want[:, 8] = want[:, 7]
    assert torch.equal(by_page, want)
    for s, t in ((20, 1), (1, 20), (-2, 1), (1, -1)):
        paged.copy_pages(by_page, *_ints([s], [t]))
        with pytest.raises(DeviceStatusError):
            _ext.check_status(cuda_device)
    paged.copy_pages(by_page, *_ints([1], [2], [17]))
    with pytest.raises(DeviceStatusError):
        _ext.check_status(cuda_device)
    assert torch.equal(by_page, want)
