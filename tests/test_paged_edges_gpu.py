"""Where the paged operators could go wrong: calls without a pause between them, values and lengths at the edges, batches
that are out of date, and the long forms of attention."""

import math

import pytest
import torch

from .paged_support import attend, paged_batch, rotate_bound, within

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(*values):
    return [torch.tensor(v, dtype=torch.int32, device="cuda") for v in values]


# -- calls without a pause between them -------------------------------------------------------------------------------

@pytest.mark.parametrize("new,steps", [(1, 60), (5, 40), (24, 24), (150, 8)])
def test_calls_back_to_back_see_what_was_written_before(new, steps):
    """Grids overlap the end of the grids before them: each must still see all that those wrote (the table that allocate,
    fork and compact change, the queries that append rotates in place). The same calls with a pause after each are the
    measure, bit for bit."""
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    seqs, page, heads, kv_heads, d = 6, 16, 8, 2, 64
    g = _gen(new)
    rope = AxisRope.wan(d)
    width = -(-(new * steps) // page) + 1
    pages = seqs * width + 8
    fused = torch.randn(steps, 4 * new, heads + 2 * kv_heads, d, generator=g, device="cuda").bfloat16()
    positions = torch.randint(0, 900, (steps, 4 * new, 3), generator=g, device="cuda", dtype=torch.int32)
    start = torch.randn(2, pages, page, kv_heads, d, generator=g, device="cuda").bfloat16()
    (cu_q,) = _ints([new * i for i in range(5)] + [4 * new] * 2)  # sequences 4 and 5 have no new tokens
    plans = []
    lens = [0] * seqs
    for step in range(steps):
        for s in range(4):
            lens[s] += new
        plan = [("allocate", _ints([3, 0, 2, 1], [lens[3], lens[0], lens[2], lens[1]]))]
        if step % 3 == 1:  # sequence 1 goes on as a fork of 0; what it held is freed
            plan += [("release", _ints([1, 4])), ("fork", _ints([0], [4], [lens[0]])), ("release", _ints([1])),
                     ("fork", _ints([4], [1], [lens[0]])), ("release", _ints([4]))]
            lens[1] = lens[0]
        if step % 5 == 4:
            plan.append(("compact", []))
        plans.append(plan)

    def run(pause):
        storage, q_rows = start.clone(), fused.clone()
        table = paged.PageTable.empty(pages, seqs, width, page, "cuda")
        outs = []
        torch.cuda.synchronize()
        if not pause:
            torch.cuda._sleep(40_000_000)  # the calls queue up behind this
        for step in range(steps):
            for op, args in plans[step][:1]:
                table.allocate(*args)
                pause and torch.cuda.synchronize()
            q, k, v = q_rows[step].split([heads, kv_heads, kv_heads], dim=1)
            paged.append(q, k, v, positions[step], rope, storage[0], storage[1], table.block_table, table.lens, cu_q, out=q)
            pause and torch.cuda.synchronize()
            outs.append(paged.attention(q, storage[0], storage[1], table.block_table, table.lens, cu_q, max_q_len=new, causal=True))
            pause and torch.cuda.synchronize()
            for op, args in plans[step][1:]:
                getattr(table, op)(*args, *([storage] if op in ("fork", "compact") else []))
                pause and torch.cuda.synchronize()
        torch.cuda.synchronize()
        return torch.stack(outs), storage, table.state

    for got, want in zip(run(False), run(True)):
        assert torch.equal(got, want)


# -- values at the edges ----------------------------------------------------------------------------------------------

def _same(got, want, bound):
    """Within the bound, or NaN on both sides."""
    return within(torch.where(want.isnan(), 0.0, got.double()), want.nan_to_num(0.0, posinf=math.inf, neginf=-math.inf),
                  bound.nan_to_num(0.0)) and torch.equal(got.isnan(), want.isnan())


# few rows clustered and as a line; the twin form; direct with one and with several CTAs; planned
EDGE_SHAPES = [([1], [700], 4, 2), ([1] * 90, [40 + 7 * i for i in range(90)], 8, 4), ([30], [400], 4, 4), ([150], [300], 4, 2),
               ([300], [3000], 2, 2), ([1100], [1500], 32, 32)]


@pytest.mark.parametrize("kind", ["nan", "inf", "-inf", "nan query"])
@pytest.mark.parametrize("new,totals,heads,kv_heads", EDGE_SHAPES)
def test_nan_and_infinite_scores(new, totals, heads, kv_heads, kind):
    """A NaN score makes its rows' outputs and log-sum-exps NaN; a score of plus infinity makes the log-sum-exp that, and
    the output NaN; one of minus infinity weighs nothing. Rows that do not see the key keep their results."""
    from reelcache_b200.ops import paged
    d, page = 64, 16
    g = _gen(31)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, page, BF16)
    q = torch.randn(sum(new), heads, d, generator=g, device="cuda").bfloat16()
    q[..., 0] = 1.0
    if kind == "nan query":
        q[sum(new) // 2, 1, 5] = math.nan
    else:
        for s, total in enumerate(totals):  # one key that the last new tokens see and the first do not, and one that all see
            for at in (total - 1 - new[s] // 3, total // 5):
                k_pages[int(table[s, at // page]), at % page, 0] = 0.0
                k_pages[int(table[s, at // page]), at % page, 0, 0] = float(kind)
    for causal, window in ((True, None), (True, 17), (False, None)):
        out, lse = paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=max(new), causal=causal, window=window, return_lse=True)
        want, want_lse, bound, lse_bound = attend(q, k_pages, v_pages, table, kv_lens, new, causal=causal, window=window)
        if kind == "-inf":  # (the bounds take magnitudes of scores: without the infinite ones)
            finite = k_pages.clone()
            finite[finite == -math.inf] = 0.0
            bound, lse_bound = attend(q, finite, v_pages, table, kv_lens, new, causal=causal, window=window)[2:]
        assert _same(lse, want_lse, lse_bound)
        assert _same(out, want, bound)
        assert kind == "-inf" or not bool(torch.isfinite(want_lse).all())


def test_rows_whose_only_score_is_nan_or_minus_infinity():
    """The first new token of a sequence without history sees one key, alone in its tile."""
    from reelcache_b200.ops import paged
    for new, heads in ((1, 2), (9, 2), (100, 2), (400, 2)):
        for value in (math.nan, -math.inf, math.inf):
            g = _gen(32)
            k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [new], [new], 1, 64, 16, BF16)
            q = torch.randn(new, heads, 64, generator=g, device="cuda").bfloat16()
            q[..., 0] = 1.0
            k_pages[int(table[0, 0]), 0] = 0.0
            k_pages[int(table[0, 0]), 0, 0, 0] = value
            out, lse = paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=new, causal=True, return_lse=True)
            if value == -math.inf:
                assert not bool(out[0].any()) and bool((lse[0] == -math.inf).all())
                assert bool(torch.isfinite(out.float()).all())
            else:
                assert bool(out.isnan().all())
                assert bool(lse.isnan().all() if math.isnan(value) else (lse == math.inf).all())


@pytest.mark.parametrize("new,totals", [([5], [2]), ([200, 1], [60, 0]), ([200, 30], [190, 30]), ([400], [390])])
def test_a_window_of_any_size(new, totals):
    """Positions before the first (more new tokens than the session holds) and a window up to the largest integer."""
    from reelcache_b200.ops import paged
    g = _gen(33)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, new, totals, 2, 64, 16, BF16, fill=math.nan)
    q = torch.randn(sum(new), 4, 64, generator=g, device="cuda").bfloat16()
    call = lambda **kw: paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=max(new), causal=True,  # noqa: E731
                                        return_lse=True, **kw)
    want = call()
    for window in (2 ** 31 - 1, 2 ** 31 - 100, 2 ** 30):
        for got, x in zip(call(window=window), want):
            assert torch.equal(got, x)


# -- derivatives that the operators do not have -----------------------------------------------------------------------

def test_forward_mode_tangents_are_refused():
    """A tangent would be lost without a word: the calls raise, as they do for gradients that they do not have."""
    from torch.autograd import forward_ad
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope, rotate
    g = _gen(41)
    rope = AxisRope.wan(64)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [3], [20], 2, 64, 16, BF16)
    (positions,) = _ints([[1, 2, 3]] * 3)
    q, k = (torch.randn(3, n, 64, generator=g, device="cuda").bfloat16() for n in (4, 2))
    append = lambda q, k, v, kp, vp: paged.append(q, k, v, positions, rope, kp, vp, table, kv_lens, cu_q)  # noqa: E731
    attention = lambda q, kp, vp: paged.attention(q, kp, vp, table, kv_lens, cu_q, max_q_len=3)  # noqa: E731
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for call, args in ((lambda a, b: rotate(a, b, positions, rope), (q, k)), (append, (q, k, k, k_pages, v_pages)),
                           (attention, (q, k_pages, v_pages))):
            for i in range(len(args)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*[dual(x) if j == i else x for j, x in enumerate(args)])
            call(*args)
    before = k_pages.clone()
    attention(q, k_pages, v_pages)
    assert torch.equal(before, k_pages)


def test_gradients_with_respect_to_positions_are_refused():
    from reelcache_b200.ops.rope import AxisRope, rotate
    q = torch.randn(3, 4, 64, device="cuda", requires_grad=True)
    positions = torch.rand(3, 3, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="positions"):
        rotate(q, None, positions, AxisRope.wan(64))
    with torch.no_grad():
        rotate(q, None, positions, AxisRope.wan(64))
    out, _ = rotate(q, None, positions.detach(), AxisRope.wan(64))
    out.sum().backward()
    assert q.grad is not None


# -- positions beyond what a float can count --------------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_rotate_positions_of_any_size(dtype, layout):
    """int32 positions up to the largest, and float32 ones beyond 2^24: the angles in 80-bit floats are off by less than
    2^31 * 2^-63 of a radian."""
    import numpy as np
    from reelcache_b200.ops.rope import AxisRope, rotate
    sections = (22, 21, 21)
    rope = AxisRope(128, sections, layout=layout)
    q = torch.randn(64, 2, 128, generator=_gen(51), device="cuda").to(dtype)
    rng = np.random.default_rng(51)
    some = rng.integers(-2 ** 31, 2 ** 31, (64, 3))
    some[0], some[1], some[2] = 2 ** 31 - 1, -2 ** 31, (2 ** 24, 2 ** 24 + 1, 2 ** 24 - 1)
    some[3:20] = rng.integers(2 ** 24, 2 ** 25, (17, 3)) | 1
    assert np.finfo(np.longdouble).nmant >= 63
    for kind in (torch.int32, FP32):
        positions = torch.tensor(some).to(kind).cuda()
        at = positions.cpu().numpy().astype(np.longdouble)
        angle = np.concatenate([at[:, a:a + 1] * np.longdouble(10000) ** (-np.arange(n, dtype=np.longdouble) / n)
                                for a, n in enumerate(sections)], axis=1)
        cos, sin = (torch.tensor(f(angle).astype(np.float64), device="cuda")[:, None] for f in (np.cos, np.sin))
        x = q.double()
        a, b = (x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else x.chunk(2, dim=-1)
        u, v, size = a * cos - b * sin, a * sin + b * cos, a.abs() + b.abs()
        pairs = [(u, v), (size, size)]
        want, size = (torch.stack(p, dim=-1).flatten(-2) if layout == "interleaved" else torch.cat(p, dim=-1) for p in pairs)
        got, _ = rotate(q, None, positions, rope)
        assert within(got, want, rotate_bound(want, size, dtype)), float(((got.double() - want).abs()).max())


# -- tokens that the lengths do not cover -----------------------------------------------------------------------------

@pytest.mark.parametrize("new,bound", [([1, 5], 2), ([1, 20], 4), ([300, 1], 200), ([200] * 40, 150), ([700, 9], 100)])
def test_more_new_tokens_than_the_bound_are_reported(cuda_device, new, bound):
    """max_q_len below a sequence's new tokens leaves rows without a result: the status says so."""
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext, paged
    g = _gen(61)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, new, [n + 50 for n in new], 2, 64, 16, BF16)
    q = torch.randn(sum(new), 4, 64, generator=g, device="cuda").bfloat16()
    call = lambda q=q, **kw: paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, **{"max_q_len": max(new), **kw})  # noqa: E731
    want, _, error, _ = attend(q, k_pages, v_pages, table, kv_lens, new)
    for most in (max(new), 10 ** 6):  # (a looser bound may take another form, and round elsewhere)
        assert within(call(max_q_len=most), want, error)
        _ext.check_status(cuda_device)
    call(max_q_len=bound)
    with pytest.raises(DeviceStatusError, match="max_q_len"):
        _ext.check_status(cuda_device)
    call(q=q[:-1])  # fewer rows than cu_q names
    with pytest.raises(DeviceStatusError, match="max_q_len"):
        _ext.check_status(cuda_device)


def test_append_without_sequences_still_rotates():
    """Tokens of no sequence are rotated, like those past the last sequence, and written nowhere."""
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope, rotate
    g = _gen(62)
    rope = AxisRope.wan(64)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [2], [10], 2, 64, 8, BF16)
    before = k_pages.clone(), v_pages.clone()
    q, k = (torch.randn(3, n, 64, generator=g, device="cuda").bfloat16() for n in (4, 2))
    positions = torch.randint(0, 900, (3, 3), generator=g, device="cuda", dtype=torch.int32)
    out = paged.append(q, k, k, positions, rope, k_pages, v_pages, table[:0], kv_lens[:0], cu_q[:1], out=torch.full_like(q, 7.0))
    assert torch.equal(out, rotate(q, None, positions, rope)[0])
    assert torch.equal(k_pages, before[0]) and torch.equal(v_pages, before[1])


# -- what is reported, and what callers can see --------------------------------------------------------------------------

def test_both_status_words_are_reported(cuda_device):
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext
    word = _ext.status_word(cuda_device)
    word[0], word[1] = 0x103, 0x402
    with pytest.raises(DeviceStatusError, match="0x103.*0x402"):
        _ext.check_status(cuda_device)
    _ext.check_status(cuda_device)


def test_written_tensors_carry_a_new_version():
    """What autograd has kept of a tensor must be seen to have changed."""
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = _gen(71)
    rope = AxisRope.wan(64)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [3], [20], 2, 64, 16, BF16)
    (positions,) = _ints([[1, 2, 3]] * 3)
    q, k = (torch.randn(3, n, 64, generator=g, device="cuda").bfloat16() for n in (4, 2))
    weight = torch.ones(64, device="cuda", dtype=BF16, requires_grad=True)
    loss = (k_pages * weight).sum()
    out = torch.empty_like(q)
    versions = [t._version for t in (k_pages, v_pages, out)]
    paged.append(q, k, k, positions, rope, k_pages, v_pages, table, kv_lens, cu_q, out=out)
    assert all(t._version > n for t, n in zip((k_pages, v_pages, out), versions))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    version = out._version
    paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=3, out=out)
    assert out._version > version
    storage = torch.randn(2, 6, 16, 8, device="cuda")
    held = paged.PageTable.empty(6, 3, 2, 16, "cuda")
    for call in (lambda: paged.copy_pages(storage, *_ints([1], [2])), lambda: held.allocate(*_ints([0], [20])),
                 lambda: held.fork(*_ints([0], [1], [20]), storage), lambda: held.release(*_ints([0])), lambda: held.compact(storage)):
        before = storage._version, held.state._version
        call()
        assert (storage._version, held.state._version) != before
    with torch.inference_mode():
        kept = k_pages.clone(), v_pages.clone()
        paged.append(q, k, k, positions, rope, *kept, table, kv_lens, cu_q)


def test_pages_that_want_a_gradient_are_refused():
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = _gen(72)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [3], [20], 2, 64, 16, BF16)
    (positions,) = _ints([[1, 2, 3]] * 3)
    q, k = (torch.randn(3, n, 64, generator=g, device="cuda").bfloat16() for n in (4, 2))
    call = lambda kp=k_pages, vp=v_pages, **kw: paged.append(q, k, k, positions, AxisRope.wan(64), kp, vp, table, kv_lens, cu_q, **kw)  # noqa: E731
    for wrong in (dict(kp=k_pages.clone().requires_grad_()), dict(vp=v_pages.clone().requires_grad_()),
                  dict(out=torch.empty_like(q).requires_grad_())):
        with pytest.raises(RuntimeError, match="gradient"):
            call(**wrong)
        with torch.no_grad():
            call(**wrong)
    with pytest.raises(RuntimeError, match="gradient"):
        paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=3, out=torch.empty_like(q).requires_grad_())
    storage = torch.randn(2, 6, 16, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="gradient"):
        paged.copy_pages(storage, *_ints([1], [2]))


def test_outputs_that_overlap_themselves_are_refused():
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = _gen(73)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [3], [20], 2, 64, 16, BF16)
    (positions,) = _ints([[1, 2, 3]] * 3)
    q, k = (torch.randn(3, n, 64, generator=g, device="cuda").bfloat16() for n in (4, 2))
    append = lambda kp=k_pages, vp=v_pages, **kw: paged.append(q, k, k, positions, AxisRope.wan(64), kp, vp, table, kv_lens, cu_q, **kw)  # noqa: E731
    thin = torch.empty(1, 4, 64, device="cuda", dtype=BF16).expand(3, 4, 64)
    for call in (lambda: append(kp=k_pages[:1].expand_as(k_pages)), lambda: append(vp=v_pages[:, :, :1].expand_as(v_pages)),
                 lambda: append(out=thin), lambda: append(vp=k_pages),
                 lambda: paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=3, out=thin)):
        with pytest.raises(RuntimeError):
            call()
    # (pages that are only read may be expanded)
    paged.attention(q, k_pages[:, :, :1].expand_as(k_pages), v_pages, table, kv_lens, cu_q, max_q_len=3)
    both = torch.randn(5, 4, 64, generator=g, device="cuda").bfloat16()
    with pytest.raises(RuntimeError):  # rows that are still to be read
        paged.append(both[:3], k, k, positions, AxisRope.wan(64), k_pages, v_pages, table, kv_lens, cu_q, out=both[1:4])
    want = paged.attention(both[:3], k_pages, v_pages, table, kv_lens, cu_q, max_q_len=3)
    assert torch.equal(paged.attention(both[:3], k_pages, v_pages, table, kv_lens, cu_q, max_q_len=3, out=both[:3]), want)


# -- which form a call takes ------------------------------------------------------------------------------------------

def _form(new, totals, heads, kv_heads, d, page, **mask):
    """The form that the checks of these sizes take (:func:`paged_batch` with two columns more)."""
    from reelcache_b200.ops import paged
    width = max(max(-(-t // page) for t in totals), 1) + 2
    return paged.attention_form(sum(new), heads, kv_heads, d, len(new), width, page, max_q_len=max(max(new), 1), **mask)


def test_a_long_sequence_among_short_ones_is_planned():
    """The direct grid has a block for every row tile that the longest sequence has, in every sequence: 2,000 here, of which
    1,859 would each take an SM to find that they have nothing to do."""
    assert _form([4000] + [1] * 15, [4096] * 16, 8, 1, 128, 64, causal=True) == "planned"
    assert _form([250] * 16, [4096] * 16, 8, 1, 128, 64, causal=True) == "direct 1"  # the same rows, evenly


def test_grids_beyond_31_bits_are_not_launched_directly():
    """One sequence of a million tokens among 10,000: 4 * 10^9 blocks would wrap, and leave rows without a result."""
    assert _form([1_000_000] + [1] * 9_999, [8] * 10_000, 8, 8, 128, 8) == "planned"


# -- the planned form of chunks ---------------------------------------------------------------------------------------

# items cut into single tiles; odd groups and pages; more items than SMs (whole rounds, then cut ones)
PLANNED = [([300, 0, 45, 1], [1100, 30, 200, 700], 6, 2, 64, 16, BF16), ([700, 129], [700, 2300], 5, 1, 128, 24, FP16),
           ([900, 0, 333, 1], [1300, 50, 1333, 800], 40, 40, 64, 200, BF16)]


def _planned(g, new, totals, heads, kv_heads, d, page, dtype, *, causal=False, window=None, sinks=0, **kw):
    """A batch with a table wide enough for 60,000 tokens of each sequence (as one has that is kept for a graph), which takes
    the planned form whatever the lengths are, and its queries."""
    from reelcache_b200.ops import paged
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, page, dtype, width_extra=60_000 // page, **kw)
    assert paged.attention_form(sum(new), heads, kv_heads, d, len(new), table.shape[1], page, max_q_len=max(new), causal=causal,
                                window=window, sinks=sinks) == "planned"
    q = torch.randn(sum(new), heads, d, generator=g, device="cuda").to(dtype)
    return q, k_pages, v_pages, table, kv_lens, cu_q


def _check(batch, new, **mask):
    from reelcache_b200.ops import paged
    out, lse = paged.attention(*batch, max_q_len=max(new), return_lse=True, **mask)
    q, k_pages, v_pages, table, kv_lens, _ = batch
    want, want_lse, bound, lse_bound = attend(q, k_pages, v_pages, table, kv_lens, new, **mask)
    assert within(out, want, bound), float(((out.double() - want).abs() - bound).max())
    assert within(lse, want_lse, lse_bound)
    return out


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("fill", [None, math.nan, math.inf, torch.finfo(BF16).min])
@pytest.mark.parametrize("shape", PLANNED)
def test_planned_shapes_and_what_no_session_holds(shape, fill, causal):
    out = _check(_planned(_gen(81), *shape, causal=causal, fill=fill if shape[-1] == BF16 or fill is None else math.nan), shape[0], causal=causal)
    assert bool(torch.isfinite(out.float()).all())


@pytest.mark.parametrize("d,dtype", [(64, BF16), (128, FP16)])
@pytest.mark.parametrize("mask", [dict(window=1, causal=True), dict(window=333, sinks=5, causal=True), dict(window=333, sinks=5),
                                  dict(window=500, sinks=130), dict(window=100, sinks=400, causal=True),
                                  dict(window=700, sinks=130, causal=True)])
def test_planned_windows_and_sinks(mask, d, dtype):
    new, totals = [900, 0, 333, 1], [1300, 50, 1333, 800]
    _check(_planned(_gen(82), new, totals, 40, 40, d, 48, dtype, fill=math.nan, **mask), new, **mask)


def test_planned_long_window():
    new, mask = [1000], dict(window=5000, sinks=200, causal=True)
    _check(_planned(_gen(83), new, [12_000], 40, 40, 64, 64, BF16, **mask), new, **mask)


@pytest.mark.parametrize("new,totals", [([300, 20], [60, 0]), ([900, 40, 1], [890, 700, 0])])
def test_planned_rows_that_see_nothing(new, totals):
    batch = _planned(_gen(84), new, totals, 4, 2, 64, 16, BF16, causal=True, fill=math.nan)
    out = _check(batch, new, causal=True)
    assert not bool(out[:new[0] - totals[0]].any())


@pytest.mark.parametrize("shape", PLANNED[:2])
def test_planned_layouts_and_strides(shape):
    """Heads outside of tokens in memory, queries out of a fused projection, outputs on 16 but not on 32 bytes."""
    from reelcache_b200.ops import paged
    new, _, heads, _, d = shape[:5]
    q, *rest = _planned(_gen(85), *shape, causal=True, layout="hnd")
    _check((q, *rest), new, causal=True)
    fused = torch.randn(sum(new), heads + 3, d, generator=_gen(86), device="cuda").to(q.dtype)
    fused[:, 1:heads + 1] = q
    want = paged.attention(q, *rest, max_q_len=max(new), causal=True)
    assert torch.equal(paged.attention(fused[:, 1:heads + 1], *rest, max_q_len=max(new), causal=True), want)
    buffer = torch.zeros(sum(new), heads + 1, d + 8, dtype=q.dtype, device="cuda")
    paged.attention(q, *rest, max_q_len=max(new), causal=True, out=buffer[:, :heads, 8:])
    assert torch.equal(buffer[:, :heads, 8:], want)
    assert not bool(buffer[:, heads].any()) and not bool(buffer[:, :, :8].any())


@pytest.mark.parametrize("shape", PLANNED)
def test_planned_repeats_bits_on_several_streams_and_in_a_graph(shape):
    """Each call has a workspace of its own; a captured call follows lengths, pages and queries."""
    from reelcache_b200.ops import paged
    new = shape[0]
    q, k_pages, v_pages, table, kv_lens, cu_q = _planned(_gen(87), *shape, causal=True)
    call = lambda q=q: paged.attention(q, k_pages, v_pages, table, kv_lens, cu_q, max_q_len=max(new), causal=True)  # noqa: E731
    others = [q * x for x in (0.5, 2.0, -1.0)]
    want = [call(x) for x in others]
    streams = [torch.cuda.Stream() for _ in others]
    got = [[] for _ in others]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(4):  # calls of all streams at once
        for stream, x, outs in zip(streams, others, got):
            with torch.cuda.stream(stream):
                outs.append(call(x))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, outs in zip(want, got) for y in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    kv_lens[0] -= 57
    table[0, :2] = table[0, :2].flip(0)
    q.mul_(0.5)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call())


# -- items of many parts ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("mask", [dict(causal=True), dict(causal=True, window=60_000, sinks=70), dict()])
@pytest.mark.parametrize("new,kv_heads,total,form", [
    (1, 1, 131_072, "few rows, line"), (8, 1, 131_072, "few rows, line"), (1, 8, 65_536, "few rows, line"), (7, 2, 100_001, "few rows, line"),
    (16, 1, 65_536, "planned"), (40, 1, 131_072, "planned"), (128, 2, 65_537, "planned"), (40, 8, 131_072, "planned"), (300, 1, 70_000, "planned")])
def test_items_joined_out_of_many_parts(new, kv_heads, total, form, mask):
    """More parts than a join takes at a time (32): statistics are carried from one pass to the next. Scores grow along the
    keys and shrink again, so the maximum moves between the passes."""
    from reelcache_b200.ops import paged
    d, page, heads = 64, 64, 2 * kv_heads
    g = _gen(new + total)
    k_pages, v_pages, table, kv_lens, cu_q = paged_batch(g, [new], [total], kv_heads, d, page, BF16)
    if kv_heads in (1, 2):
        assert paged.attention_form(new, heads, kv_heads, d, 1, table.shape[1], page, max_q_len=new, **mask) == form
    hill = 3.0 - 12.0 * (torch.arange(table.shape[1] * page, device="cuda") / total - 0.7).abs()
    k_pages[table[0].long()] += hill.view(-1, page, 1, 1).bfloat16()
    q = (torch.randn(new, heads, d, generator=g, device="cuda") * 0.3 + 0.5).bfloat16()
    _check((q, k_pages, v_pages, table, kv_lens, cu_q), [new], **mask)
