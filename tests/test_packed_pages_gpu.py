"""Pages in 8 bits on sm_100a: rows quantised as they are written, read back, and attended, against 64-bit forms."""

import math

import pytest
import torch

from .paged_support import attend, paged_batch, rotate_bound, spun, within
from .sparse_support import held, pack_pages, quantise

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _bytes(pages):
    return pages.codes.view(torch.uint8).clone(), pages.scales.view(torch.uint8).clone()


def _noise_pages(g, pages, page, kv_heads, d, layout="nhd"):
    """Pages full of any bytes."""
    from reelcache_b200.ops.paged import PackedPages
    shape = (pages, page, kv_heads, d) if layout == "nhd" else (pages, kv_heads, page, d)
    codes = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
    codes = codes if layout == "nhd" else codes.transpose(1, 2)
    scales = torch.randint(0, 256, (kv_heads, pages, page), generator=g, device="cuda", dtype=torch.uint8)
    return PackedPages(codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))


def _places(table, totals, new, page):
    where = [(int(table[s, at // page]), at % page) for s, (t, n) in enumerate(zip(totals, new)) for at in range(t - n, t)]
    return [torch.tensor(x, device="cuda") for x in zip(*where)]


def _odd_rows(x, dtype):
    """Rows at the ends and borders of the format among ordinary ones."""
    top = torch.finfo(dtype).max
    odd = [lambda r: r.zero_(), lambda r: r.mul_(torch.finfo(dtype).tiny), lambda r: r.fill_(top), lambda r: r[3].fill_(math.nan),
           lambda r: r[0].fill_(math.inf), lambda r: r[-1].fill_(-math.inf), lambda r: r.clamp_(-1, 1)[5].fill_(448.0),
           lambda r: r.clamp_(-1, 1)[5].fill_(450.0), lambda r: r.clamp_(-1, 1)[5].fill_(-1.75), lambda r: r.zero_()[1].fill_(2.0 ** -24),
           lambda r: r.clamp_(-1, 1)[2].fill_(60000.0)]
    flat = x.view(-1, x.shape[-1])
    for i, change in enumerate(odd):
        if i < len(flat):
            change(flat[(i * 7) % len(flat)])
    return x


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("new,totals,kv_heads,d,page", [
    ([1], [1], 1, 64, 8), ([3, 1, 0, 9], [30, 1, 5, 9], 2, 128, 16), ([40, 77], [100, 77], 3, 64, 24), ([700], [2000], 12, 128, 1560)])
def test_store_writes_the_format_and_only_the_new_tokens(new, totals, kv_heads, d, page, dtype, layout):
    from reelcache_b200.ops import paged
    g = _gen(d + page)
    *_, table, kv_lens, cu_q = paged_batch(g, new, totals, 1, 64, page, BF16)
    pages = int(table.max()) + 4
    k_pages, v_pages = (_noise_pages(g, pages, page, kv_heads, d, layout) for _ in range(2))
    before = [_bytes(p) for p in (k_pages, v_pages)]
    fused = torch.randn(sum(new) + 2, 2 * kv_heads, d, generator=g, device="cuda").mul_(3).to(dtype)  # two rows of no sequence
    k, v = (_odd_rows(x.contiguous(), dtype) for x in fused.split(kv_heads, dim=1))
    paged.store(k, v, k_pages, v_pages, table, kv_lens, cu_q)
    at = _places(table, totals, new, page)
    for rows, got, (codes, scales) in zip((k, v), (k_pages, v_pages), before):
        want, power = quantise(rows[:sum(new)], dtype)
        codes[at[0], at[1]] = want.float().to(torch.float8_e4m3fn).view(torch.uint8)
        scales[:, at[0], at[1]] = (power + 127).to(torch.uint8).T
        now = _bytes(got)
        nan = (codes & 127) == 127  # a NaN of either sign
        assert torch.equal(now[0].masked_fill(nan, 0), codes.masked_fill(nan, 0)) and bool(((now[0] & 127) == 127)[nan].all())
        assert torch.equal(now[1], scales)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("new,totals,heads,kv_heads,d,page", [
    ([1, 1], [40, 1], 8, 2, 128, 16), ([5, 33], [5, 80], 3, 3, 64, 8), ([900], [1700], 12, 12, 128, 1560), ([64] * 9, [64] * 9, 40, 1, 64, 64)])
def test_append_rounds_the_rotated_rows_once(new, totals, heads, kv_heads, d, page, dtype, layout):
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = _gen(heads + d)
    rope = AxisRope.wan(d, layout=layout)
    *_, table, kv_lens, cu_q = paged_batch(g, new, totals, 1, 64, page, BF16)
    k_pages, v_pages = (_noise_pages(g, int(table.max()) + 4, page, kv_heads, d) for _ in range(2))
    before = [_bytes(p) for p in (k_pages, v_pages)]
    tokens = sum(new)
    fused = torch.randn(tokens, heads + 2 * kv_heads, d, generator=g, device="cuda").to(dtype)
    q, k, v = fused.split([heads, kv_heads, kv_heads], dim=1)
    positions = torch.randint(0, 4000, (tokens, 3), generator=g, device="cuda", dtype=torch.int32)
    turned = paged.append(q, k, v, positions, rope, k_pages, v_pages, table, kv_lens, cu_q)
    want, size = spun(q, positions, rope.sections, 10000.0, layout)
    assert within(turned, want, rotate_bound(want, size, dtype))
    at = _places(table, totals, new, page)
    want, size = spun(k, positions, rope.sections, 10000.0, layout)
    got, power = held(k_pages)[at[0], at[1]], k_pages.scales.view(torch.uint8)[:, at[0], at[1]].T.to(torch.int32) - 127
    # half a step of four significant bits, or of the smallest ones; and the rotation in FP32
    assert within(got, want, want.abs() * 2.0 ** -4 + torch.exp2(power.double())[..., None] * 2.0 ** -10 + size * 2.0 ** -20)
    top = want.abs().amax(dim=-1) * torch.exp2(-power.double())
    assert float(top.max()) <= 448.0 * (1 + 2.0 ** -20) and float(top.min()) > 224.0 * (1 - 2.0 ** -20)
    codes, power = quantise(v, dtype)
    assert torch.equal(held(v_pages)[at[0], at[1]], codes * torch.exp2(power.double())[..., None])
    untouched = torch.ones(k_pages.codes.shape[:2], dtype=torch.bool, device="cuda")
    untouched[at[0], at[1]] = False
    for now, was in zip((_bytes(k_pages), _bytes(v_pages)), before):
        assert torch.equal(now[0][untouched], was[0][untouched]) and torch.equal(now[1][:, untouched], was[1][:, untouched])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens,kv_heads,d,page", [([1], 1, 64, 8), ([0, 30, 1, 0, 77], 3, 128, 16), ([2000, 13], 12, 128, 1560), ([100] * 300, 2, 64, 24)])
def test_read_gives_what_is_held(lens, kv_heads, d, page, dtype):
    from reelcache_b200.ops import paged
    g = _gen(len(lens))
    k, v, table, _, starts = paged_batch(g, lens, lens, kv_heads, d, page, torch.float32, width_extra=3)
    pages = [pack_pages(x * torch.exp2(torch.randint(-14, 6, (*x.shape[:3], 1), generator=g, device="cuda").float()), dtype) for x in (k, v)]
    total = sum(lens)
    got = paged.read(*pages, table[:, :-1], starts, total + 5, dtype=dtype)
    for x, p in zip(got, pages):
        rows = held(p)
        want = torch.cat([rows[table[s, :-(-n // page)].long()].flatten(0, 1)[:n] for s, n in enumerate(lens)])
        assert x.dtype == dtype and torch.equal(x[:total].double(), want)


def test_read_of_pages_outside_the_pool(cuda_device):
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext, paged
    g = _gen(0)
    pages = _noise_pages(g, 3, 16, 2, 64)
    pages.scales.view(torch.uint8).fill_(127)
    table = torch.tensor([[0, 7, 2]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 60], dtype=torch.int32, device="cuda")  # and longer than the table
    k, _ = paged.read(pages, pages, table, starts, 60)
    assert not k[16:32].any() and not k[48:].any()
    assert torch.equal(k[:16].double().nan_to_num(), held(pages)[0].nan_to_num())
    with pytest.raises(DeviceStatusError, match="0x403"):
        _ext.check_status(cuda_device)


# -- attention --------------------------------------------------------------------------------------------------------

def _check(new, totals, heads, kv_heads, d, page, dtype, *, seed=0, spread=1.0, scales=0, noise=False, layout="nhd", **mask):
    """Packed attention against 64 bits. Bounds: those of 16-bit pages; the codes' products take the probabilities in fp16, whose
    error is below bf16's but for values under its normal range: 2^-25 of the largest row's magnitude, twice that in
    the scale's steps, for every key."""
    from reelcache_b200.ops import paged
    g = _gen(seed + sum(totals) + d)
    k, v, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, page, torch.float32)
    packed = []
    for x in (k, v):
        if scales:
            x = x * torch.exp2(torch.randint(-scales, scales + 1, (*x.shape[:3], 1), generator=g, device="cuda").float())
        p = pack_pages(x, dtype)
        if layout == "hnd":
            p = paged.PackedPages(p.codes.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(torch.float8_e4m3fn), p.scales)
        packed.append(p)
    values = [held(p, dtype) for p in packed]
    if noise:  # what no session holds: any bytes
        free = torch.ones(k.shape[:2], dtype=torch.bool, device="cuda")
        for s, t in enumerate(totals):
            for b in range(-(-t // page)):
                free[int(table[s, b]), :min(page, t - b * page)] = False
        for p in packed:
            p.codes.view(torch.uint8)[free] = torch.randint(0, 256, p.codes[free].shape, generator=g, device="cuda", dtype=torch.uint8)
            p.scales.view(torch.uint8)[:, free] = 255
    q = (torch.randn(sum(new), heads, d, generator=g, device="cuda") * spread).to(dtype)
    out, lse = paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=max(new), return_lse=True, **mask)
    want, want_lse, bound, lse_bound = attend(q, *values, table, kv_lens, new, **mask)
    largest = max((float(x[torch.isfinite(x)].abs().max()) for x in values[1:] if x.numel()), default=0.0)
    assert within(out, want, bound + max(totals, default=0) * 2.0 ** -24 * largest)
    assert within(lse, want_lse, lse_bound)


FEW = [([1], [1]), ([1], [64]), ([1, 1, 1], [3, 700, 129]), ([1] * 30, [5 + 37 * i for i in range(30)]), ([1, 0, 1], [65, 9, 2])]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(1, 1, 64, 8), (8, 1, 128, 16), (12, 12, 128, 24), (20, 2, 64, 64), (45, 3, 128, 200)])
@pytest.mark.parametrize("new,totals", FEW)
def test_single_tokens(new, totals, heads, kv_heads, d, page, dtype):
    _check(new, totals, heads, kv_heads, d, page, dtype, causal=True, scales=6)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("new,totals,heads,kv_heads,d,page,dtype", [
    ([2, 8], [50, 8], 4, 2, 128, 16, BF16), ([16], [300], 2, 2, 64, 8, FP16), ([5, 3], [5, 4000], 3, 1, 128, 1560, BF16),
    ([17], [100], 1, 1, 128, 32, BF16), ([40, 9, 120], [333, 9, 1000], 8, 2, 64, 24, FP16), ([700], [1900], 4, 4, 128, 1560, BF16),
    ([300] * 4, [3000, 301, 500, 300], 10, 2, 128, 128, FP16)])
def test_drafts_and_chunks(new, totals, heads, kv_heads, d, page, dtype, causal):
    _check(new, totals, heads, kv_heads, d, page, dtype, causal=causal, scales=4)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("new,totals,heads,kv_heads,d", [
    ([12, 1, 0, 7], [700, 300, 40, 7], 8, 2, 128), ([12] * 40, [300 + 17 * i for i in range(40)], 8, 2, 64), ([3, 2, 1], [90, 4000, 65], 48, 3, 64),
    ([1] * 9, [50 + 333 * i for i in range(9)], 37, 1, 128), ([17], [2000], 2, 1, 128), ([24] * 20, [24 + 90 * i for i in range(20)], 2, 1, 64)])
def test_slices_of_rows(new, totals, heads, kv_heads, d, causal):
    """17 to 48 rows: slices of 16, of which some sequences have fewer, in a line and in clusters."""
    _check(new, totals, heads, kv_heads, d, 16, BF16, causal=causal, scales=4, noise=True)


@pytest.mark.parametrize("new,totals,heads,page", [([1, 1], [70, 333], 4, 16), ([3], [41], 4, 24), ([20], [141], 4, 24), ([200, 3], [333, 3], 2, 64)])
def test_what_no_session_holds_may_hold_anything(new, totals, heads, page):
    _check(new, totals, heads, 2, 128, page, BF16, noise=True, causal=True, scales=3)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (100, 64), (100, 130), (5000, 10)])
@pytest.mark.parametrize("new,totals,heads,page", [([1, 1], [500, 90], 4, 16), ([4], [900], 4, 8), ([150], [900], 3, 40)])
def test_windows_and_sinks(new, totals, heads, page, window, sinks, causal):
    _check(new, totals, heads, 1, 128, page, BF16, causal=causal, window=window, sinks=sinks, scales=3, noise=True)


@pytest.mark.parametrize("new,totals", [([5], [2]), ([60, 1], [40, 0]), ([1, 1], [0, 0])])
def test_rows_that_see_nothing(new, totals):
    _check(new, totals, 3, 1, 64, 8, BF16, causal=True)


@pytest.mark.parametrize("new", [1, 4, 60])
def test_growing_scores_and_scales(new):
    """Maxima and units that move again and again: scores that grow along the sequence, V rows of very different sizes."""
    _check([new], [2000], 4, 1, 128, 16, BF16, spread=12.0, scales=20, causal=True)
    _check([new], [700], 4, 1, 64, 16, FP16, spread=12.0, scales=6, causal=True)


@pytest.mark.parametrize("new", [1, 4, 60])
def test_page_layouts(new):
    _check([new, new], [300, 90], 4, 2, 128, 16, BF16, layout="hnd", causal=True)


@pytest.mark.parametrize("new", [1, 30])
def test_rows_that_are_not_numbers(new):
    """A row of K that holds NaN makes the scores of those that see it NaN, one of V their outputs."""
    from reelcache_b200.ops import paged
    g = _gen(new)
    k, v, table, kv_lens, cu_q = paged_batch(g, [new, new], [100, 90], 2, 64, 16, torch.float32)
    packed = [pack_pages(x, BF16) for x in (k, v)]
    page = int(table[0, 2])
    for p, head in zip(packed, (0, 1)):
        p.codes.view(torch.uint8)[page, 3, head] = 127
        p.scales.view(torch.uint8)[head, page, 3] = 255
    q = torch.randn(2 * new, 4, 64, generator=g, device="cuda").to(BF16)
    out, lse = paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=new, return_lse=True)
    assert bool(out[:new].isnan().all()) and bool(lse[:new, :2].isnan().all())
    assert bool(out[new:].isfinite().all()) and bool(lse[new:].isfinite().all()) and bool(lse[:new, 2:].isfinite().all())


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("new,totals,heads,kv_heads", [([1, 1], [100, 37], 8, 2), ([3], [90], 3, 3), ([40, 7], [300, 70], 8, 2), ([128] * 2, [700, 700], 4, 4)])
def test_a_table_for_each_kv_head(new, totals, heads, kv_heads, packed):
    """Heads that read pages of their own, against each head by itself."""
    from reelcache_b200.ops import paged
    g = _gen(7)
    k, v, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, 64, 16, BF16, extra=40)
    orders = torch.stack([torch.randperm(k.shape[0], generator=g, device="cuda") for _ in range(kv_heads)]).to(torch.int32)
    tables = torch.where(table[:, None] >= 0, orders[:, table.clamp(min=0).long()].transpose(0, 1), -1).contiguous()
    if packed:
        k, v = pack_pages(k, BF16), pack_pages(v, BF16)
        k16, v16 = held(k, BF16), held(v, BF16)
    else:
        k16, v16 = k, v
    q = torch.randn(sum(new), heads, 64, generator=g, device="cuda").to(BF16)
    out, lse = paged.attention(q, k, v, tables, kv_lens, cu_q, max_q_len=max(new), causal=True, return_lse=True)
    group = heads // kv_heads
    for h in range(kv_heads):
        mine = slice(h * group, (h + 1) * group)
        want, want_lse, bound, lse_bound = attend(q[:, mine], k16[:, :, h:h + 1], v16[:, :, h:h + 1], tables[:, h], kv_lens, new, causal=True)
        assert within(out[:, mine], want, bound + max(totals) * 2.0 ** -24 * float(v16.abs().max()))
        assert within(lse[:, mine], want_lse, lse_bound)


@pytest.mark.parametrize("new", [1, 200])
def test_pages_beyond_32_bit_offsets(new):
    from reelcache_b200.ops import paged
    g = _gen(1)
    pages, page = 2200, 1024  # 2.3 GB of codes
    codes = torch.zeros(pages, page, 8, 128, dtype=torch.uint8, device="cuda")
    scales = torch.full((8, pages, page), 127, dtype=torch.uint8, device="cuda")
    big = paged.PackedPages(codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    rows = torch.randn(3 * page - 100, 8, 128, generator=g, device="cuda").to(BF16)
    kv_lens = torch.tensor([len(rows)], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, len(rows)], dtype=torch.int32, device="cuda")
    other = paged.PackedPages.empty(pages, page, 8, 128, "cuda")
    paged.store(rows, rows, big, other, table, kv_lens, starts)
    k, v = paged.read(big, other, table, starts, len(rows))
    want, power = quantise(rows, BF16)
    assert torch.equal(k, v) and torch.equal(k.double(), want * torch.exp2(power.double())[..., None])
    q = torch.randn(new, 8, 128, generator=g, device="cuda").to(BF16)
    cu_q = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    out = paged.attention(q, big, other, table, kv_lens, cu_q, max_q_len=new, causal=True)
    flat = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    want, _, bound, _ = attend(q, k[None], v[None], flat, kv_lens, [new], causal=True)
    assert within(out, want, bound + len(rows) * 2.0 ** -24 * float(v.abs().max()))


@pytest.mark.parametrize("new", [1, 6, 150])
def test_repeats_bits_on_streams_and_in_a_graph(new, cuda_device):
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext, paged
    g = _gen(3)
    k, v, table, kv_lens, cu_q = paged_batch(g, [new] * 3, [900, 333, 150], 2, 128, 16, torch.float32)
    packed = [pack_pages(x, BF16) for x in (k, v)]
    q = torch.randn(3 * new, 8, 128, generator=g, device="cuda").to(BF16)
    rows = torch.randn(3 * new, 2, 128, generator=g, device="cuda").to(BF16)

    def step():
        paged.store(rows, rows, *packed, table, kv_lens, cu_q)
        return paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=new, causal=True)

    first = step()
    for _ in range(3):
        assert torch.equal(step(), first)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=new, causal=True))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    rows.copy_(torch.randn(rows.shape, generator=g, device="cuda"))
    q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
    kv_lens.sub_(1)
    graph.replay()
    got = out.clone()
    assert torch.equal(step(), got) and not torch.equal(got, first)
    if new == 150:  # the last sequence is now shorter than its new tokens: one has no place, which is reported
        with pytest.raises(DeviceStatusError, match="0x403"):
            _ext.check_status(cuda_device)


def test_refusals():
    from reelcache_b200.errors import ConfigurationError, UnsupportedError
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = _gen(0)
    k, v, table, kv_lens, cu_q = paged_batch(g, [2], [20], 2, 64, 16, BF16)
    kp, vp = pack_pages(k, BF16), pack_pages(v, BF16)
    rows = torch.randn(2, 2, 64, device="cuda").to(BF16)
    q = torch.randn(2, 4, 64, device="cuda").to(BF16)
    at = (table, kv_lens, cu_q)
    positions = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    rope = AxisRope.wan(64)
    for call in (lambda: paged.attention(q, kp, v, *at, max_q_len=2), lambda: paged.store(rows, rows, kp, v, *at), lambda: paged.store(rows, rows, k, v, *at),
                 lambda: paged.read(k, v, table, cu_q, 2), lambda: paged.append(q, rows, rows, positions, rope, k, vp, *at),
                 lambda: paged.blocks(kp, 12), lambda: paged.blocks(kp, 32)):
        with pytest.raises(ConfigurationError):
            call()
    for call in (lambda: paged.store(rows.cpu(), rows.cpu(), kp, vp, *at), lambda: paged.attention(q.cpu(), kp, vp, *at, max_q_len=2)):
        with pytest.raises(UnsupportedError):
            call()
    wide = PackedWith(kp, codes=kp.codes.view(torch.uint8))
    flat = PackedWith(kp, scales=kp.scales.view(torch.uint8))
    turned = PackedWith(kp, scales=kp.scales.view(torch.uint8).permute(1, 2, 0).contiguous().permute(2, 0, 1).view(torch.float8_e8m0fnu))
    fp32 = torch.randn(2, 2, 64, device="cuda")
    for call in (lambda: paged.store(rows, rows, wide, vp, *at), lambda: paged.store(rows, rows, flat, vp, *at), lambda: paged.store(rows, rows, turned, vp, *at),
                 lambda: paged.store(rows, rows, kp, kp, *at), lambda: paged.store(fp32, fp32, kp, vp, *at), lambda: paged.store(rows[:, :1], rows[:, :1], kp, vp, *at),
                 lambda: paged.store(rows, rows[:1], kp, vp, *at), lambda: paged.store(rows.clone().requires_grad_(), rows, kp, vp, *at),
                 lambda: paged.attention(q, PackedWith(kp, codes=kp.codes[:-1]), vp, *at, max_q_len=2), lambda: paged.attention(q.half(), k, v, *at, max_q_len=2),
                 lambda: paged.attention(q, kp, vp, table[:, None].expand(-1, 3, -1), kv_lens, cu_q, max_q_len=2),
                 lambda: paged.read(kp, vp, table, cu_q.long(), 2), lambda: paged.read(kp, vp, table, cu_q, 2, dtype=torch.float32),
                 lambda: paged.append(q.clone().requires_grad_(), rows, rows, positions, rope, kp, vp, *at)):
        with pytest.raises(RuntimeError):
            call()


def PackedWith(pages, **parts):
    return pages._replace(**parts)


def test_stores_of_nothing_and_without_sequences():
    from reelcache_b200.ops import paged
    pages = [paged.PackedPages.empty(2, 16, 2, 64, "cuda") for _ in range(2)]
    none = torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    zeros = torch.zeros(2, dtype=torch.int32, device="cuda")
    paged.store(none, none, *pages, table, zeros[:1], zeros)
    rows = torch.ones(3, 2, 64, dtype=BF16, device="cuda")
    paged.store(rows, rows, *pages, table[:0], zeros[:0], zeros[:1])
    assert not any(held(p).any() for p in pages)
    k, v = paged.read(*pages, table, zeros, 0)
    assert k.shape == (0, 2, 64) and v.shape == k.shape
    version = pages[0].codes._version
    paged.store(rows[:1], rows[:1], *pages, table, torch.ones_like(zeros[:1]), torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    assert pages[0].codes._version > version and float(held(pages[1])[0, 0].min()) == 1.0


@pytest.mark.parametrize("new", [1, 40])
def test_attention_over_pages_outside_the_pool(new, cuda_device):
    """Such pages read as zeros and are reported."""
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext, paged
    g = _gen(4)
    k, v, table, kv_lens, cu_q = paged_batch(g, [new], [200], 2, 128, 16, torch.float32)
    packed = [pack_pages(x, BF16) for x in (k, v)]
    values = [held(p, BF16) for p in packed]
    q = torch.randn(new, 4, 128, generator=g, device="cuda").to(BF16)
    bad = table.clone()
    bad[0, 2], bad[0, 5] = -1, 10 ** 6
    out = paged.attention(q, *packed, bad, kv_lens, cu_q, max_q_len=new, causal=True)
    with pytest.raises(DeviceStatusError, match="0x403"):
        _ext.check_status(cuda_device)
    for x in values:
        x[table[0, [2, 5]].long()] = 0.0
    want, _, bound, _ = attend(q, *values, table, kv_lens, [new], causal=True)
    assert within(out, want, bound + 200 * 2.0 ** -24 * float(values[1].abs().max()))


def test_many_kv_heads_side_by_side():
    """The line of few rows with head numbers that have no divisor up to 32, and with more heads than that."""
    _check([1] * 30, [600 + 30 * i for i in range(30)], 37, 37, 64, 64, BF16, causal=True)
    _check([1] * 20, [600 + 30 * i for i in range(20)], 80, 40, 64, 64, BF16, causal=True)


@pytest.mark.parametrize("seqs", [1, 60])
@pytest.mark.parametrize("new,bound", [(5, 1), (9, 3), (16, 9)])
def test_more_new_tokens_than_the_bound_are_reported(new, bound, seqs, cuda_device):
    """The tokens up to the bound have their results; rows that the kernel does not take are left as they were."""
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext, paged
    g = _gen(new)
    k, v, table, kv_lens, cu_q = paged_batch(g, [new] * seqs, [700 + i for i in range(seqs)], 2, 64, 16, torch.float32)
    packed = [pack_pages(x, BF16) for x in (k, v)]
    values = [held(p, BF16) for p in packed]
    q = torch.randn(new * seqs, 8, 64, generator=g, device="cuda").to(BF16)
    out = torch.full_like(q, 7.0)
    paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=bound, causal=True, out=out)
    with pytest.raises(DeviceStatusError, match="0x404"):
        _ext.check_status(cuda_device)
    want, _, error, _ = attend(q, *values, table, kv_lens, [new] * seqs, causal=True)
    # tokens of the rows that the kernel takes: eight, or slices of 16 (9 tokens of four rows: 36, three slices, 12 tokens)
    took = 2 if bound * 4 <= 8 else -(-bound * 4 // 16) * 4
    for s in range(seqs):
        rows = slice(s * new, s * new + bound)
        assert within(out[rows], want[rows], error[rows] + 800 * 2.0 ** -24 * float(values[1].abs().max()))
        assert bool((out[s * new + took:(s + 1) * new] == 7.0).all())
