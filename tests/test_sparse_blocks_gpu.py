"""Means of blocks, the choice of blocks and attention over it on sm_100a, against 64-bit forms."""

import math

import pytest
import torch

from .paged_support import attend, paged_batch, within
from .sparse_support import choose, chosen_table, held, pack_pages

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _means(values, block):
    """Means of whole blocks of pages ``[pages, page_size, kv_heads, d]`` (what earlier calls left)."""
    return values.double().unflatten(1, (-1, block)).mean(dim=2).to(values.dtype)


# -- means ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new,totals,kv_heads,d,page,block", [
    ([1], [1], 1, 64, 8, 8), ([1, 1, 0, 1], [64, 65, 9, 7], 2, 128, 64, 16), ([3, 40], [30, 41], 3, 64, 24, 24), ([700, 33], [2000, 33], 4, 128, 1560, 104),
    ([130], [140], 1, 128, 128, 128)])
def test_means_of_the_blocks_that_hold_new_tokens(new, totals, kv_heads, d, page, block, dtype, packed):
    from reelcache_b200.ops import paged
    g = _gen(d + page)
    k, _, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, page, dtype, fill=math.nan)
    pages = pack_pages(k, dtype) if packed else k
    values = held(pages) if packed else k.double()
    means = torch.randn(k.shape[0], page // block, kv_heads, d, generator=g, device="cuda").to(dtype)
    want = means.clone()
    for s, (n, total) in enumerate(zip(new, totals)):
        for b in range((total - n) // block, -(-total // block) if n else 0):
            at, row = int(table[s, b * block // page]), b * block % page
            there = min(block, total - b * block)
            want[at, b % (page // block)] = (values[at, row:row + there].sum(dim=0) / there).to(dtype)
    assert paged.block_means(pages, means, table, kv_lens, cu_q, max_q_len=max(new)) is means
    assert torch.equal(means, want)


# -- the choice -------------------------------------------------------------------------------------------------------

def _select(q, means, table, kv_lens, cu_q, new, **how):
    """select_blocks against the plain choice: tables, lengths and starts are equal."""
    from reelcache_b200.ops import paged
    chosen = paged.select_blocks(q, means, table, kv_lens, cu_q, max_q_len=max(new), **how)
    items = choose(q, means, table, kv_lens, cu_q, **how)
    rows, lens, cu = chosen_table(items, table, means.shape[1], means.shape[2], chosen.table.shape[0], chosen.table.shape[2], how["block"], int(cu_q[-1]))
    assert chosen.kv_lens.tolist() == lens and chosen.cu_q.tolist() == cu
    assert chosen.table.tolist() == rows
    return chosen, items


SHAPES = [  # new tokens, lengths, heads, KV heads, head dim, page, block
    ([1], [1], 1, 1, 64, 8, 8), ([1, 1, 1], [700, 64, 2000], 8, 2, 128, 64, 16), ([1] * 40, [100 + 61 * i for i in range(40)], 4, 4, 64, 32, 32),
    ([3, 0, 9], [90, 500, 1000], 9, 1, 128, 24, 8), ([100, 37], [900, 37], 16, 1, 64, 104, 104), ([300], [2500], 2, 2, 128, 128, 64),
    ([1], [20000], 8, 2, 128, 16, 16)]


@pytest.mark.parametrize("how", [dict(keep=4), dict(keep=3, sinks=20, recent=50), dict(keep=0, recent=7), dict(keep=10000), dict(keep=1, sinks=5000),
                                 dict(keep=17, query_block=16, recent=1), dict(keep=5, query_block=100, sinks=1)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", SHAPES)
def test_choice_is_the_plain_one(shape, dtype, causal, how):
    new, totals, heads, kv_heads, d, page, block = shape
    g = _gen(sum(totals))
    k, _, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, page, dtype)
    q = torch.randn(sum(new), heads, d, generator=g, device="cuda").to(dtype)
    _select(q, _means(k, block), table, kv_lens, cu_q, new, block=block, causal=causal, **how)


@pytest.mark.parametrize("keep", [1, 7, 40, 299])
@pytest.mark.parametrize("kind", ["equal", "few values", "close", "far apart", "one"])
@pytest.mark.parametrize("new,query_block", [([1], 1), ([33], 16)])
def test_scores_at_the_border(kind, keep, new, query_block):
    """Equal scores go to the lower block, close ones (far below what FP32 tells apart) to the larger."""
    g = _gen(keep)
    totals, block, kv_heads, d = [8 * 303 + new[0]], 8, 2, 128
    k, _, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, 16, BF16)
    q = torch.randn(new[0], 4, d, generator=g, device="cuda").to(BF16)
    means = _means(k, block)
    if kind == "equal":
        means[:] = means[0, 0]
    elif kind == "few values":
        means[:] = means[torch.randint(0, 3, means.shape[:1], generator=g, device="cuda")][:, :1]
    elif kind == "close":  # one channel of a tiny query value moves by steps of bf16 beside a large sum
        means[:] = means[0, 0]
        q[..., 5] = 2.0 ** -30
        means[..., 5] = torch.randint(1, 200, means.shape[:3], generator=g, device="cuda").to(BF16)
    elif kind == "far apart":
        means *= torch.exp2(torch.randint(-60, 60, (*means.shape[:3], 1), generator=g, device="cuda").float()).to(BF16)
    else:
        means[:] = 0.0
        means[int(table[0, 77]), 1] = q[0, 0]
    _select(q, means, table, kv_lens, cu_q, new, block=block, keep=keep, query_block=query_block, causal=True)


def test_means_that_are_not_numbers_come_last():
    g = _gen(0)
    k, _, table, kv_lens, cu_q = paged_batch(g, [1, 20], [900, 900], 2, 64, 16, BF16)
    q = torch.randn(21, 4, 64, generator=g, device="cuda").to(BF16)
    means = _means(k, 16)
    means[torch.rand(means.shape[:3], generator=g, device="cuda") < 0.3] = math.nan
    _select(q, means, table, kv_lens, cu_q, [1, 20], block=16, keep=9, query_block=4, causal=True)
    _select(q, means, table, kv_lens, cu_q, [1, 20], block=16, keep=50, query_block=20)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_queries_and_means(dtype):
    """Sums and products beyond FP32 and fp16."""
    g = _gen(5)
    k, _, table, kv_lens, cu_q = paged_batch(g, [64], [3000], 1, 64, 8, dtype)
    top = 2.0 ** 120 if dtype == BF16 else 30000.0
    q = (torch.randn(64, 2, 64, generator=g, device="cuda") * top).clamp(-top, top).to(dtype)
    means = (_means(k, 8).float() * (2.0 ** 20 if dtype == BF16 else 1000.0)).to(dtype)
    _select(q, means, table, kv_lens, cu_q, [64], block=8, keep=20, query_block=64, causal=True)


def test_many_blocks_and_clusters():
    g = _gen(6)
    k, _, table, kv_lens, cu_q = paged_batch(g, [1], [8 * 12000], 1, 64, 8, BF16)
    q = torch.randn(1, 1, 64, generator=g, device="cuda").to(BF16)
    for keep in (1, 100, 11000):
        _select(q, _means(k, 8), table, kv_lens, cu_q, [1], block=8, keep=keep, recent=20)


# -- attention over the choice ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new,totals,heads,kv_heads,d,page,block,how", [
    ([1, 1], [900, 70], 8, 2, 128, 64, 16, dict(keep=5, sinks=3, recent=20, causal=True)),
    ([6], [3000], 20, 1, 64, 32, 32, dict(keep=9, causal=True)),
    ([200, 9], [1500, 300], 4, 2, 128, 128, 64, dict(keep=4, query_block=32, sinks=64, recent=64, causal=True)),
    ([300], [2900], 3, 3, 128, 1560, 104, dict(keep=6, query_block=128)),
    ([700], [3300], 2, 1, 64, 64, 64, dict(keep=8, query_block=256, sinks=100)),
    ([2, 1], [2, 1], 4, 1, 64, 8, 8, dict(keep=3, causal=True))])
def test_attention_over_chosen_blocks(new, totals, heads, kv_heads, d, page, block, how, dtype, packed):
    """Each query block and KV head against dense attention over its chosen keys put together."""
    from reelcache_b200.ops import paged
    g = _gen(sum(totals))
    k, v, table, kv_lens, cu_q = paged_batch(g, new, totals, kv_heads, d, page, dtype)
    pages = [pack_pages(x, dtype) for x in (k, v)] if packed else [k, v]
    if packed:
        k, v = (held(p, dtype) for p in pages)
    means = _means(k, block)
    paged.block_means(pages[0], means, table, kv_lens, cu_q, max_q_len=max(new))
    q = torch.randn(sum(new), heads, d, generator=g, device="cuda").to(dtype)
    chosen, items = _select(q, means, table, kv_lens, cu_q, new, block=block, **how)
    out, lse = paged.attention(q, *(paged.blocks(p, block) for p in pages), chosen.table, chosen.kv_lens, chosen.cu_q, max_q_len=chosen.max_q_len,
                               causal=how.get("causal", False), return_lse=True)
    group = heads // kv_heads
    for first, count, end, s, blocks in items:
        for h in range(kv_heads):
            at = torch.tensor([p for b in blocks[h] for p in range(b * block, min(end, (b + 1) * block))], device="cuda")
            rows = [x[table[s, at // page].long(), at % page, h][None, :, None] for x in (k, v)]
            mine = slice(h * group, (h + 1) * group)
            want, want_lse, bound, lse_bound = attend(q[first:first + count, mine], *rows, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), [len(at)],
                                                      [count], causal=how.get("causal", False))
            extra = len(at) * 2.0 ** -24 * float(rows[1].abs().max()) if packed else 0.0
            assert within(out[first:first + count, mine], want, bound + extra)
            assert within(lse[first:first + count, mine], want_lse, lse_bound)


@pytest.mark.parametrize("new,query_block", [(1, 1), (70, 32)])
def test_a_step_in_a_graph_and_on_another_stream(new, query_block):
    from reelcache_b200.ops import paged
    g = _gen(2)
    k, v, table, kv_lens, cu_q = paged_batch(g, [new] * 3, [2000, 333, 1500], 2, 128, 64, BF16)
    means = _means(k, 16)
    q = torch.randn(3 * new, 8, 128, generator=g, device="cuda").to(BF16)

    def step():
        paged.block_means(k, means, table, kv_lens, cu_q, max_q_len=new)
        chosen = paged.select_blocks(q, means, table, kv_lens, cu_q, block=16, keep=8, query_block=query_block, max_q_len=new, causal=True)
        return paged.attention(q, paged.blocks(k, 16), paged.blocks(v, 16), chosen.table, chosen.kv_lens, chosen.cu_q, max_q_len=chosen.max_q_len,
                               causal=True)

    first = step()
    assert torch.equal(step(), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    side.synchronize()
    assert torch.equal(again, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
    kv_lens.sub_(5)
    graph.replay()
    got = out.clone()
    assert torch.equal(step(), got) and not torch.equal(got, first)


def test_what_does_not_fit_is_reported(cuda_device):
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext, paged
    g = _gen(0)
    k, v, table, kv_lens, cu_q = paged_batch(g, [5, 3], [400, 90], 1, 64, 16, BF16)
    means, q = _means(k, 16), torch.randn(8, 2, 64, generator=g, device="cuda").to(BF16)
    before = means.clone()
    paged.select_blocks(q, means, table, kv_lens, cu_q, block=16, keep=3, max_q_len=3)  # five new tokens
    with pytest.raises(DeviceStatusError, match="0x404"):
        _ext.check_status(cuda_device)
    paged.block_means(k, means, table, kv_lens, cu_q, max_q_len=4)
    with pytest.raises(DeviceStatusError, match="0x404"):
        _ext.check_status(cuda_device)
    bad = table.clone()
    bad[0, 24], bad[0, 3] = 10000, -1  # the first sequence's last page, and one of its past
    means.copy_(before)
    paged.block_means(k, means, bad, kv_lens, cu_q, max_q_len=5)
    with pytest.raises(DeviceStatusError, match="0x403"):
        _ext.check_status(cuda_device)
    chosen = paged.select_blocks(q, means, bad, kv_lens, cu_q, block=16, keep=50, max_q_len=5)
    assert int((chosen.table[0] == -1).sum()) >= 2 and int(chosen.table.max()) < k.shape[0]
    paged.attention(q, k, v, chosen.table, chosen.kv_lens, chosen.cu_q, max_q_len=1)
    with pytest.raises(DeviceStatusError, match="0x403"):
        _ext.check_status(cuda_device)


def test_refusals():
    from reelcache_b200.ops import paged
    g = _gen(0)
    k, _, table, kv_lens, cu_q = paged_batch(g, [2], [90], 2, 64, 16, BF16)
    means, q = _means(k, 8), torch.randn(2, 4, 64, generator=g, device="cuda").to(BF16)
    at = (table, kv_lens, cu_q)
    pick = lambda **k: paged.select_blocks(**{**dict(q=q, means=means, block_table=table, kv_lens=kv_lens, cu_q=cu_q, block=8, keep=2, max_q_len=2), **k})  # noqa: E731
    pick()
    for wrong in (dict(keep=-1), dict(sinks=-1), dict(recent=-1), dict(query_block=0), dict(max_q_len=0), dict(block=12), dict(block=4), dict(q=q.half()),
                  dict(q=q[:, :3]), dict(q=q.float()), dict(means=means.float()), dict(means=means[..., :32]), dict(q=q.clone().requires_grad_()),
                  dict(block_table=table[:, None].expand(-1, 2, -1)), dict(cu_q=cu_q.long()),
                  dict(block_table=table[:, :1].expand(-1, 20000), block=8)):
        with pytest.raises(RuntimeError):
            pick(**wrong)
    fp16 = means.half()
    for call in (lambda: paged.block_means(k, fp16, *at, max_q_len=2), lambda: paged.block_means(k, means[:-1], *at, max_q_len=2),
                 lambda: paged.block_means(k, means[:, :0], *at, max_q_len=2), lambda: paged.block_means(k, _means(k, 4), *at, max_q_len=2),
                 lambda: paged.block_means(k, means.clone().requires_grad_(), *at, max_q_len=2), lambda: paged.block_means(k, means, *at, max_q_len=0)):
        with pytest.raises(RuntimeError):
            call()


def test_calls_without_tokens_or_sequences():
    from reelcache_b200.ops import paged
    g = _gen(0)
    k, _, table, kv_lens, cu_q = paged_batch(g, [2], [90], 2, 64, 16, BF16)
    means, q = _means(k, 16), torch.randn(2, 4, 64, generator=g, device="cuda").to(BF16)
    none = paged.select_blocks(q[:0], means, table, kv_lens, torch.zeros_like(cu_q), block=16, keep=2, max_q_len=1)
    assert none.table.shape[0] == 0 and none.cu_q.tolist() == [0]
    rest = paged.select_blocks(q, means, table[:0], kv_lens[:0], cu_q[:1], block=16, keep=2, max_q_len=1)
    assert rest.table.shape[0] == 0
    before = means.clone()
    paged.block_means(k, means, table[:0], kv_lens[:0], cu_q[:1], max_q_len=1)
    paged.block_means(k, means, table, kv_lens, torch.zeros_like(cu_q), max_q_len=1)
    assert torch.equal(means, before)


@pytest.mark.parametrize("query_block", [1, 3])
def test_many_sequences_and_rows_of_none(query_block):
    """More sequences than a CTA has threads, rows of q before the first and behind the last of them."""
    from reelcache_b200.ops import paged
    g = _gen(8)
    new = [(i * 7) % 4 for i in range(700)]
    totals = [n + (i * 37) % 300 for i, n in enumerate(new)]
    k, v, table, kv_lens, cu_q = paged_batch(g, new, totals, 1, 64, 16, BF16)
    q = torch.randn(sum(new) + 9, 2, 64, generator=g, device="cuda").to(BF16)
    means = _means(k, 16)
    chosen, _ = _select(q, means, table, kv_lens, cu_q + 4, new, block=16, keep=2, query_block=query_block, causal=True)
    out = torch.full_like(q, 7.0)
    paged.attention(q, k, v, chosen.table, chosen.kv_lens, chosen.cu_q, max_q_len=chosen.max_q_len, causal=True, out=out)
    assert bool((out[:4] == 7.0).all()) and bool((out[sum(new) + 4:] == 7.0).all()) and not bool((out[4:sum(new) + 4] == 7.0).any())


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("new,totals", [([5], [2]), ([40, 1], [30, 0]), ([3, 2], [0, 700])])
def test_tokens_before_the_first_position(new, totals, causal):
    from reelcache_b200.ops import paged
    g = _gen(9)
    k, v, table, kv_lens, cu_q = paged_batch(g, new, totals, 2, 64, 8, BF16)
    q = torch.randn(sum(new), 4, 64, generator=g, device="cuda").to(BF16)
    means = _means(k, 8)
    paged.block_means(k, means, table, kv_lens, cu_q, max_q_len=max(new))
    chosen, _ = _select(q, means, table, kv_lens, cu_q, new, block=8, keep=200, query_block=4, causal=causal)
    out, lse = paged.attention(q, k, v, chosen.table, chosen.kv_lens, chosen.cu_q, max_q_len=chosen.max_q_len, causal=causal, return_lse=True)
    want, want_lse, bound, lse_bound = attend(q, k, v, table, kv_lens, new, causal=causal)
    assert within(out, want, bound) and within(lse, want_lse, lse_bound)


@pytest.mark.parametrize("packed", [False, True])
def test_more_rounds_than_sms(packed):
    """Items of up to 128 rows in more than one round, the last ones in clusters."""
    from reelcache_b200.ops import paged
    g = _gen(10)
    k, v, table, kv_lens, cu_q = paged_batch(g, [2700], [9000], 4, 64, 64, BF16)
    pages = [pack_pages(x, BF16) for x in (k, v)] if packed else [k, v]
    if packed:
        k, v = (held(p, BF16) for p in pages)
    q = torch.randn(2700, 4, 64, generator=g, device="cuda").to(BF16)
    chosen = paged.select_blocks(q, _means(k, 64), table, kv_lens, cu_q, block=64, keep=10000, query_block=60, max_q_len=2700, causal=True)
    assert chosen.table.shape[0] * 4 % 148 != 0 and chosen.table.shape[0] * 4 > 148
    out, lse = paged.attention(q, *pages, chosen.table, chosen.kv_lens, chosen.cu_q, max_q_len=60, causal=True, return_lse=True)
    want, want_lse, bound, lse_bound = attend(q, k, v, table, kv_lens, [2700], causal=True)
    assert within(out, want, bound) and within(lse, want_lse, lse_bound)
