"""Means of blocks in a cache whose batches are written out of turn."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _want(cache, session, rows):
    """Means of the blocks of a session's rows, rounded once."""
    size = cache.block
    return torch.stack([rows[b * size:(b + 1) * size].double().mean(dim=0) for b in range(-(-session.length // size))]).to(BF16)


def _have(cache, session):
    pages = cache.table.block_table[session.slot, :len(session.blocks)].long()
    return cache.means[0, pages].flatten(0, 1)[:-(-session.length // cache.block)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("block", [8, 24])
def test_a_batch_written_again_after_later_ones(packed, block):
    """A session takes tokens in two batches; the first is written once more, and in another order: blocks that hold tokens of both
    have the mean of all of them."""
    from reelcache_b200.ops.rope import AxisRope
    from reelcache_b200.paged_cache import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(block)
    cache = PagedKVCache(1, 2, 64, pages=20, page_size=24, max_sessions=3, max_tokens=200, packed=packed, block=block)
    rope = AxisRope.wan(64)
    a, b = cache.open(), cache.open()

    def write(batch):
        q, k, v = (torch.randn(batch.tokens, h, 64, generator=g, device="cuda").to(BF16) for h in (4, 2, 2))
        cache.append(0, batch, q, k, v, torch.zeros(batch.tokens, 3, dtype=torch.int32, device="cuda"), rope)

    def rows(session):
        if packed:
            return cache.read(0, [session])[0]
        pages = cache.table.block_table[session.slot, :len(session.blocks)].long()
        return cache.storage[0, 0, pages].flatten(0, 1)[:session.length]

    first, second = cache.extend([(a, 30), (b, 5)]), cache.extend([(a, 45), (b, 0)])
    third = cache.extend([(b, 70)])
    for batch in (first, second, third, first, third, second, first):
        write(batch)
    for s in (a, b):
        assert torch.equal(_have(cache, s), _want(cache, s, rows(s)))
    for batch in (third, second, first):  # (of the whole history again)
        write(batch)
    for s in (a, b):
        assert torch.equal(_have(cache, s), _want(cache, s, rows(s)))


def test_rows_that_a_kernel_wrote_itself():
    from reelcache_b200.paged_cache import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(0)
    cache = PagedKVCache(1, 2, 64, pages=8, page_size=16, max_sessions=2, max_tokens=100, block=16)
    a = cache.open()
    first, second = cache.extend([(a, 20)]), cache.extend([(a, 20)])
    for batch in (second, first):
        cache.token_rows(0, "K")[cache.new_rows(batch)] = torch.randn(20, 128, generator=g, device="cuda").to(BF16)
        cache.rows_written(0, batch)
    pages = cache.table.block_table[a.slot, :3].long()
    assert torch.equal(_have(cache, a), _want(cache, a, cache.storage[0, 0, pages].flatten(0, 1)[:40]))


def test_an_earlier_batch_in_a_captured_call():
    """What a captured call reads is the cache's and its own, not host memory that is reused."""
    from reelcache_b200.paged_cache import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = PagedKVCache(1, 2, 64, pages=8, page_size=16, max_sessions=2, max_tokens=100, packed=True, block=16)
    a = cache.open()
    first, second = cache.extend([(a, 20)]), cache.extend([(a, 20)])
    rows = [torch.randn(20, 2, 64, generator=g, device="cuda").to(BF16) for _ in range(4)]
    cache.store(0, second, *rows[2:])
    cache.store(0, first, *rows[:2])  # (warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.store(0, first, *rows[:2])
    for n in range(1, 40):
        cache._ints([n] * 5)  # other users of pinned memory
    rows[0].normal_(generator=g)
    cache.means.zero_()
    graph.replay()
    k, _ = cache.read(0, [a])
    want, have = _want(cache, a, k), _have(cache, a)
    assert torch.equal(have, want)
