"""Many rows over packed pages: room for what a window leaves, and results where fewer pages have a place."""

import pytest
import torch

from .paged_support import attend, paged_batch, within
from .sparse_support import held, pack_pages

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _batch(new, totals, heads, page, seed=0, width_extra=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k, v, table, kv_lens, cu_q = paged_batch(g, new, totals, 2, 64, page, torch.float32, width_extra=width_extra)
    packed = [pack_pages(x, BF16) for x in (k, v)]
    q = torch.randn(sum(new), heads, 64, generator=g, device="cuda").to(BF16)
    return q, packed, table, kv_lens, cu_q


def test_room_follows_the_window(cuda_device):
    from reelcache_b200.ops import _ext, paged
    q, packed, table, kv_lens, cu_q = _batch([100], [60000], 2, 64)
    want = paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=100, causal=True, window=500, sinks=70)
    torch.cuda.synchronize()
    held_now = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=100, causal=True, window=500, sinks=70)
    # 256 tokens of row tiles + 500 + 256 of tiles' edges + 198 of sinks: 24 pages of 2 x 16 KB, and a few bytes a page of the pool
    assert torch.cuda.max_memory_allocated() - held_now < 3 << 20
    assert torch.equal(out, want)
    exact, _, bound, _ = attend(q, *(held(p, BF16) for p in packed), table, kv_lens, [100], causal=True, window=500, sinks=70)
    assert within(out, exact, bound)
    _ext.check_status(cuda_device)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 0), (129, 1), (300, 257), (1, 128), (5000, 0)])
@pytest.mark.parametrize("new,totals,heads,page", [([60, 1, 0, 90], [700, 3000, 50, 90], 2, 8), ([700], [4100], 4, 24), ([130] * 3, [130, 2000, 131], 6, 200), ([50], [20], 2, 16)])
def test_windows(new, totals, heads, page, window, sinks, causal, cuda_device):
    from reelcache_b200.ops import _ext, paged
    q, packed, table, kv_lens, cu_q = _batch(new, totals, heads, page, width_extra=2)
    out, lse = paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=max(new), causal=causal, window=window, sinks=sinks, return_lse=True)
    want, want_lse, bound, lse_bound = attend(q, *(held(p, BF16) for p in packed), table, kv_lens, new, causal=causal, window=window, sinks=sinks)
    assert within(out, want, bound) and within(lse, want_lse, lse_bound)
    _ext.check_status(cuda_device)


@pytest.mark.parametrize("window", [None, 1, 200])
@pytest.mark.parametrize("new,bound", [(90, 30), (500, 51), (3000, 130)])
def test_more_new_tokens_than_the_bound(new, bound, window, cuda_device):
    """Reported; the tokens up to the bound have their results, whatever the ones after them read."""
    from reelcache_b200.errors import DeviceStatusError
    from reelcache_b200.ops import _ext, paged
    q, packed, table, kv_lens, cu_q = _batch([new, new], [new + 900, new], 4, 16)
    out = paged.attention(q, *packed, table, kv_lens, cu_q, max_q_len=bound, causal=True, window=window)
    with pytest.raises(DeviceStatusError, match="0x404"):
        _ext.check_status(cuda_device)
    want, _, error, _ = attend(q, *(held(p, BF16) for p in packed), table, kv_lens, [new] * 2, causal=True, window=window)
    for s in range(2):
        rows = slice(s * new, s * new + bound)
        assert within(out[rows], want[rows], error[rows])
