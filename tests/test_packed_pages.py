"""Pages in 8 bits and blocks of pages: what needs no GPU."""

import pytest
import torch

from .sparse_support import choose, held, pack_pages, quantise


def test_blocks_are_a_view():
    from reelcache_b200.errors import ConfigurationError
    from reelcache_b200.ops import paged
    pages = torch.arange(4 * 32 * 2 * 64).reshape(4, 32, 2, 64)
    cut = paged.blocks(pages, 8)
    assert cut.shape == (16, 8, 2, 64) and cut.data_ptr() == pages.data_ptr() and torch.equal(cut, pages.reshape(16, 8, 2, 64))
    packed = paged.PackedPages.empty(4, 32, 2, 64, "cpu")
    packed.scales.view(torch.uint8).copy_(torch.arange(256).reshape(2, 4, 32).to(torch.uint8))
    cut = paged.blocks(packed, 16)
    assert cut.codes.shape == (8, 16, 2, 64)
    assert torch.equal(cut.scales.view(torch.uint8), packed.scales.view(torch.uint8).reshape(2, 8, 16))
    layer = torch.zeros(2, 4, 32, 2, 64)[1]
    assert paged.blocks(layer, 32).data_ptr() == layer.data_ptr()
    for bad in (lambda: paged.blocks(pages, 4), lambda: paged.blocks(pages, 24), lambda: paged.blocks(pages, 64), lambda: paged.blocks(pages[::2], 8),
                lambda: paged.blocks(pages.transpose(1, 2).contiguous().transpose(1, 2), 8)):
        with pytest.raises(ConfigurationError):
            bad()


def test_calls_without_cuda_are_refused():
    from reelcache_b200.errors import ConfigurationError, UnsupportedError
    from reelcache_b200.ops import paged
    pages = paged.PackedPages.empty(2, 16, 1, 64, "cpu")
    plain = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    rows, table, lens, cu = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    means = torch.zeros(2, 1, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: paged.store(rows, rows, pages, pages, table, lens, cu), lambda: paged.read(pages, pages, table, cu, 1),
                 lambda: paged.attention(rows, pages, pages, table, lens, cu, max_q_len=1), lambda: paged.block_means(plain, means, table, lens, cu, max_q_len=1),
                 lambda: paged.select_blocks(rows, means, table, lens, cu, block=16, keep=1, max_q_len=1)):
        with pytest.raises(UnsupportedError):
            call()
    with pytest.raises(ConfigurationError):
        paged.read(plain, plain, table, cu, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_format_holds_numbers_of_the_type(dtype):
    """Every code times every scale of a type's range is a number of it, and a row's error is half a step at most."""
    from reelcache_b200.ops.paged import PackedPages
    from .sparse_support import RANGE
    low, high = RANGE[dtype]
    codes = torch.arange(256, dtype=torch.uint8)
    codes = codes[(codes & 127) != 127].view(torch.float8_e4m3fn)
    for k in (low, low + 1, -3, 0, high - 1, high):
        exact = codes.double() * 2.0 ** k
        assert torch.equal(exact.to(dtype).double(), exact)
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(1, 16, 3, 64, generator=g) * torch.exp2(torch.randint(-9, 9, (1, 16, 3, 1), generator=g).float())).to(dtype)
    pages = pack_pages(x, dtype)
    assert isinstance(pages, PackedPages)
    power = pages.scales.view(torch.uint8).permute(1, 2, 0).double() - 127
    assert bool(((held(pages) - x.double()).abs() <= x.double().abs() * 2.0 ** -4 + torch.exp2(power)[..., None] * 2.0 ** -10).all())
    assert torch.equal(quantise(held(pages), dtype)[0] * torch.exp2(quantise(held(pages), dtype)[1].double())[..., None], held(pages))


def test_the_plain_choice():
    """The plain form itself, on a choice that can be told by eye."""
    means = torch.zeros(1, 6, 1, 64, dtype=torch.float64)
    means[0, :, 0, 0] = torch.tensor([5.0, 1.0, 3.0, 3.0, 2.0, 9.0])
    q = torch.zeros(1, 1, 64)
    q[..., 0] = 1.0
    table, lens, cu = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([46]), torch.tensor([0, 1])
    pick = lambda **k: choose(q, means, table, lens, cu, block=8, **k)[0][4][0]  # noqa: E731
    assert pick(keep=2) == [0, 2, 5]  # equal ones: the lower
    assert pick(keep=1, sinks=9) == [0, 1, 2, 5] and pick(keep=0, recent=6) == [4, 5] and pick(keep=9) == list(range(6))
