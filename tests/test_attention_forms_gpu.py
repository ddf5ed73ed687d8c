"""What attention_form says of calls over packed pages and with a table for each KV head."""

import pytest
import torch

from .paged_support import attend, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _form(new, heads, kv_heads, seqs, width, page=16, d=128, **kw):
    from reelcache_b200.ops import paged
    return paged.attention_form(new * seqs, heads, kv_heads, d, seqs, width, page, max_q_len=new, **kw)


@pytest.mark.parametrize("d", [64, 128])
def test_packed_pages(d):
    """Up to 8 rows, 16, 48 in slices, and more over expanded pages, whose form is that of 16-bit pages."""
    assert _form(1, 8, 1, 1, 64, d=d, packed=True).startswith("few rows, cluster")
    assert _form(4, 4, 1, 48, 1024, d=d, packed=True) == "few rows, line"
    assert _form(5, 4, 1, 48, 1024, d=d, packed=True) == "2 slices, line" and _form(12, 4, 1, 1, 8, d=d, packed=True).startswith("3 slices, cluster")
    for new, heads, kv_heads, seqs, width in ((49, 1, 1, 4, 100), (13, 4, 1, 2, 30), (600, 4, 4, 1, 1000)):
        assert _form(new, heads, kv_heads, seqs, width, d=d, packed=True) == "expanded, " + _form(new, heads, kv_heads, seqs, width, d=d)
    assert _form(17, 1, 1, 4, 100).startswith("twin")


def test_a_table_for_each_kv_head():
    """Many equal items: whole rounds of them, then the rest in clusters."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    said = _form(128, 10, 10, 37, 99, page=128, tables=True)
    assert said == f"twin 1, then {370 - 370 // sms * sms} items in 2" and _form(128, 10, 10, 37, 99, page=128) != said
    assert _form(128, 1, 1, sms, 50, page=128, tables=True) == "twin 1"
    assert _form(128, 10, 10, 37, 99, page=128, tables=True, packed=True) == "expanded, " + said
    assert _form(1, 8, 2, 1, 64, tables=True) == _form(1, 8, 2, 1, 64)


@pytest.mark.parametrize("rest", [1, 5, 9, 10, 18, 19, 37, 74, 75, 147])
def test_the_rest_of_many_equal_items(rest):
    """Items beyond whole rounds go to clusters of a size that the device holds, as many as fit or in rounds; every item has its result."""
    from reelcache_b200.ops import paged
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    page, keys, kv_heads = 64, 1600, 2 if (sms + rest) % 2 == 0 else 1
    seqs = (sms + rest) // kv_heads
    said = paged.attention_form(64 * seqs, kv_heads, kv_heads, 64, seqs, keys // page, page, max_q_len=64, tables=True)
    assert said.startswith("twin")
    if "then" in said:
        number, size = (int(x) for x in said.split("then ")[1].split(" items in "))
        # (a cluster lies in one of the chip's eight parts of 20 SMs at most)
        assert number == rest and number * size <= sms and number <= 8 * (20 // size)
    g = torch.Generator(device="cuda").manual_seed(rest)
    pages = 64  # that all sequences share, in orders of their own
    k, v = (torch.randn(pages, page, kv_heads, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = torch.randint(0, pages, (seqs, kv_heads, keys // page), generator=g, device="cuda", dtype=torch.int32)
    kv_lens = torch.randint(keys - 300, keys + 1, (seqs,), generator=g, device="cuda", dtype=torch.int32)
    cu_q = torch.arange(seqs + 1, device="cuda", dtype=torch.int32) * 64
    q = torch.randn(64 * seqs, kv_heads, 64, generator=g, device="cuda").bfloat16()
    out = paged.attention(q, k, v, table, kv_lens, cu_q, max_q_len=64, causal=True)
    for h in range(kv_heads):
        want, _, bound, _ = attend(q[:, h:h + 1], k[:, :, h:h + 1], v[:, :, h:h + 1], table[:, h], kv_lens, [64] * seqs, causal=True)
        assert within(out[:, h:h + 1], want, bound)
