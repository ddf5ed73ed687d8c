"""The paged operators' refusals and bookkeeping that need no GPU."""

import pytest
import torch

from reelcache_b200.errors import ConfigurationError, UnsupportedError


@pytest.mark.parametrize("args", [
    dict(head_dim=24, sections=(12,)), dict(head_dim=512, sections=(256,)), dict(head_dim=64, sections=(16, 15)),
    dict(head_dim=64, sections=()), dict(head_dim=64, sections=(40, -8)), dict(head_dim=64, sections=(8, 8, 8, 4, 4)),
    dict(head_dim=64, sections=(32,), theta=0.0), dict(head_dim=64, sections=(32,), theta=float("inf")),
    dict(head_dim=64, sections=(32,), layout="pairs")])
def test_rotation_arguments(args):
    from reelcache_b200.ops.rope import AxisRope
    with pytest.raises(ConfigurationError):
        AxisRope(**args)


def test_wan_split_is_the_restore_tables():
    """The rotation that writes pages turns pairs as the restore's tables do."""
    from reelcache_b200.ops.rope import AxisRope
    from reelcache_b200.restore_kernels import RopeTable
    for d in (64, 128):
        assert tuple(AxisRope.wan(d).sections) == tuple(RopeTable.wan(d, 4).sections)


def test_cpu_tensors_are_refused():
    from reelcache_b200.ops import paged, rope
    from reelcache_b200.paged_cache import PagedKVCache
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    pages = torch.zeros(2, 8, 2, 64, dtype=torch.bfloat16)
    ints = torch.zeros(2, dtype=torch.int32)
    turn = rope.AxisRope.wan(64)
    with pytest.raises(UnsupportedError):
        rope.rotate(q, None, torch.zeros(1, 3, dtype=torch.int32), turn)
    with pytest.raises(UnsupportedError):
        paged.append(q, q, q, torch.zeros(1, 3, dtype=torch.int32), turn, pages, pages, ints[None], ints[:1], ints)
    with pytest.raises(UnsupportedError):
        paged.attention(q, pages, pages, ints[None], ints[:1], ints, max_q_len=1)
    with pytest.raises(UnsupportedError):
        paged.copy_pages(pages[None], ints, ints)
    with pytest.raises(UnsupportedError):
        PagedKVCache(1, 1, 64, pages=1, page_size=8, max_sessions=1, max_tokens=8, device="cpu")


def test_page_table_parts():
    from reelcache_b200.ops.paged import PageTable
    table = PageTable.empty(5, 3, 4, 16, "cpu")
    assert table.refcount.tolist() == [0] * 5 and table.lens.tolist() == [0] * 3
    assert table.block_table.shape == (3, 4) and bool((table.block_table == -1).all())
    table.block_table[1, 2] = 7
    assert int(table.state[5 + 3 + 4 + 2]) == 7  # parts of one tensor
    for state, pages, seqs in ((torch.zeros(20), 5, 3), (torch.zeros(19, dtype=torch.int32), 5, 3), (torch.zeros(8, dtype=torch.int32), 5, 3),
                               (torch.zeros(20, dtype=torch.int32), 0, 4), (torch.zeros(20, dtype=torch.int32), 5, 0)):
        with pytest.raises(ConfigurationError):
            PageTable(state, pages=pages, seqs=seqs, page_size=16)
