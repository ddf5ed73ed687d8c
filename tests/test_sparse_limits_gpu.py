"""The sizes that the choice of blocks takes, and its refusal of others."""

import pytest
import torch

from .paged_support import paged_batch
from .sparse_support import choose, chosen_table

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _call(heads, d, blocks, new=1):
    """A batch of two sequences, of which one fills its table of ``blocks`` blocks of 8."""
    g = torch.Generator(device="cuda").manual_seed(heads)
    k, _, table, kv_lens, cu_q = paged_batch(g, [new, new], [8 * blocks, 300], 1, d, 64, torch.bfloat16)
    q = torch.randn(2 * new, heads, d, generator=g, device="cuda").bfloat16()
    means = k.double().unflatten(1, (-1, 8)).mean(dim=2).bfloat16()
    return dict(q=q, means=means, block_table=table, kv_lens=kv_lens, cu_q=cu_q, block=8, keep=9, max_q_len=new, query_block=4, causal=True)


@pytest.mark.parametrize("heads,d,blocks", [(88, 128, 1024), (11, 128, 12288), (160, 64, 1024), (16, 64, 12288), (64, 128, 4096)])
@pytest.mark.parametrize("new", [1, 6])
def test_the_largest_groups_and_tables(heads, d, blocks, new):
    from reelcache_b200.ops import paged
    call = _call(heads, d, blocks, new)
    chosen = paged.select_blocks(**call)
    how = {name: call[name] for name in ("block", "keep", "query_block", "causal")}
    items = choose(call["q"], call["means"], call["block_table"], call["kv_lens"], call["cu_q"], **how)
    rows, lens, cu = chosen_table(items, call["block_table"], 8, 1, *chosen.table.shape[::2], 8, 2 * new)
    assert chosen.table.tolist() == rows and chosen.kv_lens.tolist() == lens and chosen.cu_q.tolist() == cu


@pytest.mark.parametrize("heads,d,blocks,what", [(96, 128, 1024, "a group of 96 heads with a block table of 1024 blocks"), (12, 128, 12288, "12 heads.*12288 blocks"),
                                                 (300, 64, 64, "too many heads"), (1, 64, 12296, "12296 blocks is wider")])
def test_larger_ones_are_refused(heads, d, blocks, what):
    from reelcache_b200.ops import paged
    with pytest.raises(RuntimeError, match=what):
        paged.select_blocks(**_call(heads, d, blocks))


def test_a_query_block_chooses_as_one():
    """Causal or not, all tokens of a query block make its choice: the first one's blocks follow the last one's query; with a query
    block for each token they do not."""
    from reelcache_b200.ops import paged
    call = {**_call(2, 64, 64, 4), "keep": 1}
    q = call.pop("q")
    other = q.clone()
    best = call["means"][int(call["block_table"][0, 5]), 3, 0]  # block 43
    other[3] = 1000.0 * best  # the last of the first sequence's tokens
    first, changed = (paged.select_blocks(x, **call).table for x in (q, other))
    assert first.shape[0] == changed.shape[0] == 2 and int(changed[0, 0, 0]) == int(call["block_table"][0, 5]) * 8 + 3
    assert not torch.equal(first[0], changed[0]) and torch.equal(first[1], changed[1])
    alone, after = (paged.select_blocks(x, **{**call, "query_block": 1}).table for x in (q, other))
    assert torch.equal(alone[:3], after[:3]) and not torch.equal(alone[3], after[3])
