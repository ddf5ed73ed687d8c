"""Where the paged operators could go wrong: calls without a pause between them, values and lengths at the edges, batches
that are out of date, and the long forms of attention."""

import math

import pytest
import torch

from .paged_support import attend, paged_batch, within

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
