"""Outputs of the paged operators are allocated as torch's own are: dispatch modes see them, and deterministic algorithms fill what
no kernel writes."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from .paged_support import paged_batch
from .sparse_support import pack_pages

pytestmark = pytest.mark.gpu


class _Allocations(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.shapes = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if func is torch.ops.aten.empty.memory_format:
            self.shapes.append(tuple(out.shape))
        return out


def _calls():
    """Calls with two rows of q (and of read's output) that belong to no sequence: the rows' slices of each output, by name."""
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v, table, kv_lens, cu_q = paged_batch(g, [3, 2], [70, 40], 2, 64, 16, torch.bfloat16)
    packed = [pack_pages(x, torch.bfloat16) for x in (k, v)]
    q = torch.randn(7, 4, 64, generator=g, device="cuda").bfloat16()
    long = torch.randn(7 * 40, 4, 64, generator=g, device="cuda").bfloat16()
    starts = torch.tensor([0, 70, 110], dtype=torch.int32, device="cuda")
    rows = torch.zeros(7, 2, 64, device="cuda").bfloat16()
    means = torch.zeros(k.shape[0], 1, 2, 64, device="cuda").bfloat16()
    at = (table, kv_lens, cu_q)
    return {
        "attention": lambda: paged.attention(q, k, v, *at, max_q_len=3, return_lse=True),
        "chunk attention": lambda: paged.attention(long, k, v, *at, max_q_len=40, return_lse=True),
        "packed attention": lambda: paged.attention(q, *packed, *at, max_q_len=3, return_lse=True),
        "expanded attention": lambda: paged.attention(long, *packed, *at, max_q_len=40, return_lse=True),
        "read": lambda: paged.read(*packed, table, starts, 112),
        "append": lambda: paged.append(q, rows, rows, torch.zeros(7, 3, dtype=torch.int32, device="cuda"), AxisRope.wan(64), *packed, *at),
        "choice": lambda: paged.select_blocks(q, means, *at, block=16, keep=1, max_q_len=3)[:3],
    }


@pytest.mark.parametrize("name", ["attention", "chunk attention", "packed attention", "expanded attention", "read"])
def test_rows_of_no_sequence_are_filled(name):
    call = _calls()[name]
    first = call()
    torch.use_deterministic_algorithms(True, warn_only=True)
    try:
        assert torch.utils.deterministic.fill_uninitialized_memory
        outs = call()
    finally:
        torch.use_deterministic_algorithms(False)
    held = 110 if name == "read" else 5
    for x, y in zip(outs, first):
        assert bool(x[held:].isnan().all()) and torch.equal(x[:held], y[:held])


@pytest.mark.parametrize("name", ["attention", "chunk attention", "packed attention", "expanded attention", "read", "append", "choice"])
def test_a_dispatch_mode_sees_the_outputs(name):
    call = _calls()[name]
    with _Allocations() as seen:
        outs = call()
    outs = outs if isinstance(outs, tuple) else (outs,)
    if name == "choice":  # (one allocation for the three of them)
        assert (sum(x.numel() for x in outs),) in seen.shapes
    else:
        assert all(tuple(x.shape) in seen.shapes for x in outs)
