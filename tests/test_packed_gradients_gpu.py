"""No packed operator has a gradient or a tangent: each refuses tensors that want one."""

import pytest
import torch

from .paged_support import paged_batch
from .sparse_support import pack_pages

pytestmark = pytest.mark.gpu

CALLS = ["attention", "read", "store", "append", "block_means"]


@pytest.fixture(autouse=True)
def _checked(cuda_device):
    from reelcache_b200.ops import _ext
    yield
    _ext.check_status(cuda_device)


def _setup(name):
    """A call that takes packed pages of K and V, and such pages."""
    from reelcache_b200.ops import paged
    from reelcache_b200.ops.rope import AxisRope
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v, table, kv_lens, cu_q = paged_batch(g, [2], [20], 2, 64, 16, torch.bfloat16)
    rows, q = torch.randn(2, 2, 64, device="cuda").bfloat16(), torch.randn(2, 4, 64, device="cuda").bfloat16()
    means = torch.zeros(k.shape[0], 1, 2, 64, device="cuda").bfloat16()
    positions = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    at = (table, kv_lens, cu_q)
    call = {"attention": lambda kp, vp: paged.attention(q, kp, vp, *at, max_q_len=2), "read": lambda kp, vp: paged.read(kp, vp, table, cu_q, 2),
            "store": lambda kp, vp: paged.store(rows, rows, kp, vp, *at),
            "append": lambda kp, vp: paged.append(q, rows, rows, positions, AxisRope.wan(64), kp, vp, *at),
            "block_means": lambda kp, vp: paged.block_means(kp, means, *at, max_q_len=2)}[name]
    return call, [pack_pages(x, torch.bfloat16) for x in (k, v)]


@pytest.mark.parametrize("part", ["codes", "scales"])
@pytest.mark.parametrize("name,which", [(name, which) for name in CALLS for which in (0, 1) if name != "block_means" or which == 0])
def test_pages_that_want_a_gradient_are_refused(name, which, part):
    call, pages = _setup(name)
    pages[which] = pages[which]._replace(**{part: getattr(pages[which], part).clone().requires_grad_()})
    with pytest.raises(RuntimeError, match="no gradient"):
        call(*pages)
    with torch.no_grad():
        call(*pages)


@pytest.mark.parametrize("part", ["codes", "scales"])
@pytest.mark.parametrize("name", CALLS)
def test_pages_with_a_tangent_are_refused(name, part):
    from torch.autograd import forward_ad
    call, pages = _setup(name)
    with forward_ad.dual_level():
        x = getattr(pages[0], part)
        pages[0] = pages[0]._replace(**{part: forward_ad.make_dual(x, x.clone())})
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(*pages)
