"""One tiny end-to-end pass of the flagship path on a CUDA device (used by the driver's smoke check):
restore a compressed chunk history into a KV cache with the fused sm_100a kernel, run one tcgen05 GEMM, and take a step of
two forked sessions of a paged cache (rotation with gradient, append, attention, page table) and of one in 8 bits (attention over
all of it and over chosen blocks), checking all against fp64 / fp32 references."""

from __future__ import annotations

import numpy as np
import torch

from . import _hevc
from . import restore_kernels as rk
from .ops import _ext, gemm
from .ops.rope import AxisRope, rotate
from .paged_cache import PagedKVCache


def _paged_step(device):
    """Two forked sessions: a chunk together, then a token each; the error of the last attention against FP32."""
    rope = AxisRope.wan(64)
    cache = PagedKVCache(1, 2, 64, pages=16, page_size=16, max_sessions=3, max_tokens=96, device=device)
    kept = []
    root = cache.open()

    def step(pairs):
        batch = cache.extend(pairs)
        q, k, v = (torch.randn(batch.tokens, h, 64, device=device).bfloat16() for h in (4, 2, 2))
        positions = torch.randint(0, 500, (batch.tokens, 3), device=device, dtype=torch.int32)
        turned = cache.append(0, batch, q, k, v, positions, rope)
        kept.append((rotate(k, None, positions, rope)[0], v))
        return turned, cache.attend(0, batch, turned)

    step([(root, 40)])
    (other,) = cache.fork(root, [24])
    q, out = step([(other, 1), (root, 1)])
    worst = 0.0
    for i, n in enumerate((24, 40)):
        k, v = (torch.cat([kept[0][x][:n], kept[1][x][i:i + 1]]).float().repeat_interleave(2, dim=1) for x in (0, 1))
        p = torch.softmax(torch.einsum("hd,khd->hk", q[i].float(), k) / 8.0, dim=1)
        worst = max(worst, float((out[i].float() - torch.einsum("hk,khd->hd", p, v)).abs().max()))
    cache.close(root)
    assert cache.compact() == 2
    x = torch.randn(8, 2, 64, device=device, requires_grad=True)
    turned, _ = rotate(x, None, torch.randint(0, 500, (8, 3), device=device, dtype=torch.int32), rope)
    (grad,) = torch.autograd.grad(turned, x, turned.detach())
    assert torch.allclose(grad, x, atol=1e-4), "rotation gradient mismatch"  # turned there and back
    assert worst < 5e-2, "paged attention mismatch"
    return worst


def _packed_step(device):
    """A prompt and a token in a cache in 8 bits: the error of attention over all of it against FP32, and over all of its blocks."""
    cache = PagedKVCache(1, 2, 64, pages=16, page_size=16, max_sessions=2, max_tokens=96, device=device, packed=True, block=8)
    session = cache.open()
    for n in (70, 1):
        batch = cache.extend([(session, n)])
        q, k, v = (torch.randn(n, h, 64, device=device).bfloat16() for h in (4, 2, 2))
        cache.store(0, batch, k, v)
    k, v = (x.float().repeat_interleave(2, dim=1) for x in cache.read(0, [session]))
    p = torch.softmax(torch.einsum("hd,khd->hk", q[0].float(), k) / 8.0, dim=1)
    want = torch.einsum("hk,khd->hd", p, v)
    outs = [cache.attend(0, batch, q, causal=True, **how)[0].float() for how in ({}, dict(keep=20))]
    worst = max(float((out - want).abs().max()) for out in outs)
    few = cache.attend(0, batch, q, causal=True, keep=2)
    assert bool(few.isfinite().all()) and worst < 5e-2, "packed attention mismatch"
    return worst


def run(device):
    torch.manual_seed(0)
    rng = np.random.default_rng(0)
    frames, height, width, rank, heads, head_dim = 1, 8, 16, 64, 2, 128
    tokens = frames * height * width
    values = rng.standard_normal((tokens, rank)).astype(np.float32)
    pixels, affine, norm = _hevc.quantize_coefficients(values, "per_channel")
    layout = _hevc.video_layout(frames, height, width, rank)
    canvases = torch.from_numpy(_hevc.mosaic_all(pixels, layout)).to(device)
    scale, offset = rk.expand_affine(affine, norm, rank)
    source = rk.PictureSource.from_canvases(canvases, layout, [[s] for s in range(layout["segments"])], (0, 0),
                                            scale, offset)
    basis = (torch.randn(rank, heads * head_dim) / 16).half().to(device)
    cache = torch.zeros((1, tokens, heads, head_dim), dtype=torch.bfloat16, device=device)
    table = rk.RopeTable.wan(head_dim, 32, device=device)
    job = rk.ReconstructionJob(source, rk.NativeView(cache), (frames, height, width), basis,
                               rope=rk.RopePositions(table, (0, 0, 0)))
    rk.reconstruct([job], backend="fused", precision="fp16x2").release()  # the precision its bound describes
    _ext.check_status(device)
    expect, bound = rk.kernel_error_bound(job, "fp16x2")
    got = cache[0].reshape(tokens, -1).double()
    assert bool(((got - expect).abs() <= bound).all()), "fused restore exceeded its error bound"
    a = torch.randn(256, 128, device=device, dtype=torch.bfloat16)
    b = torch.randn(192, 128, device=device, dtype=torch.bfloat16)
    out = gemm.matmul_tn(a, b)
    torch.cuda.synchronize(device)
    _ext.check_status(device)
    ref = a.float() @ b.float().t()
    assert torch.allclose(out, ref, atol=1e-2, rtol=1e-3), "tcgen05 GEMM mismatch"
    paged_err, packed_err = _paged_step(device), _packed_step(device)
    _ext.check_status(device)
    return {"restore_max_err": float((got - expect).abs().max()), "gemm_max_err": float((out - ref).abs().max()),
            "paged_max_err": paged_err, "packed_max_err": packed_err}
