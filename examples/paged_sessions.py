"""Forked video sessions over one paged KV cache on one GPU (CausVid-shaped DiT, random weights).

A session generates a few chunks; branches are forked from its head and from an earlier chunk (a rewind), every branch
generates its next chunk in one batched forward over the shared history, some branches end, and the pool is compacted.
Prints the pages that sharing saves and the time of a batched forward against one forward per session. Then a small stack of
causal attention layers with grouped heads reads a prompt and goes on token by token in forked sessions, which rotate their
rows on the way into the pages.

    python examples/paged_sessions.py --chunks 4 --branches 4
    python examples/paged_sessions.py --small          # a geometry for a quick look
"""

import argparse
import json
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from reelcache_b200.models.causal_wan import CAUSVID, CausalWanDiT  # noqa: E402
from reelcache_b200.ops import _ext  # noqa: E402
from reelcache_b200.ops.rope import AxisRope  # noqa: E402
from reelcache_b200.paged_cache import PagedKVCache  # noqa: E402

SMALL = dict(layers=2, dim=256, heads=2, ffn=512, text_dim=128, text_len=16, latent_height=8, latent_width=16)


def generate(model, cache, sessions, text_kv, latents, steps):
    """One chunk for every session: ``steps`` denoising forwards, then the clean pass that leaves the chunk's K and V."""
    chunk = model.cfg.chunk_tokens
    batch = cache.extend([(s, chunk) for s in sessions])
    x = latents
    for step in range(steps):
        flow = model.forward_sessions(x, 1000.0 * (1.0 - step / steps), cache, batch, text_kv)
        x = x - flow / steps
    model.forward_sessions(x, 0.0, cache, batch, text_kv)
    return x


def decode(*, layers=2, heads=8, kv_heads=2, head_dim=64, prompt=100, tokens=12, branches=3, device="cuda", seed=0):
    """A prompt in one session, then ``tokens`` steps of a token each in ``branches`` forks of it (outputs fed back as inputs).
    Returns the largest difference of the last step's rows from one pass over each branch's whole sequence, relative to
    their size, and the pages that the branches hold beyond the prompt's."""
    generator = torch.Generator(device=device).manual_seed(seed)
    dim = heads * head_dim
    draw = lambda *shape: torch.randn(*shape, device=device, generator=generator)  # noqa: E731
    w_in = [(draw(dim, dim + 2 * kv_heads * head_dim) / dim ** 0.5).bfloat16() for _ in range(layers)]
    w_out = [(draw(dim, dim) / dim ** 0.5).bfloat16() for _ in range(layers)]
    rope = AxisRope(head_dim, (head_dim // 2,), layout="halves")
    longest = prompt + tokens
    cache = PagedKVCache(layers, kv_heads, head_dim, pages=(branches + 1) * 2 * (longest // 16 + 2), page_size=16,
                         max_sessions=2 * branches + 1, max_tokens=longest, device=device)

    def step(pairs, x):
        batch = cache.extend(pairs)
        positions = torch.cat([torch.arange(length - n, length, dtype=torch.int32, device=device)
                               for n, length in zip(batch.counts, batch.lengths)])[:, None]
        for layer in range(layers):
            rows = (torch.nn.functional.layer_norm(x, (dim,)).bfloat16() @ w_in[layer]).view(x.shape[0], -1, head_dim)
            q, k, v = rows.split([heads, kv_heads, kv_heads], dim=1)
            q = cache.append(layer, batch, q, k, v, positions, rope)
            x = x + (cache.attend(layer, batch, q, causal=True).flatten(1) @ w_out[layer]).float()
        return x

    root = cache.open()
    x = draw(prompt, dim)
    last = step([(root, prompt)], x)[-1:]
    held = cache.pages - cache.free_pages
    forks = cache.fork(root, count=branches)
    rows = last + 0.1 * draw(branches, dim)  # every branch goes its own way
    inputs = []
    for _ in range(tokens):
        inputs.append(rows)
        out = step([(s, 1) for s in forks], rows)
        rows = torch.nn.functional.layer_norm(out, (dim,))
    beyond = cache.pages - cache.free_pages - held
    whole = [step([(cache.open(), longest)], torch.cat([x, *[r[i:i + 1] for r in inputs]]))[-1] for i in range(branches)]
    return float((out - torch.stack(whole)).abs().max() / out.abs().max()), beyond


def timed(call):
    torch.cuda.synchronize()
    start = time.perf_counter()
    result = call()
    torch.cuda.synchronize()
    return result, (time.perf_counter() - start) * 1e3


def run(cfg, *, chunks, branches, steps, device="cuda", seed=0):
    if chunks < 2 or branches < 2:
        raise ValueError("the example forks from two chunks into at least two branches")
    model = CausalWanDiT(cfg, device, seed=seed)
    generator = torch.Generator(device=device).manual_seed(seed)
    draw = lambda n: torch.randn(n, cfg.in_dim, cfg.frames_per_chunk, cfg.latent_height, cfg.latent_width,  # noqa: E731
                                 device=device, generator=generator)
    text_kv = model.encode_text(torch.randn(cfg.text_len, cfg.text_dim, device=device, generator=generator))
    frame = cfg.tokens_per_frame  # a latent frame to a page
    per_chunk = cfg.frames_per_chunk
    cache = PagedKVCache(cfg.layers, cfg.heads, cfg.head_dim, pages=(chunks + 2 * branches + 1) * per_chunk, page_size=frame,
                         max_sessions=branches + 1, max_tokens=(chunks + 2) * cfg.chunk_tokens, device=device)
    root = cache.open()
    for _ in range(chunks):
        generate(model, cache, [root], text_kv, draw(1), steps)
    history = cache.pages - cache.free_pages

    late = cache.fork(root, count=branches // 2)                                     # other continuations of the head
    early = cache.fork(root, [(chunks - 1) * cfg.chunk_tokens] * (branches - len(late)))  # a rewind by one chunk
    cache.close(root)
    sessions = late + early
    shared = cache.pages - cache.free_pages
    latents = draw(branches)
    generate(model, cache, sessions, text_kv, latents, steps)                        # warm
    batch = cache.again([(s, cfg.chunk_tokens) for s in sessions])
    together, batched_ms = timed(lambda: model.forward_sessions(latents, 500.0, cache, batch, text_kv))
    singles = [cache.again([(s, cfg.chunk_tokens)]) for s in sessions]
    apart, single_ms = timed(lambda: torch.cat([model.forward_sessions(latents[i:i + 1], 500.0, cache, b, text_kv)
                                                for i, b in enumerate(singles)]))
    difference = float((together - apart).norm() / apart.norm())

    cache.close(*sessions[::2])
    in_use = cache.compact()
    rest = sessions[1::2]
    generate(model, cache, rest, text_kv, draw(len(rest)), steps)                    # generation goes on where pages moved
    difference_by_token, beyond = decode(device=device, seed=seed)
    _ext.check_status(device)
    return {"token_by_token_difference": difference_by_token, "token_by_token_pages_of_branches": beyond, "tokens_per_page": frame, "page_bytes": cache.nbytes // cache.pages, "history_pages": history,
            "pages_after_forks": shared, "pages_if_copied": len(late) * history + len(early) * (history - per_chunk),
            "batched_forward_ms": round(batched_ms, 2), "separate_forwards_ms": round(single_ms, 2),
            "batched_vs_separate_difference": difference, "pages_after_compaction": in_use,
            "pages_used_at_the_end": cache.pages - cache.free_pages}


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--chunks", type=int, default=4, help="chunks of history before the forks")
    parser.add_argument("--branches", type=int, default=4)
    parser.add_argument("--steps", type=int, default=2, help="denoising steps of a chunk")
    parser.add_argument("--small", action="store_true")
    args = parser.parse_args(argv)
    cfg = CAUSVID.scaled(**SMALL) if args.small else CAUSVID
    print(json.dumps(run(cfg, chunks=args.chunks, branches=args.branches, steps=args.steps), indent=1))


if __name__ == "__main__":
    main()
