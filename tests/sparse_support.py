"""Plain forms of the 8-bit pages and of the choice of blocks, in 64 bits."""

import math

import torch

RANGE = {torch.bfloat16: (-124, 119), torch.float16: (-15, 7)}


def quantise(x, dtype):
    """Codes (as numbers) and exponents of rows ``x [..., d]`` of any type, by the format's definition in 64 bits: k the smallest
    integer with max|x| <= 448 * 2^k in the range of ``dtype``, codes to the nearest of four significant bits (steps of 2^-9 at
    least), ties to even. Rows with a value that is not finite: NaN, exponent 128."""
    x = x.double()
    low, high = RANGE[dtype]
    finite = torch.isfinite(x).all(dim=-1, keepdim=True)
    x = torch.where(finite, x, 0.0)
    top = x.abs().amax(dim=-1, keepdim=True)
    part, power = torch.frexp(top)  # top = part * 2^power with part from 1/2 to 1, and 448 = 0.875 * 2^9
    power = torch.where(top > 0, power - 9 + (part > 0.875), low).clamp(low, high)
    x = (x * torch.exp2(-power.double())).clamp(-448.0, 448.0)
    step = torch.exp2(torch.frexp(x.abs().clamp(min=2.0 ** -6))[1].double() - 4.0)
    codes = torch.round(x / step) * step
    return torch.where(finite, codes, math.nan), torch.where(finite, power, 128)[..., 0]


def held(pages, dtype=None):
    """What packed pages hold, 64 bits (or ``dtype``, exactly)."""
    power = pages.scales.view(torch.uint8).to(torch.int32)
    scale = torch.where(power == 255, math.nan, torch.exp2(power.double() - 127)).permute(1, 2, 0)[..., None]
    x = pages.codes.float().double() * scale
    return x if dtype is None else x.to(dtype)


def pack_pages(x, dtype):
    """Packed pages of ``x [pages, page_size, kv_heads, d]``."""
    from reelcache_b200.ops.paged import PackedPages
    codes, power = quantise(x, dtype)
    scales = (power + 127).to(torch.uint8).permute(2, 0, 1).contiguous()
    return PackedPages(codes.float().to(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))


def choose(q, means, table, kv_lens, cu_q, *, block, keep, query_block=1, causal=False, sinks=0, recent=0):
    """The choice of blocks, one query block and KV head at a time: ``[(first token, tokens, end, [blocks of each KV head])]``."""
    kv_heads, per_page = means.shape[2], means.shape[1]
    group = q.shape[1] // kv_heads
    items = []
    cu, lens = cu_q.tolist(), kv_lens.tolist()
    for s, total in enumerate(lens):
        n = cu[s + 1] - cu[s]
        for start in range(0, n, query_block):
            count = min(query_block, n - start)
            end = max(0, total - n + start + count) if causal else total
            blocks = -(-end // block)
            near = max(0, total - n + (start if causal else 0) - recent)
            high = min(blocks, near // block)
            low = min(high, -(-sinks // block))
            pooled = q[cu[s] + start:cu[s] + start + count].double().sum(dim=0)
            chosen = []
            for h in range(kv_heads):
                past = torch.arange(low, high, device=q.device)
                m = means[table[s, past // per_page].long(), past % per_page, h].double()
                score = (m @ pooled[h * group:(h + 1) * group].T).nan_to_num(nan=-math.inf).amax(dim=1) if len(past) else m.new_zeros(0)
                best = torch.sort(score, descending=True, stable=True).indices[:keep]
                chosen.append(list(range(low)) + sorted((best + low).tolist()) + list(range(high, blocks)))
            items.append((cu[s] + start, count, end, s, chosen))
    return items


def chosen_table(items, table, per_page, kv_heads, rooms, width, block, tokens_end):
    """What select_blocks returns for a choice: table, kv_lens and cu_q (lists)."""
    rows, lens, cu = [], [], []
    for first, count, end, s, chosen in items:
        rows.append([[int(table[s, b // per_page]) * per_page + b % per_page for b in blocks] + [-1] * (width - len(blocks)) for blocks in chosen])
        number = len(chosen[0])
        lens.append((number - 1) * block + end - (-(-end // block) - 1) * block if number else 0)
        cu.append(first)
    cu.append(items[-1][0] + items[-1][1] if items else tokens_end)
    while len(rows) < rooms:
        rows.append([[-1] * width for _ in range(kv_heads)])
        lens.append(0)
        cu.append(tokens_end)
    return rows, lens, cu
